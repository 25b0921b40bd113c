// Attention of one new token per request over an 8-bit cache (kv_e4m3.cuh), through block tables.
//
//     s_j = scale * 2^(Ek_j - 127) * sum_d q_d kcode_jd,   out = sum_j e^(s_j - m) 2^(Ev_j - 127) vcode_j / sum_j e^(s_j - m)
//
// over the context's positions j (the last `window` of them), m their largest s_j; float32 but for what is said below.
//
// The step is a stream of codes from memory, 2 (hd + 1) bytes per token and KV head, so all query heads of a KV head (16 at
// most, or 8) share what a block fetches.  Work is cut by the contexts themselves: requests, KV heads and tiles of 16 to 64
// tokens are numbered through, and every warp of a grid that fills the SMs once takes an equal run of tiles, wherever requests begin
// and end in it; so contexts of any lengths fill the GPU, and no scratch grows with them.  Each warp has a ring of tiles in shared
// memory of its own, filled by 16-byte asynchronous copies one to three tiles ahead (the warps of an SM have 96 KB or more under
// way) and on into the next request, so that warps never wait for one another while they stream.
//
// Bound by memory while it streams, and by latency before and after that.  Measured, us, and what the bytes take at the rate of a copy: 64
// requests of 1 to 7,650 tokens, 28 heads over 4 of 128, 251 MB 55 and 38.9 (the stream itself 36; the first tiles come after 6,
// the last pieces are added up 8 after the last tile); four of 65,536 to 131,072, 40 heads over 8, 861 MB 160 and 133; 8 of 1,024, 12 over
// 2, 4.3 MB 13 and 0.7: lengths, block table and rows are three trips to memory one after the other, and joining the pieces is four.
//
// Codes become half-precision numbers exactly (cvt) on their way into mma.sync.m16n8k16, which costs less here than it could
// save elsewhere: at the rate of memory the tensor cores are a fifth busy.  Tokens are the M side of S^T = K Q^T and the codes'
// entries the M side of O^T = V^T P^T, so that eight query heads (N) fill what sixteen would, and a thread's 16 bytes of K are
// four k-steps of one product: which entries a k-step takes is the same for K and Q and otherwise free.  For V^T P^T two tokens'
// bytes are paired by a byte permutation before cvt.  S^T's accumulators become P^T's fragments by movmatrix.
//
// Query heads are scaled by a power of two each into half precision's upper range (bfloat16's 8 bits are kept; what falls below
// 2^-39 of the head's largest entry is dropped).  The powers of K multiply scores in float32.  Those of V are taken into
// the exponent: weights are p_j = 2^(s_j log2 e + Ev_j - 127 - M + 14), M the running maximum of s_j log2 e + max(Ev_j, 67) - 127, in half
// precision (11 bits: off by at most 2^-11 of themselves, or by 2^-25, which is 2^-38 of the largest contribution).  A row of zeros
// contributes nothing, whatever its power of 127 says, and has Ev_j = 67 here: it would otherwise push the others down to where half
// precision has few bits.  (With a power below 67, values below 2^-51, an error is at most 2^-90.)  The denominator, float32, sums
// 2^(s_j log2 e - M + 14) 2^24, which p_j is made from by its power: below 2^99 a token, and no number any more only where p_j is below 2^-31.
// Sums go from one maximum to the next by a factor that is 2^-126 at least, which suffices where powers, those below 67 counting as
// that, are no more than 100 apart.
//
// A segment (request, KV head and group) that lies in one warp's run is finished by it.  At the end of its run a block adds up
// its warps' pieces of shared segments in order; the pieces of one that several blocks share go to scratch of two per block, and
// the block that comes last merges them in the blocks' order (more than 24: eight at a time first, each by the last of the
// eight).  The result does not depend on who comes last.
#include "attention_mma.cuh"
#include "kv_e4m3.cuh"

struct DecodeE4m3Params {
    const void* q; int q_stride; void* out;
    const uint8_t* k; const uint8_t* v; const uint8_t* k_exp; const uint8_t* v_exp;
    const int* block_tables; const int* ctx_lens; const int* q_start;
    int requests, nh, nkv, hd, page_size, max_blocks, num_pages, window;
    float scale;
    int* status;
    int early;               // 1: lengths, tables and all rows but a request's own newest are older than the kernel in front; 2: lengths and tables are
    // the streaming kernel
    int page_shift;          // log2 of the page size, or -1
    int teams;               // KV heads that long walks take side by side
    int groups, heads_each;  // groups of query heads per KV head, heads in a group (the last may have fewer)
    float* heads_o;          // [4 * blocks][8 or 16][hd]: ends of segments that an earlier warp began
    float* part_o;           // [blocks][teams][2][8 or 16][hd]
    float* part_ml;          // [blocks][teams][2][8 or 16][2]
    int* counters;           // [blocks][4] (by the block that a segment begins in: one of a team goes on) and [blocks][4][2], zero between launches
    int least_rows, most_rows;  // portions: the requests that are served
};

#define WARPS 4
#define LEAST_POWER 67
#define SUMS_UP 24  // sums of weights are held times 2^24
#define MERGE_AT_ONCE 8
#define MOST_TEAMS 4
#define TEAMS_FROM_BYTES 170000000LL

__device__ __forceinline__ void mma_half(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 16 bytes, or zeros where `there` is false (nothing is read then)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int HD, int NT>
struct Stream {
    static constexpr int CH = HD / 16;  // 16-byte chunks of a row
    // Tokens of a tile: what a tile costs besides its products (looking up pages, the maxima's way over the lanes) is shared by
    // more of them where rows are short, and rings stay deep enough for two blocks an SM where rows are long.
    static constexpr int TOKENS = HD <= 64 ? 64 : HD <= 128 ? 32 : 16;
    static constexpr int TILE_BYTES = TOKENS * HD;  // K or V of a tile
    static constexpr int PER_SM = HD <= 128 && NT == 1 ? 3 : 2;  // blocks on an SM (registers: 168, 255)
    static constexpr int FIT = 196608 / PER_SM / (WARPS * 2 * TILE_BYTES);
    static constexpr int ST = FIT > 8 ? 8 : FIT;       // tiles in a warp's ring
    static constexpr int RING = WARPS * ST * 2 * TILE_BYTES;
    // Where chunk c of row r lies.  Rows of 128 bytes and multiples are swizzled so that the reads below (K: two rows' four chunks
    // at a time; V: a chunk of four rows two apart) meet no bank twice; of 64 bytes: the same over lines of two rows.
    static __device__ __forceinline__ int at(int r, int c) {
        if (HD % 128 == 0) return r * HD + ((c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) << 4);
        if (HD == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
        return r * HD + (c << 4);
    }
    // A lane copies chunks lane, lane + 32, ..  Where the j-th lies, from where the first does: rows of a power of two of chunks.
    static __device__ __forceinline__ int copied(int first, int j, int lane) {
        if (HD == 128) return (first ^ ((j & 1) << 6)) + j * 512;
        if (HD == 256) return (first ^ ((j & 3) << 5)) + j * 512;
        if (32 % CH == 0) return first + j * 512;
        const int i = j * 32 + lane;
        return at(i / CH, i % CH);
    }
};

// e4m3 pairs of a word's halves as half-precision pairs
__device__ __forceinline__ void halves_of(uint32_t word, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(word));
}

// A run of tiles through requests and segments: which tile it stands at.
struct Walk {
    int s, ctx, begin, tiles;  // the request, its context, the first position it sees, its tiles
    int n, groups;             // tokens that it brings, groups of their query heads per KV head
    int seg, tile;             // KV head and group; tile of it
    int left;                  // units of the run that are left
};

// Part of a segment that several warps share.
struct Piece {
    int segment;     // the unit before its tiles, and the team; -1: there is none
    int row, head;   // the request's first row, the KV head's first query head
    int first, rows; // its rows (of token and head in the group of query heads)
    int team;
    int first_block, blocks;  // which blocks have pieces of it
};

template <int HD, int NT, bool PORTIONS>
__global__ void __launch_bounds__(WARPS * 32, Stream<HD, NT>::PER_SM) decode_e4m3_kernel(const DecodeE4m3Params p) {
    using C = Stream<HD, NT>;
    static_assert(!PORTIONS || 8 * NT <= 32, "a lane to a row");
    constexpr int ROWS = 8 * NT, ST = C::ST, CH = C::CH, TOKENS = C::TOKENS;
    constexpr int U = TOKENS / 16, HALVES = (TOKENS + 31) / 32;  // products' 16 tokens; a lane's tokens when pages are looked up
    constexpr int WORDS = HD / 32;  // a thread's 4-byte words of a V row
    extern __shared__ __align__(128) uint8_t ring_s[];
    __shared__ uint32_t row_s[WARPS][ST][TOKENS];       // 16-byte chunk where a token's row begins; ~0: it does not count
    __shared__ uint32_t power_at_s[WARPS][ST][TOKENS];  // where its powers are
    __shared__ float m_s[2 * WARPS][ROWS], l_s[2 * WARPS][ROWS], f_s[2 * WARPS][ROWS];
    __shared__ Piece piece_s[2 * WARPS];  // of every warp: the end of a segment that began before its run, and what its run ends in
    __shared__ float top_s[2 * WARPS][ROWS], total_s[2 * WARPS][ROWS];  // of a group of pieces, at its first
    __shared__ int limit_s[WARPS][PORTIONS ? ROWS : 1];
    __shared__ int shared_s[2 * MOST_TEAMS], last_s[2 * MOST_TEAMS], final_s;
    // (early: what the kernel in front writes, queries and the newest rows, is waited for only where it is first needed)
    bool waited = PORTIONS || !p.early;
    if (waited)
        pdl_enter();
    else
        pdl_launch_dependents();
    auto wait = [&]() {
        if (!waited) pdl_wait();
        waited = true;
    };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int each = p.nh / p.nkv;  // query heads of a KV head
    auto tokens_of = [&](int s) -> int {  // that request s brings; 0: it is not served here
        if (!PORTIONS) return p.q_start == nullptr || p.q_start[s + 1] - p.q_start[s] == 1 ? 1 : 0;
        const int n = p.q_start[s + 1] - p.q_start[s];
        return n >= p.least_rows && n <= p.most_rows ? n : 0;
    };
    auto context_of = [&](int s) -> int { return min(p.ctx_lens[s], p.max_blocks * p.page_size); };
    auto begin_of = [&](int ctx, int n) { return p.window > 0 ? max(0, ctx - (PORTIONS ? n : 1) + 1 - p.window) : 0; };
    auto tiles_of = [&](int ctx, int n) {
        return ctx <= 0 || n <= 0 ? 0 : (ctx + TOKENS - 1) / TOKENS - begin_of(ctx, n) / TOKENS;
    };
    auto groups_of = [&](int n) { return PORTIONS ? (n * each + ROWS - 1) / ROWS : p.groups; };
    // Units are numbered through requests, teams' worth of KV heads, groups and tiles; every team of a block has the same ones.
    // A segment is its tiles and, before them, a unit for what changing to it costs (about a tile's time).  A block's run is a
    // whole number of equal runs for a team's warps.  Every warp finds its own: four neighbouring requests per lane, 128 at a time.
    const int chunks = (p.requests + 127) / 128;
    int context[4], tokens[4], total = 0;
    auto look_at = [&](int c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = c * 128 + 4 * lane + j;
            tokens[j] = s < p.requests ? tokens_of(s) : 0;
            context[j] = tokens[j] > 0 ? context_of(s) : -1;
        }
    };
    for (int c = chunks - 1; c >= 0; --c) {  // (the last one looked at is the first: what it holds is used again below)
        look_at(c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int tiles = tiles_of(context[j], tokens[j]);
            if (tiles > 0) total += groups_of(tokens[j]) * (tiles + 1);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // Rows that are no multiple of 128 bytes share lines with their neighbours' rows (p.teams > 1), and the L2 fetches whole lines:
    // as many KV heads, neighbours in memory, are walked at the same time by teams of the block's warps, so that a line comes once.
    // Not where all that is read stays in the L2 (126 MB) until the neighbour comes anyway: one team's four warps leave a segment
    // in fewer pieces.  Measured, cold, one team and two: 16 KV heads of 64, 100 MB 36.7 and 39.0 us, 200 MB 76.5 and 56.2, 400 MB 154 and
    // 90; 2 of 96, 200 MB 53.6 and 59.4, 400 MB 137 and 92; 4 of 32 (four teams), 100 MB 50.9 and 65.0, 200 MB 106 and 93.
    const int teams = !PORTIONS && (long long)total * p.nkv * 2 * C::TILE_BYTES >= TEAMS_FROM_BYTES ? p.teams : 1;
    const int of_team = WARPS / teams, team = warp / of_team, member = warp - team * of_team, warps = gridDim.x * of_team;
    // A run's least: a unit, which takes 1.5 us, where segments then have no more blocks' pieces than are added up at once; two where they
    // are longer.  Measured, us, runs of one and of two: 2 requests of 411 and 96 tokens, 12 heads over 2, store in front, 11.3 and 12.5; 8 of 300,
    // 28 over 4 11.7 and 13.5; 8 of 1,000, 12 over 2, store in front, 13.3 and 12.7 (beginning under the kernel in front 12.9 and 11.5).
    const int least = PORTIONS || total > p.requests * p.groups * MERGE_AT_ONCE * WARPS ? 2 : 1;
    const int kv_units = p.nkv / teams;
    total *= kv_units;
    const int quota = max(least, (total + warps - 1) / warps), block_units = quota * of_team;
    const int first = (int)min((long long)(blockIdx.x * of_team + member) * quota, (long long)total);
    auto zeros = [&]() {  // the rows of requests without a context
        for (int s = blockIdx.x; s < p.requests; s += gridDim.x) {
            if (PORTIONS || tokens_of(s) == 0 || context_of(s) > 0) continue;
            const int row = p.q_start != nullptr ? p.q_start[s] : s;
            for (int i = tid; i < p.nh * HD; i += blockDim.x) ((bf16*)p.out)[(size_t)row * p.nh * HD + i] = __float2bfloat16_rn(0.f);
        }
    };
    if ((long long)blockIdx.x * block_units >= total) {
        wait();
        zeros();
        return;
    }
    Walk at = {};
    at.left = min(total, first + quota) - first;
    int seg_unit = 0;  // of the segment that the run stands in: the unit before its tiles
    if (at.left > 0) {
        int before = 0, skip = 0;
        for (int c = 0; c < chunks; ++c) {
            if (c > 0) look_at(c);
            int units[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int tiles = tiles_of(context[j], tokens[j]);
                units[j] = tiles > 0 ? kv_units * groups_of(tokens[j]) * (tiles + 1) : 0;
                sum += units[j];
            }
            int upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int chunk = __shfl_sync(0xffffffffu, upto, 31);
            if (first < before + chunk) {
                int from = before + upto - sum, mine = 0, ctx = context[0], n = tokens[0];
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (mine == j && first >= from + units[j]) {
                        from += units[j];
                        mine = j + 1;
                        ctx = context[j + 1];
                        n = tokens[j + 1];
                    }
                const int who = __ffs(__ballot_sync(0xffffffffu, first < before + upto)) - 1;
                skip = first - __shfl_sync(0xffffffffu, from, who);
                at.s = c * 128 + 4 * who + __shfl_sync(0xffffffffu, mine, who);
                at.ctx = __shfl_sync(0xffffffffu, ctx, who);
                at.n = __shfl_sync(0xffffffffu, n, who);
                break;
            }
            before += chunk;
        }
        at.tiles = max(1, tiles_of(at.ctx, at.n));
        at.begin = begin_of(at.ctx, at.n);
        at.groups = groups_of(at.n);
        at.seg = skip / (at.tiles + 1);
        skip -= at.seg * (at.tiles + 1);
        seg_unit = first - skip;
        at.tile = max(0, skip - 1);
        if (skip == 0) --at.left;
    }
    auto enter = [&](Walk& w, int s) {  // the next request from s on that has tiles
        for (; s < p.requests; ++s) {
            w.s = s;
            w.n = tokens_of(s);
            w.ctx = context_of(s);
            w.tiles = tiles_of(w.ctx, w.n);
            w.begin = begin_of(w.ctx, w.n);
            w.groups = groups_of(w.n);
            if (w.tiles > 0) return;
        }
        w.ctx = 0;  // (lengths that change under the call: tokens that do not count)
        w.tiles = 0x7FFFFFFF;
    };
    // A segment's rows: of single tokens the query heads of a group; of portions (token, head of the KV head's) in this order, 16
    // to a group.  Row x of a KV head is that of token x / each and head x % each.
    auto query_row = [&](const Walk& w) { return p.q_start != nullptr ? p.q_start[w.s] : w.s; };
    auto kv_head = [&](const Walk& w) { return (!PORTIONS && p.groups == 1 ? w.seg : w.seg / w.groups) * teams + team; };
    auto first_of = [&](const Walk& w) { return !PORTIONS && p.groups == 1 ? 0 : w.seg % w.groups * (PORTIONS ? ROWS : p.heads_each); };
    auto rows_of = [&](const Walk& w) { return PORTIONS ? min(ROWS, w.n * each - first_of(w)) : min(p.heads_each, each - first_of(w)); };
    auto row_at = [&](int row, int head, int x, int stride) {  // where row x of a KV head begins in q or out
        return PORTIONS ? (size_t)(row + x / each) * stride + (size_t)(head + x % each) * HD : (size_t)row * stride + (size_t)(head + x) * HD;
    };
    auto call_queries = [&](const Walk& w) {  // brings a segment's queries near, ahead of their use
        const int row = query_row(w), head = kv_head(w) * each, x0 = first_of(w), rows = rows_of(w);
        for (int i = lane; i < rows * (HD / 16); i += 32) {  // a sector each
            uint32_t unused;
            asm volatile("ld.global.u32 %0, [%1];" : "=r"(unused) : "l"((const bf16*)p.q + row_at(row, head, x0 + i / (HD / 16), p.q_stride) + i % (HD / 16) * 16));
        }
    };
    auto step = [&](Walk& w, int tiles) {  // so many tiles on within its segment, and on to the next one's first
        w.tile += tiles;
        w.left -= tiles;
        if (w.tile == w.tiles) {
            w.tile = 0;
            --w.left;
            if (++w.seg == kv_units * w.groups) {
                w.seg = 0;
                if (w.left > 0) enter(w, w.s + 1);
            }
            return w.left > 0;
        }
        return false;  // (whether it stands in a new segment)
    };
    uint8_t* my_ring = ring_s + warp * ST * 2 * C::TILE_BYTES;
    const uint32_t my_ring_addr = smem_addr(my_ring);
    // ---- fetching: ST - 1 tiles ahead of the products, through the segments' ends ----
    Walk ahead = at;
    int fetch_stage = 0, ahead_page[HALVES], ahead_pos = 0;
    const int copy_lane = C::at(lane / CH, lane % CH);
    auto look_up = [&]() {  // the pages of this lane's tokens of the tile that is fetched next
        if (ahead.left <= 0) return;
        ahead_pos = (ahead.begin / TOKENS + ahead.tile) * TOKENS + lane;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int pos = ahead_pos + 32 * h;
            ahead_page[h] = -1;
            if ((TOKENS >= 32 || lane < TOKENS) && pos >= ahead.begin && pos < ahead.ctx)
                ahead_page[h] = p.block_tables[(size_t)ahead.s * p.max_blocks + (p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size)];
        }
    };
    auto fetch = [&]() {
        if (ahead.left > 0) {
            if (ahead.tile == ahead.tiles - 1) wait();  // (the request's newest row is in this tile)
            const int kvh = kv_head(ahead);
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int pos = ahead_pos + 32 * h, page = ahead_page[h];
                uint32_t row = ~0u, power_at = 0;
                if (page >= 0 && page < p.num_pages) {
                    const int off = p.page_shift >= 0 ? pos & (p.page_size - 1) : pos % p.page_size;
                    row = ((uint32_t)(page * p.page_size + off) * p.nkv + kvh) * CH;
                    power_at = ((uint32_t)page * p.nkv + kvh) * p.page_size + off;
                } else if ((TOKENS >= 32 || lane < TOKENS) && pos >= ahead.begin && pos < ahead.ctx) {
                    cw_report(p.status, CW_ST_PAGE_RANGE, ahead.s, page);
                }
                if (TOKENS >= 32 || lane < TOKENS) {
                    row_s[warp][fetch_stage][32 * h + lane] = row;
                    power_at_s[warp][fetch_stage][32 * h + lane] = power_at;
                }
            }
            __syncwarp();
            const uint32_t base = my_ring_addr + fetch_stage * 2 * C::TILE_BYTES;
#pragma unroll
            for (int j = 0; j < TOKENS * CH / 32; ++j) {
                const int i = j * 32 + lane;
                const uint32_t from = row_s[warp][fetch_stage][32 % CH == 0 ? j * (32 / CH) + lane / CH : i / CH];
                const bool there = from != ~0u;
                const size_t src = (size_t)(there ? from + (32 % CH == 0 ? lane % CH : i % CH) : 0u) * 16;
                const uint32_t dst = base + C::copied(copy_lane, j, lane);
                copy16(dst, p.k + src, there);
                copy16(dst + C::TILE_BYTES, p.v + src, there);
            }
            if (++fetch_stage == ST) fetch_stage = 0;
            const bool other = step(ahead, 1);
            look_up();
            if (other) {
                wait();
                call_queries(ahead);
            }
        }
        cp_async_commit();
    };
    // a lane looks up the powers of token 8 t + g (and 32 further) a tile ahead of their use: K's, V's, and whether the token counts
    uint32_t k_power[HALVES], v_power[HALVES], counts[HALVES];
    auto look_at_powers = [&](int stage) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int token = 32 * h + 8 * (TOKENS >= 32 ? t : t & 1) + g;
            const uint32_t i = power_at_s[warp][stage][token];
            counts[h] = row_s[warp][stage][token];
            k_power[h] = p.k_exp[i];
            v_power[h] = p.v_exp[i];
        }
    };
    look_up();
    if (p.early == 2) wait();
    if (at.left > 0 && waited) call_queries(at);
#pragma unroll 1
    for (int i = 0; i < ST - 1; ++i) fetch();
    __syncwarp();
    wait();
    int stage = 0;
    if (at.left > 0) look_at_powers(0);
    if (lane < 2) piece_s[2 * warp + lane].segment = -1;
    // where this lane's K pieces and V words lie in a tile (rows 16 and 8 further: the same swizzle)
    const int k_at = C::at(g, HD % 64 == 0 ? t : t >> 1) + (HD % 64 == 0 ? 0 : 8 * (t & 1));
    constexpr int PIECE = HD % 64 == 0 ? 16 : 8, STEPS = PIECE / 4, PIECES = HD / (4 * PIECE);
    while (at.left > 0) {
        const int row = query_row(at), head = kv_head(at) * each, x0 = first_of(at), rows = rows_of(at);
        const int n_tiles = min(at.tiles - at.tile, at.left);
        // ---- the group's queries, as B fragments over the entries that a lane's pieces of K hold: half precision, a power of two out ----
        uint32_t qb[NT][PIECES][STEPS][2];
        float qf[NT][2], m[NT][2], l[NT][2], o[NT][HD / 16][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bf16* q = (const bf16*)p.q + row_at(row, head, x0 + min(8 * n + g, rows - 1), p.q_stride);
            float big = 0.f;
#pragma unroll
            for (int b = 0; b < PIECES; ++b)
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t w = 0;
                        if (8 * n + g < rows) w = *reinterpret_cast<const uint32_t*>(q + b * 4 * PIECE + t * PIECE + 4 * i + 2 * e);
                        qb[n][b][i][e] = w;
                        big = fmaxf(big, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xFFFF0000u))));
                    }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int up = big > 0.f ? min(126, 141 - (int)((__float_as_uint(big) >> 23) & 255)) : 0;  // big becomes 2^14 to 2^15
            const float by = __int_as_float((127 + up) << 23);  // (-114 <= up <= 126)
#pragma unroll
            for (int b = 0; b < PIECES; ++b)
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t w = qb[n][b][i][e];
                        qb[n][b][i][e] = half2_of(__uint_as_float(w << 16) * by, __uint_as_float(w & 0xFFFF0000u) * by);
                    }
            const float back = p.scale * 1.4426950408889634f * __int_as_float((127 - up) << 23);  // of head 8 n + g, lanes 4 g ..
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                qf[n][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
                m[n][e] = -INFINITY;
                l[n][e] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
        }
        // (portions) the last position that row x sees: of token x / each
        const int before = at.ctx - at.n, seen_by_all = before + x0 / each, seen_by_any = before + (x0 + rows - 1) / each;
        int pos0 = (at.begin / TOKENS + at.tile) * TOKENS;
        if (PORTIONS) {
            if (lane < ROWS) limit_s[warp][lane] = before + min(x0 + lane, x0 + rows - 1) / each;
            __syncwarp();
        }
        for (int i = 0; i < n_tiles; ++i, pos0 += TOKENS) {
            fetch();
            cp_async_wait<ST - 1>();
            __syncwarp();
            const int next = stage + 1 == ST ? 0 : stage + 1;
            uint32_t powers[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) powers[h] = counts[h] == ~0u ? 0u : k_power[h] | v_power[h] << 8 | 1u << 16;
            if (i + 1 < n_tiles || ahead.left > 0 || fetch_stage != next) look_at_powers(next);
            const uint8_t* kt = my_ring + stage * 2 * C::TILE_BYTES;
            const uint8_t* vt = kt + C::TILE_BYTES;
            stage = next;
            if (PORTIONS && (pos0 > seen_by_any || (p.window > 0 && pos0 + TOKENS - 1 <= seen_by_all - p.window))) {
                __syncwarp();  // no row sees any of the tile
                continue;
            }
            float sc[NT][U][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int u = 0; u < U; ++u) sc[n][u][0] = sc[n][u][1] = sc[n][u][2] = sc[n][u][3] = 0.f;
#pragma unroll
            for (int b = 0; b < PIECES; ++b) {
                const uint8_t* kb = kt + (HD % 128 == 0 ? (k_at ^ ((b & 1) << 6)) + (b >> 1) * 128 : k_at + b * 4 * PIECE);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    uint32_t lo[STEPS], hi[STEPS];  // rows g and g + 8
                    if (PIECE == 16) {
                        const uint4 x = *reinterpret_cast<const uint4*>(kb + 16 * u * HD), y = *reinterpret_cast<const uint4*>(kb + (16 * u + 8) * HD);
                        lo[0] = x.x; lo[1] = x.y; lo[STEPS - 2] = x.z; lo[STEPS - 1] = x.w;
                        hi[0] = y.x; hi[1] = y.y; hi[STEPS - 2] = y.z; hi[STEPS - 1] = y.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(kb + 16 * u * HD), y = *reinterpret_cast<const uint2*>(kb + (16 * u + 8) * HD);
                        lo[0] = x.x; lo[1] = x.y;
                        hi[0] = y.x; hi[1] = y.y;
                    }
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        uint32_t a[4];
                        halves_of(lo[k], a[0], a[2]);
                        halves_of(hi[k], a[1], a[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            if (!PORTIONS || 8 * n < rows) mma_half(sc[n][u], a, qb[n][b][k][0], qb[n][b][k][1]);
                    }
                }
            }
            bool rare = false;  // rows of zeros, or of values below 2^-51
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const uint32_t ev = (powers[h] >> 8) & 255;
                rare |= (powers[h] >> 16) != 0 && (ev == 127 || ev < LEAST_POWER);
            }
            rare = __any_sync(0xffffffffu, rare);
            if (__builtin_expect(rare, 0)) {
#pragma unroll 1
                for (int h = 0; h < HALVES; ++h) {
                    const int token = 32 * h + 8 * (TOKENS >= 32 ? t : t & 1) + g;
                    uint32_t codes = 0;
#pragma unroll 1
                    for (int c = 0; c < CH; ++c) {
                        const uint4 x = *reinterpret_cast<const uint4*>(vt + C::at(token, c));
                        codes |= x.x | x.y | x.z | x.w;
                    }
#pragma unroll
                    for (int i = 0; i < HALVES; ++i)  // (registers, not an array in memory)
                        if (i == h && ((powers[i] >> 8) & 255) == 127 && (codes & 0x7F7F7F7Fu) == 0) powers[i] = (powers[i] & ~0xFF00u) | LEAST_POWER << 8;
                }
            }
            // scores of tokens 8 x + g (x = 2 u, 2 u + 1) for heads 2 t, 2 t + 1
            float ev[2 * U], up[2 * U];  // max(Ev, 67) - 127; 2^(that - 24)
#pragma unroll
            for (int x = 0; x < 2 * U; ++x) {
                const uint32_t w = __shfl_sync(0xffffffffu, powers[x >> 2], (lane & ~3) | (x & 3));
                const float kf = kv_up(w & 255), counted = (w >> 16) != 0 ? 0.f : -INFINITY;
                const int at_least = max((int)((w >> 8) & 255), LEAST_POWER);
                ev[x] = (float)(at_least - 127);
                up[x] = kv_up(at_least - SUMS_UP);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) sc[n][x >> 1][2 * (x & 1) + e] = fmaf(sc[n][x >> 1][2 * (x & 1) + e] * qf[n][e], kf, counted);
            }
            if (PORTIONS && (pos0 + TOKENS - 1 > seen_by_all || p.window > 0)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int seen = limit_s[warp][8 * n + 2 * t + e], from = p.window > 0 ? seen - p.window : -1;
#pragma unroll
                        for (int x = 0; x < 2 * U; ++x) {
                            const int pos = pos0 + 8 * x + g;
                            if (pos > seen || pos <= from) sc[n][x >> 1][2 * (x & 1) + e] = -INFINITY;
                        }
                    }
            }
            uint32_t pb[NT][U][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (PORTIONS && 8 * n >= rows) continue;  // (an eight of rows that there is not)
                float keep[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = -INFINITY;
#pragma unroll
                    for (int u = 0; u < U; ++u) top = fmaxf(top, fmaxf(sc[n][u][e] + ev[2 * u], sc[n][u][2 + e] + ev[2 * u + 1]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float m_new = fmaxf(m[n][e], top), ref = m_new == -INFINITY ? 0.f : m_new - 14.f;
                    keep[e] = fast_exp2(m[n][e] - 14.f - ref);
                    m[n][e] = m_new;
                    float sum = 0.f;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float w = fast_exp2(sc[n][u][2 * r + e] - (ref - SUMS_UP));
                            sum += w;
                            sc[n][u][2 * r + e] = w * up[2 * u + r];
                        }
                    l[n][e] = fmaf(l[n][e], keep[e], sum);
                }
                if (__builtin_expect(rare, 0)) {
#pragma unroll
                    for (int x = 0; x < 2 * U; ++x) {
                        const uint32_t w = __shfl_sync(0xffffffffu, powers[x >> 2], (lane & ~3) | (x & 3));
                        const float less = kv_up(127 + min((int)((w >> 8) & 255) - LEAST_POWER, 0));
                        sc[n][x >> 1][2 * (x & 1)] *= less;
                        sc[n][x >> 1][2 * (x & 1) + 1] *= less;
                    }
                }
                if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) {
                        o[n][j][0] *= keep[0]; o[n][j][1] *= keep[1]; o[n][j][2] *= keep[0]; o[n][j][3] *= keep[1];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int r = 0; r < 2; ++r) pb[n][u][r] = transposed(half2_of(sc[n][u][2 * r], sc[n][u][2 * r + 1]));
            }
            // O^T += V^T P^T: a thread pairs tokens (2 t, 2 t + 1) and (2 t + 8, 2 t + 9); its words of a row: 16 bytes of every
            // 128, then 8 of 64 and 4 of 32
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t w[4][WORDS];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    constexpr int W16 = HD / 128;
                    // (of row 2 t + (x & 1); 8 and 16 rows further: the same swizzle)
                    const uint8_t* vr = vt + (16 * u + 8 * (x >> 1)) * HD;
                    const int r = 2 * t + (x & 1);
#pragma unroll
                    for (int j = 0; j < W16; ++j) {
                        const uint4 v = *reinterpret_cast<const uint4*>(vr + C::at(r, g) + 128 * j);
                        w[x][4 * j] = v.x; w[x][4 * j + 1] = v.y; w[x][4 * j + 2] = v.z; w[x][4 * j + 3] = v.w;
                    }
                    if (HD % 128 >= 64) {
                        const uint2 v = *reinterpret_cast<const uint2*>(vr + C::at(r, 8 * W16 + (g >> 1)) + 8 * (g & 1));
                        w[x][4 * W16] = v.x;
                        w[x][4 * W16 + 1] = v.y;
                    }
                    if (HD % 64 == 32) w[x][WORDS - 1] = *reinterpret_cast<const uint32_t*>(vr + C::at(r, HD / 16 - 2 + (g >> 2)) + 4 * (g & 3));
                }
#pragma unroll
                for (int j = 0; j < WORDS; ++j) {
                    uint32_t even[4], odd[4];
                    halves_of(__byte_perm(w[0][j], w[1][j], 0x5140), even[0], even[1]);
                    halves_of(__byte_perm(w[0][j], w[1][j], 0x7362), odd[0], odd[1]);
                    halves_of(__byte_perm(w[2][j], w[3][j], 0x5140), even[2], even[3]);
                    halves_of(__byte_perm(w[2][j], w[3][j], 0x7362), odd[2], odd[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (PORTIONS && 8 * n >= rows) continue;
                        mma_half(o[n][2 * j], even, pb[n][u][0], pb[n][u][1]);
                        mma_half(o[n][2 * j + 1], odd, pb[n][u][0], pb[n][u][1]);
                    }
                }
            }
            __syncwarp();  // the stage is free
        }
        // ---- the run has left the segment, or ends in it ----
        const bool begins = at.tile == 0, ends = at.tile + n_tiles == at.tiles;
        const int piece = 2 * warp + (ends ? 0 : 1);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (!(begins && ends) && g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m_s[piece][8 * n + 2 * t + e] = m[n][e];
                    l_s[piece][8 * n + 2 * t + e] = l[n][e];
                }
            if (lane == 0) {
                const int first_block = (seg_unit + 1) / block_units;
                piece_s[piece] = {seg_unit | team << 29, row, head, x0, rows, team, first_block,
                                  (seg_unit + at.tiles) / block_units - first_block + 1};
            }
        }
        if (!ends) cp_async_wait<0>();  // (nothing is in flight any more: the run is over)
        __syncwarp();
        float* sums = ends ? p.heads_o + (size_t)(blockIdx.x * WARPS + warp) * ROWS * HD : reinterpret_cast<float*>(my_ring);
        static_assert(ROWS * HD * 4 <= C::RING / WARPS, "a piece must fit over a warp's ring");
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                const int d = j < HD / 128 * 4 ? (j / 4) * 128 + 16 * g + 4 * (j % 4)
                              : (HD % 128 >= 64 && j < HD / 128 * 4 + 2) ? HD / 128 * 128 + 8 * g + 4 * (j - HD / 128 * 4) : HD - 32 + 4 * g;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = 8 * n + 2 * t + e;
                    const float4 x = make_float4(o[n][2 * j][e], o[n][2 * j][2 + e], o[n][2 * j + 1][e], o[n][2 * j + 1][2 + e]);
                    if (begins && ends) {
                        const float inv = l[n][e] == 0.f ? 0.f : (float)(1 << SUMS_UP) / l[n][e];
                        if (r < rows)
                            Vec4<bf16>::store((bf16*)p.out + row_at(row, head, x0 + r, p.nh * HD) + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
                    } else {
                        *reinterpret_cast<float4*>(sums + r * HD + d) = x;
                    }
                }
            }
        if (ends) seg_unit += at.tiles + 1;
        step(at, n_tiles);
    }
    cp_async_wait<0>();
    __syncthreads();
    // ---- the block's pieces, in order: those of one segment, which are neighbours, are added up ----
    const int segment_of_lane = lane < 2 * WARPS ? piece_s[lane].segment : -2 - lane;
    const uint32_t alike = __match_any_sync(0xffffffffu, segment_of_lane);
    const uint32_t leads = __ballot_sync(0xffffffffu, segment_of_lane >= 0 && (alike & ((1u << lane) - 1)) == 0);
    for (int i = tid; i < 2 * WARPS * ROWS; i += blockDim.x) {  // what each piece is multiplied by; the sum of weights at the group's first
        const int x = i / ROWS, r = i % ROWS;
        const uint32_t group = __shfl_sync(0xffffffffu, alike, x);
        float m[2 * WARPS], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int y = 0; y < 2 * WARPS; ++y) {
            m[y] = (group >> y) & 1 ? m_s[y][r] : -INFINITY;
            top = fmaxf(top, m[y]);
        }
#pragma unroll
        for (int y = 0; y < 2 * WARPS; ++y)
            if (m[y] != -INFINITY) sum = fmaf(fast_exp2(m[y] - top), l_s[y][r], sum);
        const float own = m_s[x][r];
        f_s[x][r] = own == -INFINITY ? 0.f : fast_exp2(own - top);
        top_s[x][r] = top;
        total_s[x][r] = sum;
    }
    __syncthreads();
    // the first pieces of segments that other blocks have pieces of as well: of every team one that came from before, one that goes on
    if (tid < 2 * MOST_TEAMS) shared_s[tid] = -1;
    __syncthreads();
#pragma unroll 1
    for (uint32_t todo = leads; todo != 0; todo &= todo - 1) {
        const int x = __ffs(todo) - 1;
        const uint32_t group = __shfl_sync(0xffffffffu, alike, x);
        const int head = __ffs(group & 0x55) - 1;  // the one piece, if any, that lies in global memory
        const Piece& s = piece_s[x];
        const bool whole = s.blocks == 1, begins_here = blockIdx.x == s.first_block;
        const size_t piece = (size_t)2 * (blockIdx.x * teams + s.team) + begins_here;
        if (!whole && tid == 0) shared_s[2 * s.team + begins_here] = x;
        float* part = p.part_o + piece * ROWS * HD;
        const int items = s.rows * (HD / 4);
#pragma unroll 1
        for (int i0 = tid; i0 < items; i0 += 2 * WARPS * 32) {  // four outputs each, two such at a time: all loads before their use
            float4 v[2][WARPS + 1];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = i0 + e * WARPS * 32;
                v[e][WARPS] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (head >= 0 && i < items) v[e][WARPS] = *reinterpret_cast<const float4*>(p.heads_o + (size_t)(blockIdx.x * WARPS + (head >> 1)) * ROWS * HD + i * 4);
#pragma unroll
                for (int w = 0; w < WARPS; ++w)
                    v[e][w] = i < items && (group >> (2 * w + 1)) & 1 ? *reinterpret_cast<const float4*>(ring_s + w * ST * 2 * C::TILE_BYTES + i * 16)
                                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = i0 + e * WARPS * 32, r = i / (HD / 4);
                if (i >= items) break;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w <= WARPS; ++w) {
                    const float f = w < WARPS ? ((group >> (2 * w + 1)) & 1 ? f_s[2 * w + 1][r] : 0.f) : head >= 0 ? f_s[head][r] : 0.f;
                    sum.x = fmaf(f, v[e][w].x, sum.x); sum.y = fmaf(f, v[e][w].y, sum.y); sum.z = fmaf(f, v[e][w].z, sum.z); sum.w = fmaf(f, v[e][w].w, sum.w);
                }
                const float total = total_s[x][r];
                if (whole) {
                    const float inv = total == 0.f ? 0.f : (float)(1 << SUMS_UP) / total;
                    Vec4<bf16>::store((bf16*)p.out + row_at(s.row, s.head, s.first + r, p.nh * HD) + i % (HD / 4) * 4, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
                } else {
                    *reinterpret_cast<float4*>(part + i * 4) = sum;
                    if (i % (HD / 4) == 0) *reinterpret_cast<float2*>(p.part_ml + (piece * ROWS + r) * 2) = make_float2(top_s[x][r], total);
                }
            }
        }
    }
    zeros();
    // ---- segments that other blocks have pieces of: thread e counts this block in at its counter ----
    // (pieces by number: y is of block first_block + y, its second one where the segment begins in it)
    auto by_eights = [&](const Piece& s) { return s.blocks > 3 * MERGE_AT_ONCE; };  // added up by eights first
    auto place = [&](const Piece& s, int y) { return (size_t)2 * ((s.first_block + y) * teams + s.team) + (y == 0 ? 1 : 0); };
    // the barrier orders all threads' stores before the release; the last block's acquire, followed by the next barrier, its
    // threads' loads behind everybody's stores
    auto count_in = [&](int* counter, int count) {
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
        if (before == count - 1) *counter = 0;
        return before == count - 1;
    };
    __syncthreads();
    if (tid < 2 * teams) {
        const int x = shared_s[tid];
        bool is_last = false;
        if (x >= 0) {
            const Piece& s = piece_s[x];
            const int y = blockIdx.x - s.first_block, from = y - y % MERGE_AT_ONCE;
            if (by_eights(s))
                is_last = count_in(p.counters + gridDim.x * MOST_TEAMS + place(s, from), min(MERGE_AT_ONCE, s.blocks - from));
            else
                is_last = count_in(p.counters + s.first_block * teams + s.team, s.blocks);
        }
        last_s[tid] = is_last;
    }
    __syncthreads();
#pragma unroll 1
    for (int e = 0; e < 2 * teams; ++e) {
        if (!last_s[e]) continue;
        const Piece s = piece_s[shared_s[e]];
        const int y = blockIdx.x - s.first_block;
        bool final = !by_eights(s);
        int from = final ? 0 : y - y % MERGE_AT_ONCE, count = final ? s.blocks : min(MERGE_AT_ONCE, s.blocks - from), stride = 1;
#pragma unroll 1
        for (;;) {
            const int items = s.rows * (HD / 4);
#pragma unroll 1
            for (int i0 = tid; i0 < items; i0 += 2 * WARPS * 32) {  // two at a time, eight pieces of each: one trip to the L2
                float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f};
                float4 sum[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 1
                for (int y0 = 0; y0 < count; y0 += MERGE_AT_ONCE) {
                    float2 ml[2][MERGE_AT_ONCE];
                    float4 v[2][MERGE_AT_ONCE];
                    // (in units of a piece's rows; the segment's very first piece lies one further)
                    size_t at_piece = (size_t)2 * ((s.first_block + from + y0 * stride) * teams + s.team);
#pragma unroll
                    for (int k = 0; k < MERGE_AT_ONCE; ++k) {
                        const size_t here = (at_piece + (k == 0 && from + y0 == 0 ? 1 : 0)) * ROWS;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int i = i0 + e * WARPS * 32;
                            ml[e][k] = make_float2(-INFINITY, 0.f);
                            v[e][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (y0 + k < count && i < items) {
                                ml[e][k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + here + i / (HD / 4));
                                v[e][k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + here * HD) + i);
                            }
                        }
                        at_piece += 2 * teams * stride;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float next = top[e];
#pragma unroll
                        for (int k = 0; k < MERGE_AT_ONCE; ++k) next = fmaxf(next, ml[e][k].x);
                        const float keep = top[e] == -INFINITY ? 0.f : fast_exp2(top[e] - next);
                        total[e] *= keep; sum[e].x *= keep; sum[e].y *= keep; sum[e].z *= keep; sum[e].w *= keep;
                        top[e] = next;
#pragma unroll
                        for (int k = 0; k < MERGE_AT_ONCE; ++k) {
                            const float f = ml[e][k].x == -INFINITY ? 0.f : fast_exp2(ml[e][k].x - next);
                            total[e] = fmaf(f, ml[e][k].y, total[e]);
                            sum[e].x = fmaf(f, v[e][k].x, sum[e].x); sum[e].y = fmaf(f, v[e][k].y, sum[e].y);
                            sum[e].z = fmaf(f, v[e][k].z, sum[e].z); sum[e].w = fmaf(f, v[e][k].w, sum[e].w);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int i = i0 + e * WARPS * 32;
                    if (i >= items) break;
                    if (final) {
                        const float inv = total[e] == 0.f ? 0.f : (float)(1 << SUMS_UP) / total[e];
                        Vec4<bf16>::store((bf16*)p.out + row_at(s.row, s.head, s.first + i / (HD / 4), p.nh * HD) + i % (HD / 4) * 4,
                                          make_float4(sum[e].x * inv, sum[e].y * inv, sum[e].z * inv, sum[e].w * inv));
                    } else {  // over the first of the eight, whose four sums this thread alone reads and writes
                        *reinterpret_cast<float4*>(p.part_o + place(s, from) * ROWS * HD + i * 4) = sum[e];
                        if (i % (HD / 4) == 0) {
                            top_s[0][i / (HD / 4)] = top[e];
                            total_s[0][i / (HD / 4)] = total[e];
                        }
                    }
                }
            }
            __syncthreads();  // (maxima and sums of the pieces are read by all; top_s and total_s are free)
            if (final) break;
            if (tid < s.rows) *reinterpret_cast<float2*>(p.part_ml + (place(s, from) * ROWS + tid) * 2) = make_float2(top_s[0][tid], total_s[0][tid]);
            from = 0;
            count = (s.blocks + MERGE_AT_ONCE - 1) / MERGE_AT_ONCE;
            stride = MERGE_AT_ONCE;
            final = true;
            __syncthreads();
            if (tid == 0) final_s = count_in(p.counters + s.first_block * teams + s.team, count);
            __syncthreads();
            if (final_s == 0) break;
        }
    }
    cw_trace_end();
}

#define ANY_TOKENS 128
// Any head size and both types of a run: a block per (request, query head), 128 tokens at a time, first a token per thread for
// the scores, then entries per thread for the values.
template <typename T>
__global__ void __launch_bounds__(ANY_TOKENS) decode_e4m3_any_kernel(const DecodeE4m3Params p) {
    __shared__ float q_s[256], w_s[ANY_TOKENS], scratch[33];
    __shared__ int slot_s[ANY_TOKENS];
    pdl_enter();
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, kvh = h / (p.nh / p.nkv);
    int row = s;
    if (p.q_start != nullptr) {
        row = p.q_start[s];
        if (p.q_start[s + 1] - row != 1) return;
    }
    const int ctx = min(p.ctx_lens[s], p.max_blocks * p.page_size), begin = p.window > 0 ? max(0, ctx - p.window) : 0;
    const T* q = (const T*)p.q + (size_t)row * p.q_stride + (size_t)h * p.hd;
    for (int d = tid; d < p.hd; d += ANY_TOKENS) q_s[d] = to_f(q[d]) * p.scale * 1.4426950408889634f;  // (2^x below)
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};  // entries tid and tid + 128
    for (int j0 = begin; j0 < ctx; j0 += ANY_TOKENS) {
        const int j = j0 + tid;
        float sc = -INFINITY, up = 0.f;
        int slot = -1;
        if (j < ctx) {
            const int page = p.block_tables[(size_t)s * p.max_blocks + j / p.page_size], off = j % p.page_size;
            if (page < 0 || page >= p.num_pages) {
                cw_report(p.status, CW_ST_PAGE_RANGE, s, page);
            } else {
                slot = page * p.page_size + off;
                const uint4* k = reinterpret_cast<const uint4*>(p.k + ((size_t)slot * p.nkv + kvh) * p.hd);
                float dot = 0.f;
                for (int c = 0; c < p.hd / 16; ++c) {
                    const uint4 raw = k[c];
                    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 lo = kv_float2(w[i]), hi = kv_float2(w[i] >> 16);
                        const float* x = q_s + 16 * c + 4 * i;
                        dot = fmaf(x[0], lo.x, fmaf(x[1], lo.y, fmaf(x[2], hi.x, fmaf(x[3], hi.y, dot))));
                    }
                }
                const size_t at = ((size_t)page * p.nkv + kvh) * p.page_size + off;
                sc = dot * kv_up(p.k_exp[at]);
                up = kv_up(p.v_exp[at]);
            }
        }
        const float m_new = fmaxf(m, block_max(sc, scratch));
        const float keep = m == -INFINITY ? 0.f : exp2f(m - m_new), w = sc == -INFINITY ? 0.f : exp2f(sc - m_new);
        l = l * keep + block_sum(w, scratch);
        m = m_new;
        w_s[tid] = w * up;
        slot_s[tid] = slot;
        __syncthreads();
        const int n = min(ANY_TOKENS, ctx - j0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = tid + e * ANY_TOKENS;
            if (d < p.hd) {
                float a = acc[e] * keep;
                for (int i = 0; i < n; ++i) {
                    if (slot_s[i] < 0) continue;
                    const uint32_t code = p.v[((size_t)slot_s[i] * p.nkv + kvh) * p.hd + d];
                    a = fmaf(w_s[i], kv_float2(code).x, a);
                }
                acc[e] = a;
            }
        }
        __syncthreads();
    }
    T* out = (T*)p.out + ((size_t)row * p.nh + h) * p.hd;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (tid + e * ANY_TOKENS < p.hd) out[tid + e * ANY_TOKENS] = from_f<T>(l > 0.f ? acc[e] / l : (l == l ? 0.f : l));
}

template <int HD, int NT, bool PORTIONS>
static int stream_launch(const DecodeE4m3Params& p, int sms, cudaStream_t stream) {
    using C = Stream<HD, NT>;
    static bool configured[64] = {};  // (per device)
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= 64 || !configured[device]) {
        const cudaError_t e = cudaFuncSetAttribute(decode_e4m3_kernel<HD, NT, PORTIONS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::RING);
        if (e != cudaSuccess) return (int)e;
        if (device >= 0 && device < 64) configured[device] = true;
    }
    return cw_launch(decode_e4m3_kernel<HD, NT, PORTIONS>, dim3(sms * C::PER_SM), dim3(WARPS * 32), C::RING, stream, 1u, p);
}
template <int HD>
static int stream_launch_heads(const DecodeE4m3Params& p, int sms, cudaStream_t stream) {
    if (p.heads_each <= 8) return stream_launch<HD, 1, false>(p, sms, stream);
    return stream_launch<(HD <= 128 ? HD : 32), 2, false>(p, sms, stream);  // (head sizes beyond 128 come in groups of 8)
}

// How a KV head's query heads are shared out: groups of 16 at most, of 8 where heads are so large that the sums of 16 would not
// stay in registers; 0: the streaming kernel does not take the head size or the type.
static int groups_of(int nh, int nkv, int hd, int dtype) {
    if (dtype != 1 || hd % 32) return 0;
    const int each = nh / nkv, most = hd <= 128 ? 16 : 8;
    return (each + most - 1) / most;
}

// Scratch of the calls: float32 words, and zeroed int32 words (which are zero again when a call has run).  It goes by the GPU and the
// head size alone: two pieces per block and team, the ends of segments per warp; 16 rows of three blocks an SM with four teams.
#define SCRATCH_PIECES(sms) (6LL * (sms) * MOST_TEAMS)
extern "C" int cw_attention_e4m3_scratch(int hd, int sms, long long* floats, int* words) {
    if (hd <= 0 || hd > 256 || sms <= 0) return CW_ERR_BAD_SIZE;
    *floats = SCRATCH_PIECES(sms) * 16 * (hd + 2) + 12LL * sms * 16 * hd;
    *words = (int)(3 * sms * MOST_TEAMS + SCRATCH_PIECES(sms));
    return CW_OK;
}

static bool streams(DecodeE4m3Params& p, long long groups, int sms, float* floats, int* words) {
    const long long slots = (long long)p.num_pages * p.page_size, tiles = (long long)p.max_blocks * p.page_size / 16 + 2;
    if (floats == nullptr || words == nullptr || (uintptr_t)p.q % 4 || p.q_stride % 2) return false;  // (queries are read in pairs)
    if (slots * p.nkv * (p.hd / 16) >= 0xFFFFFFFFLL || p.nkv * groups * tiles >= 1LL << 29) return false;
    p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
    p.part_o = floats;
    p.part_ml = p.part_o + SCRATCH_PIECES(sms) * 16 * p.hd;
    p.heads_o = p.part_ml + SCRATCH_PIECES(sms) * 16 * 2;
    p.counters = words;
    return true;
}

// q [rows, q_stride >= nh * hd], out [rows, nh * hd]; request s owns row s, or with q_start rows q_start[s] .. q_start[s + 1], and
// then only requests with one row are served.  A context of length 0 gives zeros.  `floats`, `words`: the scratch.
extern "C" int cw_attention_decode_e4m3(const char* block) {
    ArgumentWords w(block);
    const void* q = w.pointer(); void* out = w.pointer();
    const uint8_t *k = (const uint8_t*)w.pointer(), *v = (const uint8_t*)w.pointer(), *k_exp = (const uint8_t*)w.pointer(), *v_exp = (const uint8_t*)w.pointer();
    const int *block_tables = (const int*)w.pointer(), *ctx_lens = (const int*)w.pointer(), *q_start = (const int*)w.pointer();
    float* floats = (float*)w.pointer();
    int *words = (int*)w.pointer(), *status = (int*)w.pointer();
    const cudaStream_t stream = (cudaStream_t)w.pointer();
    const int q_stride = w.number(), requests = w.number(), nh = w.number(), nkv = w.number(), hd = w.number(), page_size = w.number(),
              max_blocks = w.number(), num_pages = w.number(), window = w.number(), dtype = w.number(), sms = w.number(),
              early = w.number();
    const float scale = (float)w.real();
    if (requests == 0) return CW_OK;
    if (requests < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || hd % 16 || hd > 256 || page_size <= 0 || max_blocks <= 0 ||
        num_pages <= 0 || window < 0 || q_stride < nh * hd || ((uintptr_t)k | (uintptr_t)v) % 16 || requests > 65535 || sms <= 0 ||
        (long long)num_pages * page_size > 0x7FFFFFFF || (long long)max_blocks * page_size > 0x7FFFFFFF)
        return CW_ERR_BAD_SIZE;
    DecodeE4m3Params p = {q, q_stride, out, k, v, k_exp, v_exp, block_tables, ctx_lens, q_start, requests, nh, nkv, hd, page_size,
                          max_blocks, num_pages, window, scale, status};
    p.early = early;
    const int groups = groups_of(nh, nkv, hd, dtype);
    if (groups && streams(p, (long long)requests * groups, sms, floats, words)) {
        p.groups = groups;
        p.heads_each = (nh / nkv + groups - 1) / groups;
        p.teams = hd == 32 && nkv % 4 == 0 ? 4 : hd < 128 && nkv % 2 == 0 ? 2 : 1;
        switch (hd) {
            case 32: return stream_launch_heads<32>(p, sms, stream);
            case 64: return stream_launch_heads<64>(p, sms, stream);
            case 96: return stream_launch_heads<96>(p, sms, stream);
            case 128: return stream_launch_heads<128>(p, sms, stream);
            case 160: return stream_launch_heads<160>(p, sms, stream);
            case 192: return stream_launch_heads<192>(p, sms, stream);
            case 224: return stream_launch_heads<224>(p, sms, stream);
            case 256: return stream_launch_heads<256>(p, sms, stream);
        }
    }
    if (dtype == 0) return cw_launch(decode_e4m3_any_kernel<float>, dim3(nh, requests), dim3(ANY_TOKENS), 0, stream, 1u, p);
    if (dtype == 1) return cw_launch(decode_e4m3_any_kernel<bf16>, dim3(nh, requests), dim3(ANY_TOKENS), 0, stream, 1u, p);
    return CW_ERR_BAD_DTYPE;
}

// Causal attention of the portions of requests that bring `least_rows` to `most_rows` rows, q_start[s] .. q_start[s + 1] of q and out
// (other rows are left alone), the last of the ctx_lens[s] tokens that each has in the cache; `rows`: the most rows that all of them
// bring together.  bfloat16, head sizes 32, 64, 96 and 128.
extern "C" int cw_attention_portions_e4m3(const char* block) {
    ArgumentWords w(block);
    const void* q = w.pointer(); void* out = w.pointer();
    const uint8_t *k = (const uint8_t*)w.pointer(), *v = (const uint8_t*)w.pointer(), *k_exp = (const uint8_t*)w.pointer(), *v_exp = (const uint8_t*)w.pointer();
    const int *block_tables = (const int*)w.pointer(), *ctx_lens = (const int*)w.pointer(), *q_start = (const int*)w.pointer();
    float* floats = (float*)w.pointer();
    int *words = (int*)w.pointer(), *status = (int*)w.pointer();
    const cudaStream_t stream = (cudaStream_t)w.pointer();
    const int q_stride = w.number(), requests = w.number(), nh = w.number(), nkv = w.number(), hd = w.number(), page_size = w.number(),
              max_blocks = w.number(), num_pages = w.number(), window = w.number(), sms = w.number(), rows = w.number(), least_rows = w.number(),
              most_rows = w.number();
    const float scale = (float)w.real();
    if (requests == 0 || rows == 0) return CW_OK;
    if (requests < 0 || nh <= 0 || nkv <= 0 || nh % nkv || page_size <= 0 || max_blocks <= 0 || num_pages <= 0 || window < 0 ||
        q_stride < nh * hd || ((uintptr_t)k | (uintptr_t)v) % 16 || sms <= 0 || rows < 0 || least_rows < 1 || most_rows < least_rows ||
        q_start == nullptr || (long long)num_pages * page_size > 0x7FFFFFFF || (long long)max_blocks * page_size > 0x7FFFFFFF)
        return CW_ERR_BAD_SIZE;
    DecodeE4m3Params p = {q, q_stride, out, k, v, k_exp, v_exp, block_tables, ctx_lens, q_start, requests, nh, nkv, hd, page_size,
                          max_blocks, num_pages, window, scale, status};
    p.groups = p.teams = 1;
    p.least_rows = least_rows;
    p.most_rows = most_rows;
    if (!streams(p, (long long)rows * (nh / nkv) / 16 + requests, sms, floats, words)) return CW_ERR_UNSUPPORTED;
    switch (hd) {
        case 32: return stream_launch<32, 2, true>(p, sms, stream);
        case 64: return stream_launch<64, 2, true>(p, sms, stream);
        case 96: return stream_launch<96, 2, true>(p, sms, stream);
        case 128: return stream_launch<128, 2, true>(p, sms, stream);
    }
    return CW_ERR_UNSUPPORTED;
}

CW_TRACE_TU(attention_decode_e4m3)
