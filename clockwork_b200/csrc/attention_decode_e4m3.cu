// Attention of one new token per request over an 8-bit cache (kv_e4m3.cuh), through block tables.
//
//     s_j = scale * 2^(Ek_j - 127) * sum_d q_d kcode_jd,   out = sum_j e^(s_j - m) 2^(Ev_j - 127) vcode_j / sum_j e^(s_j - m)
//
// over the context's positions j (the last `window` of them), m their largest s_j; float32 but for what is said below.
//
// The step is a stream of codes from memory, 2 (hd + 1) bytes per token and KV head, so all query heads of a KV head (16 at
// most, or 8) share what a block fetches.  Work is cut by the contexts themselves: requests, KV heads and tiles of 32 tokens
// are numbered through, and every block of a grid that fills the SMs once takes an equal run of tiles, wherever requests begin
// and end in it (units_of_block); so contexts of any lengths fill the GPU, and no scratch grows with them.  A run's tiles go to
// four warps in turn.  Each warp has a ring of tiles in shared memory of its own, filled by 16-byte asynchronous copies two or
// more tiles ahead, so that warps never wait for one another while they stream.
//
// Codes become half-precision numbers exactly (cvt) on their way into mma.sync.m16n8k16, which costs less here than it could
// save elsewhere: at the rate of memory the tensor cores are a fifth busy.  Tokens are the M side of S^T = K Q^T and the codes'
// entries the M side of O^T = V^T P^T, so that eight query heads (N) fill what sixteen would, and a thread's 16 bytes of K are
// four k-steps of one product: which entries a k-step takes is the same for K and Q and otherwise free.  For V^T P^T two tokens'
// bytes are paired by a byte permutation before cvt.  S^T's accumulators become P^T's fragments by movmatrix.
//
// Query heads are scaled by a power of two each into half precision's upper range (bfloat16's 8 bits are kept; what falls below
// 2^-39 of the head's largest entry is dropped).  The powers of K multiply scores in float32.  Those of V are taken into
// the exponent: weights are p_j = 2^(s_j log2 e + Ev_j - 127 - M + 14), M the running maximum of s_j log2 e + Ev_j - 127, in half precision
// (11 bits, off by at most 2^-12 of themselves, or by 2^-39 of the largest contribution), and the denominator, float32, sums
// p_j 2^(127 - Ev_j).  (It overflows, and the result is 0, where a context's values are all below 2^-88.)
//
// A segment (request, KV head) that lies in one block's run is finished there; the pieces of one that several blocks share go
// to scratch of two pieces per block, and the block that comes last merges them in the blocks' order (more than 24: twelve at a time
// first, each by the last of the twelve).  The result does not depend on who comes last.
#include "attention_mma.cuh"
#include "kv_e4m3.cuh"

struct DecodeE4m3Params {
    const void* q; int q_stride; void* out;
    const uint8_t* k; const uint8_t* v; const uint8_t* k_exp; const uint8_t* v_exp;
    const int* block_tables; const int* ctx_lens; const int* q_start;
    int requests, nh, nkv, hd, page_size, max_blocks, num_pages, window;
    float scale;
    int* status;
    // the streaming kernel
    int page_shift;          // log2 of the page size, or -1
    int groups, heads_each;  // groups of query heads per KV head, heads in a group (the last may have fewer)
    float* part_o;           // [2 * blocks][heads of a group][hd]
    float* part_ml;          // [2 * blocks][heads of a group][2]
    int* counters;           // [requests * nkv * groups] and [2 * blocks], zero between launches
};

#define TILE_TOKENS 32
#define WARPS 4
#define MERGE_AT_ONCE 12

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

template <int HD>
struct Stream {
    static constexpr int CH = HD / 16;                 // 16-byte chunks of a row
    static constexpr int TILE_BYTES = TILE_TOKENS * HD;  // K or V of a tile
    static constexpr int PER_SM = HD <= 128 ? 2 : 1;   // blocks on an SM
    static constexpr int FIT = (PER_SM == 2 ? 98304 : 196608) / (WARPS * 2 * TILE_BYTES);
    static constexpr int ST = FIT > 8 ? 8 : FIT;       // tiles in a warp's ring
    static constexpr int RING = WARPS * ST * 2 * TILE_BYTES;
    // Where chunk c of row r lies.  Rows of 128 bytes and multiples are swizzled so that the reads below (K: two rows' four chunks
    // at a time; V: a chunk of four rows two apart) meet no bank twice; of 64 bytes: the same over lines of two rows.
    static __device__ __forceinline__ int at(int r, int c) {
        if (HD % 128 == 0) return r * HD + ((c ^ ((((r >> 1) & 3) << 1) ^ ((r & 1) << 2))) << 4);
        if (HD == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
        return r * HD + (c << 4);
    }
};

template <int HD, int NT>
__global__ void __launch_bounds__(WARPS * 32, Stream<HD>::PER_SM) decode_e4m3_kernel(const DecodeE4m3Params p) {
    using C = Stream<HD>;
    constexpr int ROWS = 8 * NT, ST = C::ST;
    constexpr int WORDS = HD / 32;  // a thread's 4-byte words of a V row
    extern __shared__ __align__(128) uint8_t ring_s[];
    __shared__ __align__(16) __half q_s[ROWS][HD + 8];
    __shared__ float qf_s[ROWS];
    __shared__ int slot_s[WARPS][ST][TILE_TOKENS];
    __shared__ uint32_t power_at_s[WARPS][ST][TILE_TOKENS];
    __shared__ float m_s[WARPS][ROWS], l_s[WARPS][ROWS], w_s[ROWS][WARPS + 2];
    __shared__ int sh[36];
    __shared__ int last_s;
    pdl_enter();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int per_request = p.nkv * p.groups;
    auto context_of = [&](int s) -> int {  // -1: not served here
        if (p.q_start != nullptr && p.q_start[s + 1] - p.q_start[s] != 1) return -1;
        return min(p.ctx_lens[s], p.max_blocks * p.page_size);
    };
    auto begin_of = [&](int ctx) { return p.window > 0 ? max(0, ctx - p.window) : 0; };
    auto tiles_of = [&](int ctx) {
        return ctx <= 0 ? 0 : (ctx + TILE_TOKENS - 1) / TILE_TOKENS - begin_of(ctx) / TILE_TOKENS;
    };
    const UnitRange range =
        units_of_block([&](int s) { return per_request * tiles_of(context_of(s)); }, p.requests, WARPS, gridDim.x, blockIdx.x, sh);
    for (int s = blockIdx.x; s < p.requests; s += gridDim.x) {  // rows without a context: zeros
        if (context_of(s) != 0) continue;
        const int row = p.q_start != nullptr ? p.q_start[s] : s;
        for (int i = tid; i < p.nh * HD; i += blockDim.x) ((bf16*)p.out)[(size_t)row * p.nh * HD + i] = __float2bfloat16_rn(0.f);
    }
    uint8_t* my_ring = ring_s + warp * ST * 2 * C::TILE_BYTES;
    const uint32_t my_ring_addr = smem_addr(my_ring);
    int s = range.request, offset = range.offset;
    for (int unit = range.first; unit < range.last; ++s, offset = 0) {
        const int ctx = context_of(s), tiles = tiles_of(ctx);
        if (tiles <= 0) continue;
        const int begin = begin_of(ctx), tile_base = begin / TILE_TOKENS;
        const int row = p.q_start != nullptr ? p.q_start[s] : s;
        const int* table = p.block_tables + (size_t)s * p.max_blocks;
        for (int seg = offset / tiles; seg < per_request && unit < range.last; ++seg) {
            const int seg_first = unit - (offset - seg * tiles);  // the segment's first unit
            const int ta = offset - seg * tiles, tb = min(tiles, ta + range.last - unit);
            const int kvh = seg / p.groups, h0 = kvh * (p.nh / p.nkv) + (seg % p.groups) * p.heads_each;
            const int rows = min(p.heads_each, p.nh / p.nkv - (seg % p.groups) * p.heads_each);
            unit += tb - ta;
            offset = (seg + 1) * tiles;
            // ---- the group's queries in half precision, a power of two out of each ----
            for (int r = warp; r < ROWS; r += WARPS) {
                constexpr int E = HD / 32;
                float x[E], big = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    x[e] = r < rows ? __bfloat162float(((const bf16*)p.q)[(size_t)row * p.q_stride + (size_t)(h0 + r) * HD + e * 32 + lane]) : 0.f;
                    big = fmaxf(big, fabsf(x[e]));
                }
                big = warp_max(big);
                const int sh_q = big > 0.f ? min(126, 14 - (int)((__float_as_uint(big) >> 23) & 255) + 127) : 0;
#pragma unroll
                for (int e = 0; e < E; ++e) q_s[r][e * 32 + lane] = __float2half_rn(ldexpf(x[e], sh_q));
                if (lane == 0) qf_s[r] = ldexpf(p.scale * 1.4426950408889634f, -sh_q);
            }
            __syncthreads();
            // k-steps of K's 16-byte (or, in rows that are no multiple of 64, 8-byte) pieces: B fragments of the same entries
            constexpr int PIECE = HD % 64 == 0 ? 16 : 8, STEPS = PIECE / 4, PIECES = HD / (4 * PIECE);
            uint32_t qb[NT][PIECES][STEPS][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < PIECES; ++b)
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        const uint2 w = *reinterpret_cast<const uint2*>(&q_s[8 * n + g][b * 4 * PIECE + t * PIECE + 4 * i]);
                        qb[n][b][i][0] = w.x;
                        qb[n][b][i][1] = w.y;
                    }
            float qf[NT][2], m[NT][2], l[NT][2], o[NT][HD / 16][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    qf[n][e] = qf_s[8 * n + 2 * t + e];
                    m[n][e] = -INFINITY;
                    l[n][e] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < HD / 16; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
            }
            // ---- this warp's tiles ----
            const int mine = tb - ta > warp ? (tb - ta - warp + WARPS - 1) / WARPS : 0;
            auto position = [&](int i) { return (tile_base + ta + warp + i * WARPS) * TILE_TOKENS + lane; };
            auto page_of = [&](int i) -> int {  // of this lane's token of tile i
                const int pos = position(i);
                if (i >= mine || pos < begin || pos >= ctx) return -1;
                return table[p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size];
            };
            auto fetch = [&](int i, int page) {
                if (i < mine) {
                    const int stage = i % ST, pos = position(i);
                    int slot = -1;
                    uint32_t power_at = 0;
                    if (page >= 0 && page < p.num_pages) {
                        const int off = p.page_shift >= 0 ? pos & (p.page_size - 1) : pos % p.page_size;
                        slot = page * p.page_size + off;
                        power_at = ((uint32_t)page * p.nkv + kvh) * p.page_size + off;
                    } else if (pos >= begin && pos < ctx) {
                        cw_report(p.status, CW_ST_PAGE_RANGE, s, page);
                    }
                    slot_s[warp][stage][lane] = slot;
                    power_at_s[warp][stage][lane] = power_at;
                    __syncwarp();
                    const uint32_t base = my_ring_addr + stage * 2 * C::TILE_BYTES;
#pragma unroll
                    for (int j = 0; j < C::CH; ++j) {
                        const int idx = j * 32 + lane, r = idx / C::CH, c = idx % C::CH;
                        const int sl = slot_s[warp][stage][r];
                        const size_t src = ((size_t)max(sl, 0) * p.nkv + kvh) * HD + c * 16;
                        copy16(base + C::at(r, c), p.k + src, sl >= 0);
                        copy16(base + C::TILE_BYTES + C::at(r, c), p.v + src, sl >= 0);
                    }
                }
                cp_async_commit();
            };
            // a lane holds the powers of token 8 t + g: K's, V's, and whether the token counts
            auto powers_of = [&](int i) -> uint32_t {
                if (i >= mine) return 0;
                const int token = 8 * t + g, stage = i % ST;
                if (slot_s[warp][stage][token] < 0) return 0;
                const uint32_t at = power_at_s[warp][stage][token];
                return (uint32_t)p.k_exp[at] | (uint32_t)p.v_exp[at] << 8 | 1u << 16;
            };
            for (int i = 0; i < ST - 1; ++i) fetch(i, page_of(i));
            int page_ahead = page_of(ST - 1);
            __syncwarp();
            uint32_t powers = powers_of(0);
            for (int i = 0; i < mine; ++i) {
                fetch(i + ST - 1, page_ahead);
                page_ahead = page_of(i + ST);
                cp_async_wait<ST - 1>();
                __syncwarp();
                const uint32_t powers_next = powers_of(i + 1);
                const uint8_t* kt = my_ring + (i % ST) * 2 * C::TILE_BYTES;
                const uint8_t* vt = kt + C::TILE_BYTES;
                float sc[NT][2][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u) sc[n][u][0] = sc[n][u][1] = sc[n][u][2] = sc[n][u][3] = 0.f;
#pragma unroll
                for (int b = 0; b < PIECES; ++b)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t lo[STEPS], hi[STEPS];  // rows g and g + 8
                        if (PIECE == 16) {
                            const uint4 x = *reinterpret_cast<const uint4*>(kt + C::at(16 * u + g, 4 * b + t));
                            const uint4 y = *reinterpret_cast<const uint4*>(kt + C::at(16 * u + 8 + g, 4 * b + t));
                            lo[0] = x.x; lo[1] = x.y; lo[STEPS - 2] = x.z; lo[STEPS - 1] = x.w;
                            hi[0] = y.x; hi[1] = y.y; hi[STEPS - 2] = y.z; hi[STEPS - 1] = y.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2*>(kt + C::at(16 * u + g, 2 * b + (t >> 1)) + 8 * (t & 1));
                            const uint2 y = *reinterpret_cast<const uint2*>(kt + C::at(16 * u + 8 + g, 2 * b + (t >> 1)) + 8 * (t & 1));
                            lo[0] = x.x; lo[1] = x.y;
                            hi[0] = y.x; hi[1] = y.y;
                        }
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) {
                            const uint32_t a[4] = {kv_half2(lo[k] & 0xFFFF), kv_half2(hi[k] & 0xFFFF), kv_half2(lo[k] >> 16), kv_half2(hi[k] >> 16)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_half(sc[n][u], a, qb[n][b][k][0], qb[n][b][k][1]);
                        }
                    }
                // scores of tokens 8 x + g (x = 2 u, 2 u + 1) for heads 2 t, 2 t + 1
                float vs[4];  // 2^(127 - Ev)
                {
                    float ev[4], kf[4];
                    bool there[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t w = __shfl_sync(0xffffffffu, powers, (lane & ~3) | x);
                        kf[x] = kv_up(w & 255);
                        ev[x] = (float)((int)((w >> 8) & 255) - 127);
                        vs[x] = kv_down((w >> 8) & 255);
                        there[x] = (w >> 16) != 0;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int x = 2 * u + (e >> 1);
                                sc[n][u][e] = there[x] ? fmaf(sc[n][u][e] * qf[n][e & 1], kf[x], ev[x]) : -INFINITY;
                            }
                }
                uint32_t pb[NT][2][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float keep[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(fmaxf(sc[n][0][e], sc[n][0][2 + e]), fmaxf(sc[n][1][e], sc[n][1][2 + e]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float m_new = fmaxf(m[n][e], top), ref = m_new == -INFINITY ? 0.f : m_new - 14.f;
                        keep[e] = fast_exp2(m[n][e] - 14.f - ref);
                        m[n][e] = m_new;
                        float sum = 0.f;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float w = fast_exp2(sc[n][u][2 * r + e] - ref);
                                sc[n][u][2 * r + e] = w;
                                sum = fmaf(w, vs[2 * u + r], sum);
                            }
                        l[n][e] = fmaf(l[n][e], keep[e], sum);
                    }
                    if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
                        for (int j = 0; j < HD / 16; ++j) {
                            o[n][j][0] *= keep[0]; o[n][j][1] *= keep[1]; o[n][j][2] *= keep[0]; o[n][j][3] *= keep[1];
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < 2; ++r) pb[n][u][r] = transposed(half2_of(sc[n][u][2 * r], sc[n][u][2 * r + 1]));
                }
                // O^T += V^T P^T: a thread pairs tokens (2 t, 2 t + 1) and (2 t + 8, 2 t + 9); its words of a row: 16 bytes of every
                // 128, then 8 of 64 and 4 of 32
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t w[4][WORDS];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int r = 16 * u + 2 * t + (x & 1) + 8 * (x >> 1);
                        constexpr int W16 = HD / 128;
#pragma unroll
                        for (int j = 0; j < W16; ++j) {
                            const uint4 v = *reinterpret_cast<const uint4*>(vt + C::at(r, 8 * j + g));
                            w[x][4 * j] = v.x; w[x][4 * j + 1] = v.y; w[x][4 * j + 2] = v.z; w[x][4 * j + 3] = v.w;
                        }
                        if (HD % 128 >= 64) {
                            const uint2 v = *reinterpret_cast<const uint2*>(vt + C::at(r, 8 * W16 + (g >> 1)) + 8 * (g & 1));
                            w[x][4 * W16] = v.x;
                            w[x][4 * W16 + 1] = v.y;
                        }
                        if (HD % 64 == 32) w[x][WORDS - 1] = *reinterpret_cast<const uint32_t*>(vt + C::at(r, HD / 16 - 2 + (g >> 2)) + 4 * (g & 3));
                    }
#pragma unroll
                    for (int j = 0; j < WORDS; ++j) {
                        const uint32_t a01 = __byte_perm(w[0][j], w[1][j], 0x5140), a23 = __byte_perm(w[0][j], w[1][j], 0x7362);
                        const uint32_t b01 = __byte_perm(w[2][j], w[3][j], 0x5140), b23 = __byte_perm(w[2][j], w[3][j], 0x7362);
                        const uint32_t even[4] = {kv_half2(a01 & 0xFFFF), kv_half2(a01 >> 16), kv_half2(b01 & 0xFFFF), kv_half2(b01 >> 16)};
                        const uint32_t odd[4] = {kv_half2(a23 & 0xFFFF), kv_half2(a23 >> 16), kv_half2(b23 & 0xFFFF), kv_half2(b23 >> 16)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma_half(o[n][2 * j], even, pb[n][u][0], pb[n][u][1]);
                            mma_half(o[n][2 * j + 1], odd, pb[n][u][0], pb[n][u][1]);
                        }
                    }
                }
                powers = powers_next;
                __syncwarp();  // the stage is free
            }
            cp_async_wait<0>();
            // ---- the four warps' shares ----
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                    if (g == 0) {
                        m_s[warp][8 * n + 2 * t + e] = m[n][e];
                        l_s[warp][8 * n + 2 * t + e] = l[n][e];
                    }
                }
            __syncthreads();  // the rings are read: the partial sums lie over them
            float* sums = reinterpret_cast<float*>(ring_s);  // [WARPS][ROWS][HD]
            static_assert(WARPS * ROWS * HD * 4 <= C::RING, "the partial sums must fit over the rings");
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < WORDS; ++j) {
                    const int d = j < HD / 128 * 4 ? (j / 4) * 128 + 16 * g + 4 * (j % 4)
                                  : (HD % 128 >= 64 && j < HD / 128 * 4 + 2) ? HD / 128 * 128 + 8 * g + 4 * (j - HD / 128 * 4) : HD - 32 + 4 * g;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4*>(sums + (warp * ROWS + 8 * n + 2 * t + e) * HD + d) =
                            make_float4(o[n][2 * j][e], o[n][2 * j][2 + e], o[n][2 * j + 1][e], o[n][2 * j + 1][2 + e]);
                }
            if (tid < ROWS) {
                float top = -INFINITY, total = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) top = fmaxf(top, m_s[w][tid]);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float f = m_s[w][tid] == -INFINITY ? 0.f : fast_exp2(m_s[w][tid] - top);
                    w_s[tid][w] = f;
                    total += f * l_s[w][tid];
                }
                w_s[tid][WARPS] = top;
                w_s[tid][WARPS + 1] = total;
            }
            __syncthreads();
            const int first_block = seg_first / range.quota, last_block = (seg_first + tiles - 1) / range.quota;
            const int pieces = last_block - first_block + 1;
            const int my_piece = 2 * blockIdx.x + (seg_first < range.first ? 0 : 1);
            for (int i = tid; i < rows * (HD / 4); i += blockDim.x) {
                const int r = i / (HD / 4), d = i % (HD / 4) * 4;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(sums + (w * ROWS + r) * HD + d);
                    const float f = w_s[r][w];
                    sum.x = fmaf(f, x.x, sum.x); sum.y = fmaf(f, x.y, sum.y); sum.z = fmaf(f, x.z, sum.z); sum.w = fmaf(f, x.w, sum.w);
                }
                if (pieces == 1) {
                    const float total = w_s[r][WARPS + 1], inv = total == 0.f ? 0.f : 1.f / total;
                    Vec4<bf16>::store((bf16*)p.out + ((size_t)row * p.nh + h0 + r) * HD + d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
                } else {
                    *reinterpret_cast<float4*>(p.part_o + ((size_t)my_piece * ROWS + r) * HD + d) = sum;
                    if (d == 0) *reinterpret_cast<float2*>(p.part_ml + ((size_t)my_piece * ROWS + r) * 2) = make_float2(w_s[r][WARPS], w_s[r][WARPS + 1]);
                }
            }
            if (pieces > 1) {
                // piece number x of the segment: of block first_block + x, its second one where the segment begins in it
                auto place = [&](int x) { return (size_t)2 * (first_block + x) + (x == 0 ? 1 : 0); };
                int from = 0, count = pieces, step = 1;
                int* counter = p.counters + s * per_request + seg;
                bool final = true;
                if (pieces > 2 * MERGE_AT_ONCE) {
                    const int x = blockIdx.x - first_block;
                    from = x - x % MERGE_AT_ONCE;
                    count = min(MERGE_AT_ONCE, pieces - from);
                    counter = p.counters + p.requests * per_request + place(from);
                    final = false;
                }
                for (;;) {
                    // the barrier orders all threads' stores before thread 0's release; the last block's acquire, followed by the
                    // next barrier, its threads' loads behind everybody's stores
                    __syncthreads();
                    if (tid == 0) {
                        int before;
                        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
                        last_s = before == count - 1;
                        if (last_s) *counter = 0;
                    }
                    __syncthreads();
                    if (!last_s) break;
                    for (int i = tid; i < rows * (HD / 4); i += blockDim.x) {
                        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
                        float top = -INFINITY, total = 0.f;
                        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                        for (int x0 = 0; x0 < count; x0 += MERGE_AT_ONCE) {
                            float2 ml[MERGE_AT_ONCE];
                            float4 v[MERGE_AT_ONCE];
#pragma unroll
                            for (int x = 0; x < MERGE_AT_ONCE; ++x) {
                                ml[x] = make_float2(-INFINITY, 0.f);
                                v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (x0 + x < count) {
                                    const size_t at = place(from + (x0 + x) * step) * ROWS + r;
                                    ml[x] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + at);
                                    v[x] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD + d));
                                }
                            }
                            float next = top;
#pragma unroll
                            for (int x = 0; x < MERGE_AT_ONCE; ++x) next = fmaxf(next, ml[x].x);
                            const float keep = top == -INFINITY ? 0.f : fast_exp2(top - next);
                            total *= keep; sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
                            top = next;
#pragma unroll
                            for (int x = 0; x < MERGE_AT_ONCE; ++x) {
                                const float f = ml[x].x == -INFINITY ? 0.f : fast_exp2(ml[x].x - top);
                                total = fmaf(f, ml[x].y, total);
                                sum.x = fmaf(f, v[x].x, sum.x); sum.y = fmaf(f, v[x].y, sum.y);
                                sum.z = fmaf(f, v[x].z, sum.z); sum.w = fmaf(f, v[x].w, sum.w);
                            }
                        }
                        if (final) {
                            const float inv = total == 0.f ? 0.f : 1.f / total;
                            Vec4<bf16>::store((bf16*)p.out + ((size_t)row * p.nh + h0 + r) * HD + d,
                                              make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
                        } else {  // over the first of the twelve, whose four sums this thread alone reads and writes
                            *reinterpret_cast<float4*>(p.part_o + (place(from) * ROWS + r) * HD + d) = sum;
                            if (d == 0) {
                                w_s[r][0] = top;
                                w_s[r][1] = total;
                            }
                        }
                    }
                    if (final) break;
                    __syncthreads();  // (their maxima and sums are read by all)
                    if (tid < rows) *reinterpret_cast<float2*>(p.part_ml + (place(from) * ROWS + tid) * 2) = make_float2(w_s[tid][0], w_s[tid][1]);
                    from = 0;
                    count = (pieces + MERGE_AT_ONCE - 1) / MERGE_AT_ONCE;
                    step = MERGE_AT_ONCE;
                    counter = p.counters + s * per_request + seg;
                    final = true;
                }
            }
            __syncthreads();  // before the rings, the queries and the factors are written again
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

template <int HD, int NT>
static int stream_launch(const DecodeE4m3Params& p, int sms, cudaStream_t stream) {
    using C = Stream<HD>;
    static bool configured[64] = {};  // (per device)
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= 64 || !configured[device]) {
        const cudaError_t e = cudaFuncSetAttribute(decode_e4m3_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::RING);
        if (e != cudaSuccess) return (int)e;
        if (device >= 0 && device < 64) configured[device] = true;
    }
    return cw_launch(decode_e4m3_kernel<HD, NT>, dim3(sms * C::PER_SM), dim3(WARPS * 32), C::RING, stream, 1u, p);
}
template <int HD>
static int stream_launch_heads(const DecodeE4m3Params& p, int sms, cudaStream_t stream) {
    if (p.heads_each <= 8) return stream_launch<HD, 1>(p, sms, stream);
    return stream_launch<(HD <= 128 ? HD : 32), 2>(p, sms, stream);  // (head sizes beyond 128 come in groups of 8)
}

// How a KV head's query heads are shared out: groups of 16 at most, of 8 where heads are so large that the sums of 16 would not
// stay in registers; 0: the streaming kernel does not take the head size or the type.
static int groups_of(int nh, int nkv, int hd, int dtype) {
    if (dtype != 1 || hd % 32) return 0;
    const int each = nh / nkv, most = hd <= 128 ? 16 : 8;
    return (each + most - 1) / most;
}

// Scratch of the call: float32 words and zeroed int32 words (which are zero again when it has run).
extern "C" int cw_attention_decode_e4m3_scratch(int requests, int nh, int nkv, int hd, int dtype, int sms, long long* floats, int* words) {
    if (requests < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || hd > 256 || sms <= 0) return CW_ERR_BAD_SIZE;
    const int groups = groups_of(nh, nkv, hd, dtype);
    const long long pieces = groups ? 4LL * sms : 0;  // two blocks an SM, two pieces a block
    *floats = pieces * 16 * (hd + 2);
    *words = groups ? (int)(requests * nkv * groups + pieces) : 0;
    return CW_OK;
}

// q [rows, q_stride >= nh * hd], out [rows, nh * hd]; request s owns row s, or with q_start rows q_start[s] .. q_start[s + 1], and
// then only requests with one row are served.  A context of length 0 gives zeros.  `floats`, `words`: the scratch.
extern "C" int cw_attention_decode_e4m3(const void* q, int q_stride, void* out, const uint8_t* k, const uint8_t* v, const uint8_t* k_exp,
                                        const uint8_t* v_exp, const int* block_tables, const int* ctx_lens, const int* q_start,
                                        int requests, int nh, int nkv, int hd, int page_size, int max_blocks, int num_pages, int window,
                                        float scale, int dtype, int sms, float* floats, int* words, int* status, cudaStream_t stream) {
    if (requests == 0) return CW_OK;
    if (requests < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || hd % 16 || hd > 256 || page_size <= 0 || max_blocks <= 0 ||
        num_pages <= 0 || window < 0 || q_stride < nh * hd || ((uintptr_t)k | (uintptr_t)v) % 16 || requests > 65535 || sms <= 0 ||
        (long long)num_pages * page_size > 0x7FFFFFFF || (long long)max_blocks * page_size > 0x7FFFFFFF)
        return CW_ERR_BAD_SIZE;
    DecodeE4m3Params p = {q, q_stride, out, k, v, k_exp, v_exp, block_tables, ctx_lens, q_start, requests, nh, nkv, hd, page_size,
                          max_blocks, num_pages, window, scale, status};
    const int groups = groups_of(nh, nkv, hd, dtype);
    if (groups && floats != nullptr && words != nullptr && (long long)num_pages * page_size * nkv < (1LL << 32) &&
        (long long)requests * nkv * groups * ((long long)max_blocks * page_size / TILE_TOKENS + 2) < 0x7FFFFFFF) {
        p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
        p.groups = groups;
        p.heads_each = (nh / nkv + groups - 1) / groups;
        p.part_o = floats;
        p.part_ml = floats + 4LL * sms * 16 * hd;
        p.counters = words;
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

CW_TRACE_TU(attention_decode_e4m3)
