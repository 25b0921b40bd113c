// Writing the paged cache behind the norms of the heads and the position rotation, and reading an 8-bit cache back.
//
// norm_rotate_store, per token t and head: x = the head's entries of the [q | k | v] row, float32;
//     q, k:  x <- x * rsqrt(mean(x^2) + eps) * w        (where the layer norms its heads)
//            (x_j, x_{j + rot/2}) turned by position * inv_freq[j], j < rot/2
// q is rounded once to the run's type and handed on; k (float32, not rounded before) and v become rows of the cache: 8-bit rows
// (kv_e4m3.cuh) or rows of the run's type.  Angles, their sines and cosines are worked out in float64 and
// rounded once: position * inv_freq is exact there, so that a position of a million is turned as exactly as the first, and a key's
// last bits, which decide between two codes, are not the sine's.  (An angle serves all heads: 64 of them beside 4,608 entries.)
//
// read_pages: code * 2^(E - 127) in bfloat16 (exact) or float32 for the positions of every request's context, at the same page
// and slot of a plain cache; the rest of a request's last page becomes zero.  Both are streams over memory.
#include "kv_e4m3.cuh"

struct StoreParams {
    const void* qkv; void* q_out;
    const int* positions; const int* slots;
    const float* inv_freq; const float* q_weight; const float* k_weight;
    void* k_cache; void* v_cache; uint8_t* k_exp; uint8_t* v_exp;  // k_exp null: a plain cache
    int N, nh, nkv, hd, rot, page_size, num_slots;
    float eps;
    int early;  // positions, slots and frequencies are older than the kernel in front: angles are worked out while that one finishes
    int* status;
};

// LG neighbouring lanes hold a head, a lane two octets of it (octet i, i < rot / 8: four entries and the four that turn with them;
// behind those, eight neighbours), so that pairs never leave a thread, the mean of squares and the largest magnitude are shuffles
// among LG lanes, and accesses are of 8 or 16 bytes.  A thread keeps its head and its entries for a block's tokens, whose rows are
// loaded one ahead: weights, offsets and the kind of head are found out once.  Blocks have as many tokens as leave the SMs two
// blocks each, eight at most.
#define STORE_TOKENS 8
template <typename T, int LG>
__global__ void __launch_bounds__(512) norm_rotate_store_kernel(const StoreParams p, int most_tokens, int block_heads) {
    extern __shared__ float turn[];  // per token: cos[rot / 2], sin[rot / 2]
    __shared__ int slot_s[STORE_TOKENS], off_s[STORE_TOKENS];  // a token's slot (-1: none) and its place in its page
    if (p.early)
        pdl_launch_dependents();
    else
        pdl_enter();
    const int t0 = blockIdx.x * most_tokens, tokens = min(most_tokens, p.N - t0), half = p.rot >> 1;
    const int heads = p.nh + 2 * p.nkv, l = threadIdx.x % LG, turning = p.rot >> 3;
    const int own = threadIdx.x / LG, head = blockIdx.y * block_heads + own;
    const bool live = own < block_heads && head < heads, is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
    int a_at[2], b_at[2];
    bool there[2], turns[2];
    float4 a_next[2], b_next[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int octet = l + e * LG;
        there[e] = live && octet < (p.hd >> 3);
        turns[e] = octet < turning && !is_v;
        a_at[e] = octet < turning ? 4 * octet : p.rot + 8 * (octet - turning);
        b_at[e] = octet < turning ? half + 4 * octet : a_at[e] + 4;
        a_next[e] = b_next[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const T* row = (const T*)p.qkv + ((size_t)t0 * heads + head) * p.hd;
    auto load = [&]() {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (there[e]) {
                a_next[e] = Vec4<T>::load(row + a_at[e]);
                b_next[e] = Vec4<T>::load(row + b_at[e]);
            }
        row += (size_t)heads * p.hd;
    };
    if (!p.early) load();
    if (threadIdx.x < tokens) {
        int slot = p.slots[t0 + threadIdx.x];
        if (slot >= p.num_slots) {
            if (blockIdx.y == 0) cw_report(p.status, CW_ST_SLOT_RANGE, t0 + threadIdx.x, slot);
            slot = -1;
        }
        slot_s[threadIdx.x] = slot;
        off_s[threadIdx.x] = max(slot, 0) % p.page_size;
    }
    for (int i = threadIdx.x; i < tokens * half; i += blockDim.x) {
        const int t = i / half, j = i - t * half;
        turn_of(p.positions[t0 + t], p.inv_freq[j], turn[t * p.rot + half + j], turn[t * p.rot + j]);
    }
    const float* weight = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
    float4 wa[2], wb[2];
    if (weight != nullptr)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (there[e]) {
                wa[e] = *reinterpret_cast<const float4*>(weight + a_at[e]);
                wb[e] = *reinterpret_cast<const float4*>(weight + b_at[e]);
            }
    const bool any_norm = __any_sync(0xffffffffu, live && weight != nullptr), any_kv = __any_sync(0xffffffffu, live && !is_q);
    const int kvh = is_v ? head - p.nh - p.nkv : head - p.nh;
    if (p.early) {
        pdl_wait();
        load();
    }
    __syncthreads();
    for (int t = 0; t < tokens; ++t) {
        float4 a[2] = {a_next[0], a_next[1]}, b[2] = {b_next[0], b_next[1]};
        if (t + 1 < tokens) load();
        if (any_norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // (entries that there are not: zeros)
                sum = fmaf(a[e].x, a[e].x, fmaf(a[e].y, a[e].y, fmaf(a[e].z, a[e].z, fmaf(a[e].w, a[e].w, sum))));
                sum = fmaf(b[e].x, b[e].x, fmaf(b[e].y, b[e].y, fmaf(b[e].z, b[e].z, fmaf(b[e].w, b[e].w, sum))));
            }
#pragma unroll
            for (int o = LG / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (weight != nullptr) {
                const float r = __frcp_rn(__fsqrt_rn(__fdiv_rn(sum, (float)p.hd) + p.eps));
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (there[e]) {
                        a[e].x *= r * wa[e].x; a[e].y *= r * wa[e].y; a[e].z *= r * wa[e].z; a[e].w *= r * wa[e].w;
                        b[e].x *= r * wb[e].x; b[e].y *= r * wb[e].y; b[e].z *= r * wb[e].z; b[e].w *= r * wb[e].w;
                    }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (turns[e]) {
                const float* at = turn + t * p.rot + a_at[e];
                const float4 cs = *reinterpret_cast<const float4*>(at), sn = *reinterpret_cast<const float4*>(at + half), x = a[e], y = b[e];
                a[e].x = x.x * cs.x - y.x * sn.x; a[e].y = x.y * cs.y - y.y * sn.y; a[e].z = x.z * cs.z - y.z * sn.z; a[e].w = x.w * cs.w - y.w * sn.w;
                b[e].x = y.x * cs.x + x.x * sn.x; b[e].y = y.y * cs.y + x.y * sn.y; b[e].z = y.z * cs.z + x.z * sn.z; b[e].w = y.w * cs.w + x.w * sn.w;
            }
        const int slot = slot_s[t];
        const bool stores = live && !is_q && slot >= 0;
        const size_t at = ((size_t)max(slot, 0) * p.nkv + kvh) * p.hd;
        if ((live && is_q) || (stores && p.k_exp == nullptr)) {  // rows of the run's type
            T* out = is_q ? (T*)p.q_out + ((size_t)(t0 + t) * p.nh + head) * p.hd : (T*)(is_v ? p.v_cache : p.k_cache) + at;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (there[e]) {
                    Vec4<T>::store(out + a_at[e], a[e]);
                    Vec4<T>::store(out + b_at[e], b[e]);
                }
        }
        if (!any_kv || p.k_exp == nullptr) continue;
        float big = 0.f;  // (NaN has no say)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            big = fmaxf(big, fmaxf(fmaxf(fmaxf(fabsf(a[e].x), fabsf(a[e].y)), fmaxf(fabsf(a[e].z), fabsf(a[e].w))),
                                   fmaxf(fmaxf(fabsf(b[e].x), fabsf(b[e].y)), fmaxf(fabsf(b[e].z), fabsf(b[e].w)))));
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        if (big > KV_BIGGEST) {
            big = KV_BIGGEST;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[e].x = kv_clamped(a[e].x); a[e].y = kv_clamped(a[e].y); a[e].z = kv_clamped(a[e].z); a[e].w = kv_clamped(a[e].w);
                b[e].x = kv_clamped(b[e].x); b[e].y = kv_clamped(b[e].y); b[e].z = kv_clamped(b[e].z); b[e].w = kv_clamped(b[e].w);
            }
        }
        if (stores) {
            const int power = kv_power(big), off = off_s[t];
            const float d = kv_down(power);
            uint8_t* out = (uint8_t*)(is_v ? p.v_cache : p.k_cache) + at;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (there[e]) {
                    *reinterpret_cast<uint32_t*>(out + a_at[e]) = kv_codes(a[e].x * d, a[e].y * d, a[e].z * d, a[e].w * d);
                    *reinterpret_cast<uint32_t*>(out + b_at[e]) = kv_codes(b[e].x * d, b[e].y * d, b[e].z * d, b[e].w * d);
                }
            // (slot - off: the page times page_size, and a page has nkv rows of page_size powers)
            if (l == 0) (is_v ? p.v_exp : p.k_exp)[(size_t)(slot - off) * p.nkv + (size_t)kvh * p.page_size + off] = (uint8_t)power;
        }
    }
}

// Any even rotary span and any alignment: a warp per head, an entry per lane and round.
template <typename T>
__global__ void norm_rotate_store_any_kernel(const StoreParams p) {
    extern __shared__ float turn[];
    pdl_enter();
    const int t = blockIdx.x, half = p.rot >> 1, lane = threadIdx.x & 31;
    const int pos = p.positions[t];
    for (int j = threadIdx.x; j < half; j += blockDim.x) turn_of(pos, p.inv_freq[j], turn[half + j], turn[j]);
    int slot = p.slots[t];
    if (slot >= p.num_slots) {
        if (threadIdx.x == 0) cw_report(p.status, CW_ST_SLOT_RANGE, t, slot);
        slot = -1;
    }
    const int page = slot >= 0 ? slot / p.page_size : 0, off = slot >= 0 ? slot - page * p.page_size : 0;
    __syncthreads();
    const int heads = p.nh + 2 * p.nkv;
    for (int head = threadIdx.x >> 5; head < heads; head += blockDim.x >> 5) {
        const bool is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
        const T* x = (const T*)p.qkv + ((size_t)t * heads + head) * p.hd;
        const float* weight = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
        float r = 1.f;
        if (weight != nullptr) {
            float sum = 0.f;
            for (int j = lane; j < p.hd; j += 32) sum += to_f(x[j]) * to_f(x[j]);
            r = __frcp_rn(__fsqrt_rn(__fdiv_rn(warp_sum(sum), (float)p.hd) + p.eps));
        }
        auto normed = [&](int j) { return weight != nullptr ? to_f(x[j]) * (r * weight[j]) : to_f(x[j]); };
        auto entry = [&](int j) {
            if (is_v || j >= p.rot) return normed(j);
            return j < half ? normed(j) * turn[j] - normed(j + half) * turn[half + j]
                            : normed(j) * turn[j - half] + normed(j - half) * turn[j];
        };
        const int kvh = is_v ? head - p.nh - p.nkv : head - p.nh;
        const size_t at = ((size_t)(slot < 0 ? 0 : slot) * p.nkv + kvh) * p.hd;
        if (is_q) {
            for (int j = lane; j < p.hd; j += 32) ((T*)p.q_out)[((size_t)t * p.nh + head) * p.hd + j] = from_f<T>(entry(j));
        } else if (slot >= 0 && p.k_exp == nullptr) {
            for (int j = lane; j < p.hd; j += 32) ((T*)(is_v ? p.v_cache : p.k_cache))[at + j] = from_f<T>(entry(j));
        } else if (slot >= 0) {
            float big = 0.f;
            for (int j = lane; j < p.hd; j += 32) big = fmaxf(big, fabsf(kv_clamped(entry(j))));
            const int power = kv_power(warp_max(big));
            uint8_t* out = (uint8_t*)(is_v ? p.v_cache : p.k_cache) + at;
            for (int j = lane; j < p.hd; j += 32)
                out[j] = __nv_cvt_float_to_fp8(kv_clamped(entry(j)) * kv_down(power), __NV_SATFINITE, __NV_E4M3);
            if (lane == 0) (is_v ? p.v_exp : p.k_exp)[((size_t)page * p.nkv + kvh) * p.page_size + off] = (uint8_t)power;
        }
    }
}

static inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

template <typename T>
static int store_launch(const StoreParams& p, int N, cudaStream_t stream) {
    const int heads = p.nh + 2 * p.nkv, smem = p.rot * (int)sizeof(float);
    const int w = 4 * (int)sizeof(T);
    const bool quads = p.rot % 8 == 0 && p.hd % 8 == 0 && aligned(p.qkv, w) && aligned(p.q_out, w) &&
                       aligned(p.k_cache, p.k_exp ? 4 : w) && aligned(p.v_cache, p.k_exp ? 4 : w) && aligned(p.q_weight, 16) &&
                       aligned(p.k_weight, 16);
    if (!quads) {
        const int threads = heads < 8 ? heads * 32 : 256;
        return cw_launch(norm_rotate_store_any_kernel<T>, dim3(N), dim3(threads), smem, stream, 1u, p);
    }
    int lg = 1;
    while (lg * 16 < p.hd) lg *= 2;
    const int chunks = (heads * lg + 511) / 512, block_heads = (heads + chunks - 1) / chunks;
    const int tokens = max(1, min(STORE_TOKENS, (N * chunks + 2 * 148 - 1) / (2 * 148)));
    const dim3 grid((N + tokens - 1) / tokens, chunks), block((block_heads * lg + 31) / 32 * 32);
    const size_t room = (size_t)tokens * smem;
    switch (lg) {
        case 1: return cw_launch(norm_rotate_store_kernel<T, 1>, grid, block, room, stream, 1u, p, tokens, block_heads);
        case 2: return cw_launch(norm_rotate_store_kernel<T, 2>, grid, block, room, stream, 1u, p, tokens, block_heads);
        case 4: return cw_launch(norm_rotate_store_kernel<T, 4>, grid, block, room, stream, 1u, p, tokens, block_heads);
        case 8: return cw_launch(norm_rotate_store_kernel<T, 8>, grid, block, room, stream, 1u, p, tokens, block_heads);
        default: return cw_launch(norm_rotate_store_kernel<T, 16>, grid, block, room, stream, 1u, p, tokens, block_heads);
    }
}

// q_out [N, nh * hd]; slots[t] < 0: the token is not stored.  k_exp and v_exp null: the cache is of the run's type.
// rot 0: nothing turns (inv_freq may be null).  The norms' weights are float32 [hd] or null.
// The arguments come as one block of words (kv_e4m3.cuh), in the order of the names below.
extern "C" int cw_norm_rotate_store(const char* block) {
    ArgumentWords w(block);
    const void* qkv = w.pointer(); void* q_out = w.pointer();
    const int *positions = (const int*)w.pointer(), *slots = (const int*)w.pointer();
    const float *inv_freq = (const float*)w.pointer(), *q_weight = (const float*)w.pointer(), *k_weight = (const float*)w.pointer();
    void *k_cache = w.pointer(), *v_cache = w.pointer();
    uint8_t *k_exp = (uint8_t*)w.pointer(), *v_exp = (uint8_t*)w.pointer();
    int* status = (int*)w.pointer();
    const cudaStream_t stream = (cudaStream_t)w.pointer();
    const int N = w.number(), nh = w.number(), nkv = w.number(), hd = w.number(), rot = w.number(), page_size = w.number(), num_pages = w.number(),
              dtype = w.number(), early = w.number();
    const float eps = (float)w.real();
    if (N == 0) return CW_OK;
    if (N < 0 || nh <= 0 || nkv <= 0 || hd <= 0 || hd > 256 || rot < 0 || rot > hd || rot % 2 || page_size <= 0 || num_pages <= 0 ||
        (long long)num_pages * page_size > 0x7FFFFFFF || (rot > 0 && inv_freq == nullptr) || (k_exp == nullptr) != (v_exp == nullptr))
        return CW_ERR_BAD_SIZE;
    const StoreParams p = {qkv, q_out, positions, slots, inv_freq, q_weight, k_weight, k_cache, v_cache, k_exp, v_exp,
                           N, nh, nkv, hd, rot, page_size, num_pages * page_size, eps, early, status};
    if (dtype == 0) return store_launch<float>(p, N, stream);
    if (dtype == 1) return store_launch<bf16>(p, N, stream);
    return CW_ERR_BAD_DTYPE;
}

struct ReadParams {
    const uint8_t* k; const uint8_t* v; const uint8_t* k_exp; const uint8_t* v_exp;
    void* k_out; void* v_out;
    const int* block_tables; const int* ctx_lens; const int* q_start;
    int requests, nkv, hd, page_size, max_blocks, num_pages, window, least_rows;
    int* status;
};

__device__ __forceinline__ void store8(float* at, float a, float b, float c, float d, float e, float f, float g, float h) {
    *reinterpret_cast<float4*>(at) = make_float4(a, b, c, d);
    *reinterpret_cast<float4*>(at + 4) = make_float4(e, f, g, h);
}
__device__ __forceinline__ void store8(bf16* at, float a, float b, float c, float d, float e, float f, float g, float h) {
    const __nv_bfloat162 x[4] = {__floats2bfloat162_rn(a, b), __floats2bfloat162_rn(c, d), __floats2bfloat162_rn(e, f), __floats2bfloat162_rn(g, h)};
    *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(x);
}

// x / d for x * d < 2^32, by a multiplication.
struct Quotient {
    uint32_t d, magic;
    static Quotient by(uint32_t d) { return {d, d == 1 ? 0u : (uint32_t)(((1ULL << 32) + d - 1) / d)}; }
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return d == 1 ? x : __umulhi(x, magic); }
};

// Units are pages of a request, keys and values apart, a warp to each, so that thousands are on their way at once.  A page's codes
// are one run of memory, and so is where they go; a lane takes 8 codes at a time (they share a row and its power), so that a
// warp writes whole lines.
#define READ_AT_ONCE 8
template <typename T>
__global__ void __launch_bounds__(256) read_pages_kernel(const ReadParams p, const Quotient by_chunks, const Quotient by_heads) {
    __shared__ int sh[36];
    pdl_enter();
    auto span = [&](int s, int& from) {  // a request's blocks that are read: how many, and the first
        int ctx = p.ctx_lens[s], first = ctx;
        if (p.q_start != nullptr) {
            const int rows = p.q_start[s + 1] - p.q_start[s];
            if (rows < p.least_rows) return 0;
            first = ctx - rows + 1;  // (a portion's first row sees `window` keys, its own among them: the window reaches back from there)
        }
        from = p.window > 0 ? max(0, first - p.window) / p.page_size : 0;
        return max(0, min((ctx + p.page_size - 1) / p.page_size, p.max_blocks) - from);
    };
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    const UnitRange r = units_of_block([&](int s) { int from; return 2 * span(s, from); }, p.requests, warps, gridDim.x, blockIdx.x, sh);
    const int chunks = p.page_size * p.nkv * (p.hd >> 3);
    int s = r.request, at = r.offset + (threadIdx.x >> 5);  // units of a block go to its warps in turn
    for (int u = r.first + (threadIdx.x >> 5); u < r.last; u += warps, at += warps) {
        int from = 0, n = 2 * span(s, from);
        while (at >= n && s + 1 < p.requests) {
            at -= n;
            n = 2 * span(++s, from);
        }
        const bool is_v = at & 1;
        const int block = from + (at >> 1), page = block < p.max_blocks ? p.block_tables[(size_t)s * p.max_blocks + block] : -1;
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) cw_report(p.status, CW_ST_PAGE_RANGE, s, page);
            continue;
        }
        const uint2* src = reinterpret_cast<const uint2*>(is_v ? p.v : p.k) + (size_t)page * chunks;
        const uint8_t* powers = (is_v ? p.v_exp : p.k_exp) + (size_t)page * p.nkv * p.page_size;
        T* dst = (T*)(is_v ? p.v_out : p.k_out) + (size_t)page * chunks * 8;
        const int live = min(p.page_size, p.ctx_lens[s] - block * p.page_size) * p.nkv;  // rows that hold something
        for (int i0 = lane; i0 < chunks; i0 += 32 * READ_AT_ONCE) {
            uint2 codes[READ_AT_ONCE];
            uint32_t power[READ_AT_ONCE];
#pragma unroll
            for (int k = 0; k < READ_AT_ONCE; ++k) {
                const int i = i0 + 32 * k, row = by_chunks.of(i), token = by_heads.of(row);
                codes[k] = make_uint2(0, 0);
                power[k] = 0;
                if (i < chunks && row < live) {
                    codes[k] = __ldcs(src + i);
                    power[k] = powers[(row - token * p.nkv) * p.page_size + token];
                }
            }
#pragma unroll
            for (int k = 0; k < READ_AT_ONCE; ++k) {
                const int i = i0 + 32 * k;
                if (i >= chunks) break;
                const float up = kv_up(power[k]);
                const float2 x0 = kv_float2(codes[k].x), x1 = kv_float2(codes[k].x >> 16), x2 = kv_float2(codes[k].y), x3 = kv_float2(codes[k].y >> 16);
                store8(dst + (size_t)i * 8, x0.x * up, x0.y * up, x1.x * up, x1.y * up, x2.x * up, x2.y * up, x3.x * up, x3.y * up);
            }
        }
    }
}

// q_start (or null): only requests with at least `least_rows` rows (1 or more) are read.  window > 0: from the page on that the first of a request's
// rows (its last position without q_start) still sees.
extern "C" int cw_read_pages(const char* block) {
    ArgumentWords w(block);
    const uint8_t *k = (const uint8_t*)w.pointer(), *v = (const uint8_t*)w.pointer(), *k_exp = (const uint8_t*)w.pointer(), *v_exp = (const uint8_t*)w.pointer();
    void *k_out = w.pointer(), *v_out = w.pointer();
    const int *block_tables = (const int*)w.pointer(), *ctx_lens = (const int*)w.pointer(), *q_start = (const int*)w.pointer();
    int* status = (int*)w.pointer();
    const cudaStream_t stream = (cudaStream_t)w.pointer();
    const int requests = w.number(), nkv = w.number(), hd = w.number(), page_size = w.number(), max_blocks = w.number(), num_pages = w.number(),
              window = w.number(), least_rows = w.number(), blocks = w.number(), dtype = w.number();
    if (requests == 0) return CW_OK;
    if (requests < 0 || nkv <= 0 || hd <= 0 || hd % 16 || page_size <= 0 || max_blocks <= 0 || num_pages <= 0 || window < 0 || blocks <= 0 || least_rows < 1 ||
        !aligned(k, 16) || !aligned(v, 16) || !aligned(k_out, 16) || !aligned(v_out, 16) ||
        (long long)page_size * nkv * (hd >> 3) * max(hd >> 3, nkv) > 0x7FFFFFFF)  // (Quotient's range)
        return CW_ERR_BAD_SIZE;
    const ReadParams p = {k, v, k_exp, v_exp, k_out, v_out, block_tables, ctx_lens, q_start, requests, nkv, hd, page_size,
                          max_blocks, num_pages, window, least_rows, status};
    const Quotient by_chunks = Quotient::by(hd >> 3), by_heads = Quotient::by(nkv);
    if (dtype == 0) return cw_launch(read_pages_kernel<float>, dim3(blocks), dim3(256), 0, stream, 1u, p, by_chunks, by_heads);
    if (dtype == 1) return cw_launch(read_pages_kernel<bf16>, dim3(blocks), dim3(256), 0, stream, 1u, p, by_chunks, by_heads);
    return CW_ERR_BAD_DTYPE;
}

CW_TRACE_TU(kv_e4m3)
