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
// and slot of a plain cache; what no request holds of a last page becomes zero.  Both are streams over memory.
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

// sin and cos of position * freq (a product that float64 holds exactly), rounded once: the angle less the nearest multiple k of pi/2,
// which leaves |x| <= pi/4, then the Taylor sums to x^11 and x^10 (the next terms are below 2^-33), turned by k quarters.
__device__ __forceinline__ void turn_of(int position, float freq, float& sn, float& cs) {
    const double angle = (double)position * (double)freq, k = rint(angle * 0.63661977236758134308);
    // pi/2 as a float64 and what that leaves of it
    const double x = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, angle)), y = x * x;
    const double s = x * fma(y, fma(y, fma(y, fma(y, fma(y, -1.0 / 39916800, 1.0 / 362880), -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
    const double c = fma(y, fma(y, fma(y, fma(y, fma(y, -1.0 / 3628800, 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
    const int quarter = (int)((long long)k & 3);
    const float a = (float)(quarter & 1 ? c : s), b = (float)(quarter & 1 ? s : c);
    sn = quarter & 2 ? -a : a;
    cs = (quarter == 1 || quarter == 2) ? -b : b;
}

// Two float32 products, or products and sums, at a time.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)),
        "l"(*reinterpret_cast<unsigned long long*>(&b)), "l"(*reinterpret_cast<unsigned long long*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}

// Four neighbouring entries in float32.
struct Pairs {
    float2 x, y;
    __device__ Pairs() {}
    __device__ explicit Pairs(const float* at) {
        const float4 v = *reinterpret_cast<const float4*>(at);
        x = make_float2(v.x, v.y);
        y = make_float2(v.z, v.w);
    }
    __device__ float4 four() const { return make_float4(x.x, x.y, y.x, y.y); }
    __device__ float largest() const { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))); }
    __device__ void clamp() {
        x = make_float2(kv_clamped(x.x), kv_clamped(x.y));
        y = make_float2(kv_clamped(y.x), kv_clamped(y.y));
    }
    __device__ uint32_t codes(float2 down) const {
        const float2 u = mul2(x, down), v = mul2(y, down);
        return kv_codes(u.x, u.y, v.x, v.y);
    }
};

// The same as they lie in memory.
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 v = {0.f, 0.f, 0.f, 0.f};
    __device__ void load(const float* at) { v = *reinterpret_cast<const float4*>(at); }
    __device__ Pairs pairs() const {
        Pairs r;
        r.x = make_float2(v.x, v.y);
        r.y = make_float2(v.z, v.w);
        return r;
    }
};
template <>
struct Four<bf16> {
    uint2 v = {0u, 0u};
    __device__ void load(const bf16* at) { v = *reinterpret_cast<const uint2*>(at); }
    __device__ Pairs pairs() const {
        Pairs r;
        r.x = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u));
        r.y = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
        return r;
    }
};

// LG neighbouring lanes hold a head, a lane two octets of it (octet i, i < rot / 8: four entries and the four that turn with them;
// behind those, eight neighbours), so that pairs never leave a thread, the mean of squares and the largest magnitude are shuffles
// among LG lanes, and accesses are of 8 or 16 bytes.  A thread keeps its head and its entries for a block's tokens, whose rows are
// loaded one ahead: weights, offsets and the kind of head are found out once.  Neither memory nor issue slots are full (304 instructions a warp and
// token take half of them, 18 warps an SM at 78 registers a thread, a row under way in each); fewer instructions a row were what helped, products two at a time
// and the root by an estimate and a step: 2,048 tokens of 36 normed heads of 128 13.7 -> 10.9 us (in the L2), 8,192 64 -> 38; what the bytes take: 5.5 and 22.
#define STORE_TOKENS 8
template <typename T, int LG>
__global__ void __launch_bounds__(512) norm_rotate_store_kernel(const StoreParams p, int most_tokens, int block_heads) {
    extern __shared__ float turn[];  // per token: cosines [rot / 2], sines and their opposites
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
    const T* row = (const T*)p.qkv + ((size_t)t0 * heads + head) * p.hd;
    Four<T> a_next[2], b_next[2];  // the row of the next token (of entries that there are not: zeros)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int octet = l + e * LG;
        there[e] = live && octet < (p.hd >> 3);
        turns[e] = octet < turning && !is_v;
        a_at[e] = octet < turning ? 4 * octet : p.rot + 8 * (octet - turning);
        b_at[e] = octet < turning ? half + 4 * octet : a_at[e] + 4;
    }
    auto load = [&]() {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (there[e]) {
                a_next[e].load(row + a_at[e]);
                b_next[e].load(row + b_at[e]);
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
        float sn;
        turn_of(p.positions[t0 + t], p.inv_freq[j], sn, turn[t * 3 * half + j]);
        turn[t * 3 * half + half + j] = sn;
        turn[t * 3 * half + 2 * half + j] = -sn;
    }
    const float* weight = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
    Pairs wa[2], wb[2];
    if (weight != nullptr)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (there[e]) {
                wa[e] = Pairs(weight + a_at[e]);
                wb[e] = Pairs(weight + b_at[e]);
            }
    const bool any_norm = __any_sync(0xffffffffu, live && weight != nullptr), any_kv = __any_sync(0xffffffffu, live && !is_q);
    const int kvh = is_v ? head - p.nh - p.nkv : head - p.nh;
    if (p.early) {
        pdl_wait();
        load();
    }
    __syncthreads();
    const float inv_hd = 1.f / (float)p.hd;
    T* q_to = (T*)p.q_out + ((size_t)t0 * p.nh + head) * p.hd;
#pragma unroll 1
    for (int t = 0; t < tokens; ++t) {
        Pairs a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            a[e] = a_next[e].pairs();
            b[e] = b_next[e].pairs();
        }
        if (t + 1 < tokens) load();
        if (any_norm) {
            float2 sums = mul2(a[0].x, a[0].x);
            sums = fma2(a[0].y, a[0].y, sums);
            float2 more = mul2(b[0].x, b[0].x);
            more = fma2(b[0].y, b[0].y, more);
            sums = fma2(a[1].x, a[1].x, sums);
            more = fma2(b[1].x, b[1].x, more);
            sums = fma2(a[1].y, a[1].y, sums);
            more = fma2(b[1].y, b[1].y, more);
            float sum = (sums.x + sums.y) + (more.x + more.y);
#pragma unroll
            for (int o = LG / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (weight != nullptr) {
                // 1 / sqrt by an estimate (off by two last places at most) and a step of Newton's, which leaves less than one
                const float mean = fmaf(sum, inv_hd, p.eps), y = rsqrtf(mean), z = mean * y, nearer = fmaf(0.5f * y, fmaf(-z, y, 1.f), y);
                const float r = z - z == 0.f ? nearer : y;  // (means of 0 and infinity)
                const float2 rr = make_float2(r, r);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    a[e].x = mul2(a[e].x, mul2(rr, wa[e].x)); a[e].y = mul2(a[e].y, mul2(rr, wa[e].y));
                    b[e].x = mul2(b[e].x, mul2(rr, wb[e].x)); b[e].y = mul2(b[e].y, mul2(rr, wb[e].y));
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (turns[e]) {
                const float* at = turn + t * 3 * half + a_at[e];
                const Pairs cs(at), sn(at + half), minus(at + 2 * half), x = a[e], y = b[e];
                a[e].x = fma2(x.x, cs.x, mul2(y.x, minus.x)); a[e].y = fma2(x.y, cs.y, mul2(y.y, minus.y));
                b[e].x = fma2(y.x, cs.x, mul2(x.x, sn.x)); b[e].y = fma2(y.y, cs.y, mul2(x.y, sn.y));
            }
        if (live && is_q) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (there[e]) {
                    Vec4<T>::store(q_to + a_at[e], a[e].four());
                    Vec4<T>::store(q_to + b_at[e], b[e].four());
                }
        }
        q_to += (size_t)p.nh * p.hd;
        if (!any_kv) continue;
        const int slot = slot_s[t];
        const bool stores = live && !is_q && slot >= 0;
        const size_t at = ((size_t)max(slot, 0) * p.nkv + kvh) * p.hd;
        if (p.k_exp == nullptr) {  // rows of the run's type
            T* out = (T*)(is_v ? p.v_cache : p.k_cache) + at;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (stores && there[e]) {
                    Vec4<T>::store(out + a_at[e], a[e].four());
                    Vec4<T>::store(out + b_at[e], b[e].four());
                }
            continue;
        }
        float big = 0.f;  // (NaN has no say)
#pragma unroll
        for (int e = 0; e < 2; ++e) big = fmaxf(big, fmaxf(a[e].largest(), b[e].largest()));
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        if (big > KV_BIGGEST) {
            big = KV_BIGGEST;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[e].clamp();
                b[e].clamp();
            }
        }
        if (stores) {
            const int power = kv_power(big), off = off_s[t];
            const float2 down = make_float2(kv_down(power), kv_down(power));
            uint8_t* out = (uint8_t*)(is_v ? p.v_cache : p.k_cache) + at;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (there[e]) {
                    *reinterpret_cast<uint32_t*>(out + a_at[e]) = a[e].codes(down);
                    *reinterpret_cast<uint32_t*>(out + b_at[e]) = b[e].codes(down);
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
    // tokens of a block: as many as end soonest, if a round of the blocks that fit on the SMs (80 registers a thread) takes what two
    // tokens and each of its tokens do
    const int threads = (block_heads * lg + 31) / 32 * 32, resident = 148 * max(1, 65536 / 80 / threads);
    int tokens = 1;
    long long least = 1LL << 62;
    for (int t = 1; t <= STORE_TOKENS; ++t) {
        const long long blocks = (long long)((N + t - 1) / t) * chunks, cost = (blocks + resident - 1) / resident * (t + 2);
        if (cost < least) {
            least = cost;
            tokens = t;
        }
    }
    const dim3 grid((N + tokens - 1) / tokens, chunks), block(threads);
    const size_t room = (size_t)tokens * smem / 2 * 3;
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

// The requests' work, cut evenly over the blocks of a grid: request s brings units(s) units, numbered through all requests;
// block b owns units [b * quota, (b + 1) * quota), quota = ceil(total / blocks), at least `least`.  Every block works this out
// from the lengths on the device (so that a captured launch follows them).  Where there are fewer units than the grid has warps each
// is cut into up to `most_parts`, units of their own.  All threads of the block call it; `sh`: 36 words of shared memory, free
// again after a barrier of the caller's.
struct UnitRange {
    int total, quota;
    int parts;           // of a unit
    int first, last;     // this block's units [first, last)
    int request, offset; // where unit `first` lies: request and unit within it
};
template <class F>
__device__ __forceinline__ UnitRange units_of_block(F units, int requests, int least, int most_parts, int blocks, int block, int* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    UnitRange r;
    int sum = 0;
    const int mine = threadIdx.x < requests ? units(threadIdx.x) : 0;  // (looked up once where a thread per request suffices)
    sum = mine;
    for (int s = threadIdx.x + blockDim.x; s < requests; s += blockDim.x) sum += units(s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh[warp] = sum;
    __syncthreads();
    r.total = 0;
    for (int w = 0; w < warps; ++w) r.total += sh[w];
    r.parts = max(1, min(most_parts, blocks * warps / max(r.total, 1)));
    r.total *= r.parts;
    r.quota = max(least, (r.total + blocks - 1) / blocks);
    r.first = (int)min((long long)block * r.quota, (long long)r.total);
    r.last = min(r.total, r.first + r.quota);
    r.request = r.offset = 0;
    if (r.first >= r.last) return r;
    int base = 0;
    for (int s0 = 0; s0 < requests; s0 += blockDim.x) {
        const int s = s0 + threadIdx.x;
        const int n = (s0 == 0 ? mine : s < requests ? units(s) : 0) * r.parts;
        int upto = n;  // units of this chunk's requests up to and with s
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();  // (the words of the round before are read)
        if (lane == 31) sh[warp] = upto;
        if (threadIdx.x == 0) sh[32] = -1;
        __syncthreads();
        int before = base, chunk = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) before += sh[w];
            chunk += sh[w];
        }
        const int from = before + upto - n;
        if (from <= r.first && r.first < from + n) {
            sh[32] = s;
            sh[33] = r.first - from;
        }
        __syncthreads();
        if (sh[32] >= 0) {
            r.request = sh[32];
            r.offset = sh[33];
            break;
        }
        base += chunk;
    }
    return r;
}

struct ReadParams {
    const uint8_t* k; const uint8_t* v; const uint8_t* k_exp; const uint8_t* v_exp;
    void* k_out; void* v_out;
    const int* block_tables; const int* ctx_lens; const int* q_start;
    int requests, nkv, hd, page_size, max_blocks, num_pages, window, least_rows;
    int behind_zeros;  // zero_rests_kernel is the kernel in front
    int* status;
};

// The blocks of request s that are read: how many, and the first.
__device__ __forceinline__ int read_span(const ReadParams& p, int s, int& from) {
    int ctx = p.ctx_lens[s], first = ctx;
    if (p.q_start != nullptr) {
        const int rows = p.q_start[s + 1] - p.q_start[s];
        if (rows < p.least_rows) return 0;
        first = ctx - rows + 1;  // (a portion's first row sees `window` keys, its own among them: the window reaches back from there)
    }
    from = p.window > 0 ? max(0, first - p.window) / p.page_size : 0;
    return max(0, min((ctx + p.page_size - 1) / p.page_size, p.max_blocks) - from);
}

// Zeros behind the last token of every request that is read, to the end of its last page.  Requests may share a page of which one
// holds more than the other (a table may also name a page twice), so these come before any value is written, in a kernel of their own: the
// rows that a request holds are then written by read_pages_kernel whoever's zeros lay there, with the same numbers by all who hold them.
// (That kernel's set-up runs beside this one: 5,778 tokens of two KV heads 5.8 us for both, 6.8 with the zeros in its own pages' units.)
template <typename T>
__global__ void __launch_bounds__(256) zero_rests_kernel(const ReadParams p) {
    pdl_enter();
    const int s = blockIdx.x;
    int from = 0;
    const int n = read_span(p, s, from);
    if (n == 0) return;
    const int block = from + n - 1, page = p.block_tables[(size_t)s * p.max_blocks + block], live = p.ctx_lens[s] - block * p.page_size;
    if (page < 0 || page >= p.num_pages || live >= p.page_size) return;  // (reported by read_pages_kernel)
    const int row_words = p.nkv * (p.hd * (int)sizeof(T) / 16);
    uint4* to = reinterpret_cast<uint4*>(blockIdx.y ? p.v_out : p.k_out) + (size_t)page * p.page_size * row_words;
    for (int i = live * row_words + threadIdx.x; i < p.page_size * row_words; i += blockDim.x) to[i] = make_uint4(0, 0, 0, 0);
}

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

// Units are pages of a request, keys and values apart, a warp to each, so that thousands are on their way at once; where there are few,
// parts of a page that a warp reads in one go (5,778 tokens of two KV heads of 128 8.3 -> 6.7 us, now 5.8, 16,000 of eight 26.9 -> 18.4).  A page's codes
// are one run of memory, and so is where they go; a lane takes 8 codes at a time (they share a row and its power), so that a
// warp writes whole lines.
#define READ_AT_ONCE 8
template <typename T>
__global__ void __launch_bounds__(256) read_pages_kernel(const ReadParams p, const Quotient by_chunks, const Quotient by_heads) {
    __shared__ int sh[36];
    // (the kernel of zeros lets this one come when all in front of it is complete: the lengths can be looked at beside it)
    if (!p.behind_zeros) pdl_enter();
    auto span = [&](int s, int& from) { return read_span(p, s, from); };
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    const int chunks = p.page_size * p.nkv * (p.hd >> 3), at_once = 32 * READ_AT_ONCE;
    const UnitRange r = units_of_block([&](int s) { int from; return 2 * span(s, from); }, p.requests, warps, (chunks + at_once - 1) / at_once,
                                       gridDim.x, blockIdx.x, sh);
    if (p.behind_zeros) pdl_enter();
    int s = r.request, at = r.offset + (threadIdx.x >> 5);  // units of a block go to its warps in turn
    for (int u = r.first + (threadIdx.x >> 5); u < r.last; u += warps, at += warps) {
        int from = 0, n = 2 * r.parts * span(s, from);
        while (at >= n && s + 1 < p.requests) {
            at -= n;
            n = 2 * r.parts * span(++s, from);
        }
        const int plane = at / r.parts, part = at - plane * r.parts;
        const bool is_v = plane & 1;
        const int block = from + (plane >> 1), page = block < p.max_blocks ? p.block_tables[(size_t)s * p.max_blocks + block] : -1;
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) cw_report(p.status, CW_ST_PAGE_RANGE, s, page);
            continue;
        }
        const uint2* src = reinterpret_cast<const uint2*>(is_v ? p.v : p.k) + (size_t)page * chunks;
        const uint8_t* powers = (is_v ? p.v_exp : p.k_exp) + (size_t)page * p.nkv * p.page_size;
        T* dst = (T*)(is_v ? p.v_out : p.k_out) + (size_t)page * chunks * 8;
        const int live = min(p.page_size, p.ctx_lens[s] - block * p.page_size) * p.nkv;  // rows that hold something
        for (int i0 = part * at_once + lane; i0 < chunks; i0 += r.parts * at_once) {
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
                if (i >= chunks || (int)by_chunks.of(i) >= live) break;
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
                          max_blocks, num_pages, window, least_rows, page_size > 1, status};
    if (dtype != 0 && dtype != 1) return CW_ERR_BAD_DTYPE;
    if (p.behind_zeros) {
        const int result = dtype == 0 ? cw_launch(zero_rests_kernel<float>, dim3(requests, 2), dim3(256), 0, stream, 1u, p)
                                      : cw_launch(zero_rests_kernel<bf16>, dim3(requests, 2), dim3(256), 0, stream, 1u, p);
        if (result != CW_OK) return result;
    }
    const Quotient by_chunks = Quotient::by(hd >> 3), by_heads = Quotient::by(nkv);
    if (dtype == 0) return cw_launch(read_pages_kernel<float>, dim3(blocks), dim3(256), 0, stream, 1u, p, by_chunks, by_heads);
    return cw_launch(read_pages_kernel<bf16>, dim3(blocks), dim3(256), 0, stream, 1u, p, by_chunks, by_heads);
}

CW_TRACE_TU(kv_e4m3)
