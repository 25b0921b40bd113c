// Attention of one new token per request over an 8-bit cache (kv_e4m3.cuh), through block tables.
//
//     s_j = scale * 2^(Ek_j - 127) * sum_d q_d kcode_jd,   out = sum_j e^(s_j - m) 2^(Ev_j - 127) vcode_j / sum_j e^(s_j - m)
//
// over the context's positions j (the last `window` of them), m their largest s_j; float32 throughout.
#include "kv_e4m3.cuh"

struct DecodeE4m3Params {
    const void* q; int q_stride; void* out;
    const uint8_t* k; const uint8_t* v; const uint8_t* k_exp; const uint8_t* v_exp;
    const int* block_tables; const int* ctx_lens; const int* q_start;
    int requests, nh, nkv, hd, page_size, max_blocks, num_pages, window;
    float scale;
    int* status;
};

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

// q [rows, q_stride >= nh * hd], out [rows, nh * hd]; request s owns row s, or with q_start rows q_start[s] .. q_start[s + 1], and
// then only requests with one row are served.  A context of length 0 gives zeros.
extern "C" int cw_attention_decode_e4m3(const void* q, int q_stride, void* out, const uint8_t* k, const uint8_t* v, const uint8_t* k_exp,
                                        const uint8_t* v_exp, const int* block_tables, const int* ctx_lens, const int* q_start,
                                        int requests, int nh, int nkv, int hd, int page_size, int max_blocks, int num_pages, int window,
                                        float scale, int dtype, int* status, cudaStream_t stream) {
    if (requests == 0) return CW_OK;
    if (requests < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || hd % 16 || hd > 256 || page_size <= 0 || max_blocks <= 0 ||
        num_pages <= 0 || window < 0 || q_stride < nh * hd || ((uintptr_t)k | (uintptr_t)v) % 16 || requests > 65535 ||
        (long long)num_pages * page_size > 0x7FFFFFFF || (long long)max_blocks * page_size > 0x7FFFFFFF)
        return CW_ERR_BAD_SIZE;
    const DecodeE4m3Params p = {q, q_stride, out, k, v, k_exp, v_exp, block_tables, ctx_lens, q_start, requests, nh, nkv, hd, page_size,
                                max_blocks, num_pages, window, scale, status};
    if (dtype == 0) return cw_launch(decode_e4m3_any_kernel<float>, dim3(nh, requests), dim3(ANY_TOKENS), 0, stream, 1u, p);
    if (dtype == 1) return cw_launch(decode_e4m3_any_kernel<bf16>, dim3(nh, requests), dim3(ANY_TOKENS), 0, stream, 1u, p);
    return CW_ERR_BAD_DTYPE;
}

CW_TRACE_TU(attention_decode_e4m3)
