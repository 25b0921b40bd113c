// The 8-bit form of cached keys and values.  A row (one token's key or value in one KV head) is `hd` e4m3 codes and one byte E;
// entry = code * 2^(E - 127).  E is the smallest, from 3 on, that keeps the row's largest magnitude within 448, e4m3's largest
// number: a power of two, so that scaling is exact in both directions (the code's 4 bits are the only rounding, at most half a
// step, 2^-4 of an entry that is no subnormal code), every held entry is a bfloat16 number, and the tensor cores can multiply
// codes and leave the powers to float32.  Magnitudes beyond 1.875 * 2^127 are held as that (infinities too: the largest number
// whose code times its power is finite); a NaN entry is held as NaN and has no say in E; a row of zeros has E = 127.
//
// Codes lie like the plain cache, [pages, page_size, nkv, hd]; the powers [pages, nkv, page_size], so that those of a head's
// tokens in a page are neighbours.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <string.h>
#include "common.cuh"

// Arguments of an entry point as one block of 8-byte words, read in order.  Whole numbers that no int holds become -1, which every
// entry point refuses as a size.
struct ArgumentWords {
    const char* at;
    explicit ArgumentWords(const char* block) : at(block) {}
    template <typename T>
    T next() {
        T x;
        memcpy(&x, at, sizeof(T));
        at += sizeof(T);
        return x;
    }
    void* pointer() { return (void*)next<uint64_t>(); }
    int number() {
        const long long x = next<long long>();
        return x < -1 || x > 0x7FFFFFFF ? -1 : (int)x;
    }
    double real() { return next<double>(); }
};

#define KV_BIGGEST __int_as_float(0x7F700000)  // 1.875 * 2^127

// NaN passes through (fminf and fmaxf would drop it)
__device__ __forceinline__ float kv_clamped(float x) { return fabsf(x) > KV_BIGGEST ? copysignf(KV_BIGGEST, x) : x; }

// E for the largest magnitude of a row (0 <= big <= KV_BIGGEST)
__device__ __forceinline__ int kv_power(float big) {
    const uint32_t bits = __float_as_uint(big);
    if (bits == 0) return 127;
    return max(3, (int)(bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000 ? 1 : 0));  // 448 = 1.75 * 2^8
}
__device__ __forceinline__ float kv_down(int power) { return __int_as_float((254 - power) << 23); }  // 2^(127 - E): to codes
__device__ __forceinline__ float kv_up(int power) { return __int_as_float(power << 23); }            // 2^(E - 127) (E = 0: 0)

// four numbers, already divided by the row's power, as four codes
__device__ __forceinline__ uint32_t kv_codes(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// two codes as two half-precision numbers (exact: the format's 4 exponent and 3 fraction bits fit)
__device__ __forceinline__ uint32_t kv_half2(uint32_t codes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
    return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ float2 kv_float2(uint32_t codes) {
    const uint32_t h = kv_half2(codes & 0xFFFF);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
