// kv_cache.cuh — what the kernels of the paged 8-bit cache share: the batch
// on the device, page scales, e4m3 codes, 8-channel row pieces.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b3_internal.h"

namespace b3 {

constexpr int kScaleExpLo = -40, kScaleExpHi = 40;   // 2^e of a page's scale
constexpr int64_t kMostTokens = 0x7fffffff - 1023;   // of a sequence

// Checks of b3_kv_cache / b3_kv_batch that the host can make (kv_append.cu).
int kv_check(const b3_kv_cache* c, const b3_kv_batch* b);

__device__ __forceinline__ void kv_flag(int32_t* status, int bit) {
    if (status) atomicOr(status, bit);
}

// The last b in [0, n) with key(b) <= t, for a non-decreasing key with
// key(0) <= t: a 33-way search by one warp (two rounds cover 1024 sequences,
// each one load latency).  Any contents of the array keep b within [0, n).
template <typename Key>
__device__ __forceinline__ int kv_search(Key key, int n, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 31) >> 5;
        const int at = lane * step;
        const bool le = at < len && key(lo + at) <= t;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        const int k = m ? (31 - __clz(m)) * step : 0;
        lo += k;
        len = min(step, len - k);
    }
    return lo;
}

// The sequence of token t (0 <= t < tokens).  A batch with one new token for
// each sequence is recognised by two loads.
__device__ __forceinline__ int kv_seq_of(const b3_kv_batch& b, int t) {
    if (b.n_seq == b.tokens && __ldg(b.cu_q + t) == t && __ldg(b.cu_q + t + 1) == t + 1) return t;
    return kv_search([&](int i) { return __ldg(b.cu_q + i); }, b.n_seq, t);
}

// The least e with amax <= 448 * 2^e, clamped to the range of a page's scale.
__device__ __forceinline__ int scale_exp(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = static_cast<int>(bits >> 23) - 126 - 9 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(e, kScaleExpLo), kScaleExpHi);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Exponent of a page's scale as stored (a power of two; anything else, as in
// a page that was never written, is brought into the range).
__device__ __forceinline__ int stored_exp(float scale) {
    const int e = static_cast<int>((__float_as_uint(scale) >> 23) & 0xff) - 127;
    return min(max(e, kScaleExpLo), kScaleExpHi);
}

// Magnitude of x if finite, else 0: infinities and NaN have no say in a scale.
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}

// Eight e4m3 codes (round to nearest even, saturating, NaN stays NaN).
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv_scale) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * inv_scale, x[2 * i + 1] * inv_scale), __NV_SATFINITE,
                                        __NV_E4M3);
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

__device__ __forceinline__ __half2 decode2(uint32_t two) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two), __NV_E4M3));
}

__device__ __forceinline__ void decode8(uint2 c, float (&x)[8]) {
    const uint32_t w[4] = {c.x & 0xffffu, c.x >> 16, c.y & 0xffffu, c.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(decode2(w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float x, float& y) { y = x; }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

// Eight consecutive channels.  VEC: the address is 16-byte aligned.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    T v[8];
    if (VEC) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {   // p is 16-byte aligned
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) from_f32(x[i], v[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(v);
}

}  // namespace b3
