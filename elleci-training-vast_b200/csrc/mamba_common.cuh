// Shared device helpers of the operators between a Mamba block's projections (causal_conv.cu, selective_scan.cu, block_norm.cu): vectors of
// channels in the three activation types, and the exponential functions in float32.
#pragma once
#include "row_stream.cuh"

namespace el {
namespace mamba {

// V consecutive channels of a token as float32.  ALIGNED: one or two vector accesses (the host has checked base, strides and that V
// divides the channels); otherwise element by element, the first `valid` of them, zeros behind.
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void load(const T* p, int valid, float v[V]) {
    static_assert(V == 4 || V == 8, "vectors of 4 or 8 channels");
    if constexpr (!ALIGNED) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < valid ? to_float<T>(p[j]) : 0.0f;
    } else if constexpr (V == 8) {
        rowio::Io<T>::load8(p, v);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        rowio::Quad<T> q;
        q.a = *reinterpret_cast<const uint2*>(p);
        rowio::f32x2 w[2];
        rowio::unpack2<T>(q, w);
        v[0] = rowio::lo_of(w[0]); v[1] = rowio::hi_of(w[0]); v[2] = rowio::lo_of(w[1]); v[3] = rowio::hi_of(w[1]);
    }
}
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void store(T* p, int valid, const float v[V]) {
    if constexpr (!ALIGNED) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < valid) p[j] = from_float<T>(v[j]);
    } else if constexpr (V == 8) {
        rowio::Io<T>::store8(p, v);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        *reinterpret_cast<uint2*>(p) = rowio::pack2<T>(rowio::pair(v[0], v[1]), rowio::pair(v[2], v[3])).a;
    }
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float ex2_denormals(float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

// the larger of the two, NaN if either is one
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// e^-|x|: 2^t at t = -|x| log2(e) rounded, times 1 + ln(2) (-|x| log2(e) - t); without the second factor the rounding of t alone costs |t| 2^-24.
// Results below 2^-126 are kept: a step size of that magnitude still carries a gradient.
__device__ __forceinline__ float exp_minus_abs(float x) {
    x = max_nan(-fabsf(x), -150.0f);                   // 2^-216 is 0 in float32 and the remainder stays finite
    const float t = __fmul_rn(x, LOG2E);
    const float r = __fmaf_rn(x, 1.92596299e-8f, __fmaf_rn(x, LOG2E, -t));       // log2(e) = LOG2E + 1.92596299e-8
    const float e = ex2_denormals(t);
    return __fmaf_rn(e, __fmul_rn(r, LN2), e);
}
// 1 / (1 + e^-x) from e = e^-|x|
__device__ __forceinline__ float sigmoid_of(float x, float e) {
    const float r = rcp(1.0f + e);
    return x < 0.0f ? __fmul_rn(e, r) : r;
}
__device__ __forceinline__ float sigmoid(float x) { return sigmoid_of(x, exp_minus_abs(x)); }
// d/dx of x sigmoid(x), from s = sigmoid(x)
__device__ __forceinline__ float silu_slope(float x, float s) { return __fmul_rn(s, __fmaf_rn(x, 1.0f - s, 1.0f)); }

// log(1 + e^x) from e = e^-|x|: max(x, 0) + log1p(e), log1p(e) = 2 artanh(s) = 2 (s + s^3/3 + s^5/5 + ..), s = e / (2 + e) <= 1/3; the
// first term left out is s^15/15, 1.4e-8 of the whole at most.  The logarithm of 1 + e in float32 would have an absolute error of 6e-8,
// which is large against the step sizes of 0.001 that a model has.
__device__ __forceinline__ float softplus_of(float x, float e) {
    const float s = __fmul_rn(e, rcp(2.0f + e)), q = __fmul_rn(s, s);
    float p = __fmaf_rn(q, 1.0f / 13.0f, 1.0f / 11.0f);
    p = __fmaf_rn(p, q, 1.0f / 9.0f);
    p = __fmaf_rn(p, q, 1.0f / 7.0f);
    p = __fmaf_rn(p, q, 1.0f / 5.0f);
    p = __fmaf_rn(p, q, 1.0f / 3.0f);
    const float s2 = 2.0f * s;
    return max_nan(x, 0.0f) + __fmaf_rn(s2, __fmul_rn(p, q), s2);
}

}  // namespace mamba
}  // namespace el
