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
// Four channels (or states) as they lie in memory, for values that are fetched long before they are used; elements from `valid` on are zeros.
template <typename T> __device__ __forceinline__ rowio::Quad<T> quad_zero() {
    rowio::Quad<T> q;
    if constexpr (sizeof(T) == 4) q.a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    else q.a = make_uint2(0u, 0u);
    return q;
}
template <typename T> __device__ __forceinline__ rowio::Quad<T> fetch_quad(const T* p, int valid, bool aligned) {
    rowio::Quad<T> q = quad_zero<T>();
    if (valid <= 0) return q;
    if (aligned) {
        q.a = *reinterpret_cast<const decltype(q.a)*>(p);
    } else {
        T v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < valid ? p[j] : T(0.0f);
        q = *reinterpret_cast<const rowio::Quad<T>*>(v);
    }
    return q;
}
template <typename T> __device__ __forceinline__ float4 widen(const rowio::Quad<T>& q) {
    rowio::f32x2 v[2];
    rowio::unpack2<T>(q, v);
    return make_float4(rowio::lo_of(v[0]), rowio::hi_of(v[0]), rowio::lo_of(v[1]), rowio::hi_of(v[1]));
}
template <typename T> __device__ __forceinline__ void store_quad(T* p, int valid, bool aligned, float4 v);

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

template <typename T> __device__ __forceinline__ void store_quad(T* p, int valid, bool aligned, float4 v) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    if (aligned && valid > 0) store<T, 4, true>(p, 4, f);
    else store<T, 4, false>(p, valid, f);
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

// e^-|x|.  Results below 2^-126 are kept: a step size of that magnitude still carries a gradient.
__device__ __forceinline__ float exp_minus_abs(float x) { return ex2_denormals(__fmul_rn(-fabsf(x), LOG2E)); }
// 1 / (1 + e^-x); an exponential that overflows gives 0
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.0f + ex2(__fmul_rn(x, -LOG2E))); }
// 1 / (1 + e^-x) from e = e^-|x|, with all the digits of a small result
__device__ __forceinline__ float sigmoid_of(float x, float e) {
    const float r = rcp(1.0f + e);
    return x < 0.0f ? __fmul_rn(e, r) : r;
}
// d/dx of x sigmoid(x), from s = sigmoid(x)
__device__ __forceinline__ float silu_slope(float x, float s) { return __fmul_rn(s, __fmaf_rn(x, 1.0f - s, 1.0f)); }

// log(1 + e^x) from e = e^-|x|: max(x, 0) + log1p(e), log1p(e) = 2 artanh(s) = 2 (s + s^3/3 + s^5/5 + ..), s = e / (2 + e) <= 1/3; the
// first term left out is s^15/15, 1.4e-8 of the whole at most.  The logarithm of 1 + e in float32 would have an absolute error of 6e-8,
// which is large against the step sizes of 0.001 that a model has.  Two values at a time: half the instructions.
__device__ __forceinline__ rowio::f32x2 softplus2(float x0, float x1, float e0, float e1) {
    using namespace rowio;
    const f32x2 e = pair(e0, e1), d = add2(e, pair(2.0f, 2.0f));
    const f32x2 s = mul2(e, pair(rcp(lo_of(d)), rcp(hi_of(d)))), q = mul2(s, s);
    auto both = [](float v) { return pair(v, v); };
    f32x2 p = fma2(q, both(1.0f / 13.0f), both(1.0f / 11.0f));
    p = fma2(p, q, both(1.0f / 9.0f));
    p = fma2(p, q, both(1.0f / 7.0f));
    p = fma2(p, q, both(1.0f / 5.0f));
    p = fma2(p, q, both(1.0f / 3.0f));
    const f32x2 s2 = add2(s, s);
    return add2(pair(max_nan(x0, 0.0f), max_nan(x1, 0.0f)), fma2(s2, mul2(p, q), s2));
}
__device__ __forceinline__ float softplus_of(float x, float e) { return rowio::lo_of(softplus2(x, x, e, e)); }

}  // namespace mamba
}  // namespace el
