// Shared device helpers of the operators between a Mamba block's projections (causal_conv.cu, selective_scan.cu, block_norm.cu): vectors of
// channels in the three activation types, and the exponential functions in float32.
#pragma once
#include "row_stream.cuh"

namespace el {
namespace mamba {

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V values of a row as they lie in memory, and as pairs of float32.  ALIGNED: adjacent ones in one or two vector accesses (the host has
// checked base, strides and that V divides the row).  Otherwise every STRIDE-th one by itself, STRIDE the number of threads side by side,
// so that neighbouring threads still read neighbouring values; `valid` is the distance from the first to the row's end, zeros behind it.
// Held as 32-bit words: registers, whatever T is.
template <typename T, int V> struct alignas(V * sizeof(T) < 16 ? 8 : 16) Vec { uint32_t w[V * sizeof(T) / 4]; };
template <typename T> __device__ __forceinline__ uint32_t bits_of(T v) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(v);
    else return *reinterpret_cast<const unsigned short*>(&v);
}
template <typename T, int V> __device__ __forceinline__ Vec<T, V> zeros() {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) r.w[i] = 0u;
    return r;
}
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ Vec<T, V> fetch(const T* p, int valid, int stride) {
    constexpr int WORDS = V * sizeof(T) / 4;
    Vec<T, V> r = zeros<T, V>();
    if constexpr (ALIGNED && WORDS == 2) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        r.w[0] = a.x; r.w[1] = a.y;
    } else if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 a = reinterpret_cast<const uint4*>(p)[i / 4];
            r.w[i] = a.x; r.w[i + 1] = a.y; r.w[i + 2] = a.z; r.w[i + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t b = j * stride < valid ? bits_of<T>(p[j * stride]) : 0u;
            if constexpr (sizeof(T) == 4) r.w[j] = b;
            else r.w[j / 2] |= b << (16 * (j & 1));
        }
    }
    return r;
}
template <typename T> __device__ __forceinline__ rowio::f32x2 widen_word(uint32_t w) {            // of a 16-bit type
    if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        return rowio::pair(f.x, f.y);
    } else {
        return rowio::pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
}
template <typename T, int V> __device__ __forceinline__ void widen(const Vec<T, V>& r, rowio::f32x2 v[V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = rowio::pair(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
        else v[i] = widen_word<T>(r.w[i]);
    }
}
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void put(T* p, int valid, int stride, const rowio::f32x2 v[V / 2]) {       // rounds to T
    constexpr int WORDS = V * sizeof(T) / 4;
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float a = rowio::lo_of(v[i]), b = rowio::hi_of(v[i]);
        if constexpr (sizeof(T) == 4) {
            w[2 * i] = __float_as_uint(a);
            w[2 * i + 1] = __float_as_uint(b);
        } else {
            w[i] = std::is_same<T, __half>::value ? pack_f16x2(a, b) : pack_bf16x2(a, b);
        }
    }
    if constexpr (ALIGNED && WORDS == 2) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j * stride >= valid) continue;
            if constexpr (sizeof(T) == 4) {
                p[j * stride] = __uint_as_float(w[j]);
            } else {
                const unsigned short h = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
                p[j * stride] = *reinterpret_cast<const T*>(&h);
            }
        }
    }
}
__device__ __forceinline__ rowio::f32x2 both(float v) { return rowio::pair(v, v); }

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
        alignas(16) T v[4];
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
template <typename T> __device__ __forceinline__ void store_quad(T* p, int valid, bool aligned, float4 v) {
    const rowio::f32x2 f[2] = {rowio::pair(v.x, v.y), rowio::pair(v.z, v.w)};
    if (!aligned) put<T, 4, false>(p, valid, 1, f);
    else if (valid > 0) put<T, 4, true>(p, valid, 1, f);
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

// e^-|x|, to a relative error of 2.4e-7 + 7.3e-8 |x|: the product with log2(e), rounded to float32, and log2(e) itself are what |x| counts in.
// Results below 2^-126 are kept: a step size of that magnitude still carries a gradient.
__device__ __forceinline__ float exp_minus_abs(float x) { return ex2_denormals(__fmul_rn(-fabsf(x), LOG2E)); }
// 1 / (1 + e^-x), small results as exact as e^-|x| above; an exponential that overflows gives 0
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.0f + ex2(__fmul_rn(x, -LOG2E))); }
__device__ __forceinline__ rowio::f32x2 sigmoid2(rowio::f32x2 x) {
    using namespace rowio;
    const f32x2 t = mul2(x, both(-LOG2E)), d = add2(pair(ex2(lo_of(t)), ex2(hi_of(t))), both(1.0f));
    return pair(rcp(lo_of(d)), rcp(hi_of(d)));
}
// 1 / (1 + e^-x) from e = e^-|x|; a small result is as exact as e
__device__ __forceinline__ float sigmoid_of(float x, float e) {
    const float r = rcp(1.0f + e);
    return x < 0.0f ? __fmul_rn(e, r) : r;
}
// d/dx of x sigmoid(x), from s = sigmoid(x)
__device__ __forceinline__ rowio::f32x2 silu_slope2(rowio::f32x2 x, rowio::f32x2 s) {
    using namespace rowio;
    return mul2(s, fma2(x, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
}

// log(1 + e^x) from e = e^-|x|: max(x, 0) + log1p(e), log1p(e) = 2 artanh(s) = 2 (s + s^3/3 + s^5/5 + ..), s = e / (2 + e) <= 1/3; the
// first term left out is s^15/15, 1.4e-8 of the whole at most.  The logarithm of 1 + e in float32 would have an absolute error of 6e-8,
// which is large against the step sizes of 0.001 that a model has.  Relative error 4.1e-7 beside e's.  Two values at a time: half the instructions.
__device__ __forceinline__ rowio::f32x2 softplus2(float x0, float x1, float e0, float e1) {
    using namespace rowio;
    const f32x2 e = pair(e0, e1), d = add2(e, pair(2.0f, 2.0f));
    const f32x2 s = mul2(e, pair(rcp(lo_of(d)), rcp(hi_of(d)))), q = mul2(s, s);
    f32x2 p = fma2(q, both(1.0f / 13.0f), both(1.0f / 11.0f));
    p = fma2(p, q, both(1.0f / 9.0f));
    p = fma2(p, q, both(1.0f / 7.0f));
    p = fma2(p, q, both(1.0f / 5.0f));
    p = fma2(p, q, both(1.0f / 3.0f));
    const f32x2 s2 = add2(s, s);
    return add2(pair(max_nan(x0, 0.0f), max_nan(x1, 0.0f)), fma2(s2, mul2(p, q), s2));
}
__device__ __forceinline__ float softplus_of(float x, float e) { return rowio::lo_of(softplus2(x, x, e, e)); }

// out[map(i)] = sum of the parts' i-th values, for `cols` of them.  A block covers 32 columns; its W warps each add every W-th part in order, and
// the first warp adds their results in order: the same bits for a given width.  Few columns take 32 warps: there the chain of loads counts.
template <typename F>
__global__ void __launch_bounds__(1024)
column_sums_kernel(const float* __restrict__ partial, int n_parts, int cols, F store_at) {
    __shared__ float part[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int k = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (k < cols) {
#pragma unroll 8
        for (int p = warp; p < n_parts; p += warps) s += partial[(long long)p * cols + k];
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && k < cols) {
        s = 0.0f;
        for (int w = 0; w < warps; ++w) s += part[w][lane];
        store_at(k, s);
    }
}
template <typename F> static int launch_column_sums(const float* partial, int n_parts, int cols, F store_at, cudaStream_t st) {
    int sms = 148;
    device_sm_count(&sms);
    const int blocks = (cols + 31) / 32;
    column_sums_kernel<<<blocks, blocks <= 2 * sms && n_parts > 64 ? 1024 : 256, 0, st>>>(partial, n_parts, cols, store_at);
    return check_launch();
}

}  // namespace mamba
}  // namespace el
