// The norm after a block, its gate and residual scale, the residual addition and the norm before the next block, in one pass.
//
//   p = w1 y r1,  r1 = 1/sqrt(mean y^2 + eps);   h' = h + s sigmoid(g) p;   n = w2 h' r2,  r2 = 1/sqrt(mean h'^2 + eps)
// backward (yn = y r1, hn = h' r2, both formed again from the inputs):
//   dh = dh' + r2 (dn w2 - hn mean(dn w2 hn));  dw2 = sum dn hn;  ds = sum dh sigmoid(g) p;  dg = dh s p sigmoid'(g)
//   dp = dh s sigmoid(g);  dw1 = sum dp yn;  dy = r1 (dp w1 - yn mean(dp w1 yn))
// The second mean is linear in the first one, c2: with q = s sigmoid(g) w1 yn it is mean((dh' + r2 dn w2) q) - c2 r2 mean(hn q), so that a row's
// three sums are taken together, behind one barrier.
// Row sums in float32: a thread adds 8 to 32 squares, the block adds the threads' in a fixed order.
//
// Blocks walk over the rows; a thread owns the same vectors of 8 columns in each.  Bound: memory, 5 values read or written per column forward, 8
// backward, if enough rows are on their way: the next row's values are fetched before this one's two sums over the block.
#include "mamba_common.cuh"

namespace el {
using namespace mamba;
using rowio::add2;
using rowio::f32x2;
using rowio::fma2;
using rowio::hi_of;
using rowio::lo_of;
using rowio::mul2;
using rowio::pair;

constexpr int NORM_MAX_WARPS = 32;

// Sum over the block, the same bits in every thread.  `red` alternates between two buffers from call to call, so that one barrier is enough.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int lane = threadIdx.x & 31;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same of three sums at once.
__device__ __forceinline__ void block_sums(float v[3], float (*red)[NORM_MAX_WARPS]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int q = 0; q < 3; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
    const int lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
        for (int q = 0; q < 3; ++q) red[q][threadIdx.x >> 5] = v[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 3; ++q) v[q] = lane < (int)(blockDim.x >> 5) ? red[q][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int q = 0; q < 3; ++q) v[q] += __shfl_xor_sync(0xffffffffu, v[q], o);
}

// 1 / sqrt(sum / K + eps)
__device__ __forceinline__ float rms_inverse(float sum, int K, float eps) { return __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)K), eps)); }
template <int P = 4> __device__ __forceinline__ float dot(const f32x2 a[P], const f32x2 b[P], float sum) {
    f32x2 s = mul2(a[0], b[0]);
#pragma unroll
    for (int i = 1; i < P; ++i) s = fma2(a[i], b[i], s);
    return sum + (lo_of(s) + hi_of(s));
}

// First column of a thread's vector c, and the distance of its elements: adjacent, or as many apart as the block has threads.
template <bool ALIGNED> __device__ __forceinline__ int norm_column(int c) { return ALIGNED ? (c * blockDim.x + threadIdx.x) * 8 : c * 8 * blockDim.x + threadIdx.x; }

// A thread's columns of the weights, ones for a scale that is not there, in its own slots of shared memory: 48 KB at 4096 columns, which the rows would
// drive out of the L1 cache (backward 4096 x 4096 bfloat16: 78 us with the weights read from there, 67 so).
template <int V, bool ALIGNED> struct HeldWeights {
    float4* mine;
    __device__ __forceinline__ void hold(int q, const float* p, int k, int K) {
        f32x2 w[V / 2];
        if (p && k < K) widen<float, V>(fetch<float, V, ALIGNED>(p + k, K - k, blockDim.x), w);
        else
#pragma unroll
            for (int i = 0; i < V / 2; ++i) w[i] = both(1.0f);
#pragma unroll
        for (int i = 0; i < V / 4; ++i) mine[(q * (V / 4) + i) * blockDim.x] = make_float4(lo_of(w[2 * i]), hi_of(w[2 * i]), lo_of(w[2 * i + 1]), hi_of(w[2 * i + 1]));
    }
    __device__ __forceinline__ void read(int q, f32x2 w[V / 2]) const {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 x = mine[(q * (V / 4) + i) * blockDim.x];
            w[2 * i] = pair(x.x, x.y);
            w[2 * i + 1] = pair(x.z, x.w);
        }
    }
};

template <typename T> struct NormRow { Vec<T, 8> h, y, g; };

template <typename T, int VECS, bool ALIGNED>
__global__ void __launch_bounds__(512, VECS == 1 ? 2 : 1)
block_norm_kernel(const el_block_norm_t a) {
    __shared__ float red[2][NORM_MAX_WARPS];
    extern __shared__ uint4 slots[];                          // one vector a thread: its weights
    const int K = a.width, stride = blockDim.x;
    HeldWeights<8, ALIGNED> held{reinterpret_cast<float4*>(slots) + threadIdx.x};
    auto weight = [&](int q, const float* p, int k, f32x2 w[4]) {
        if (VECS == 1) held.read(q, w);
        else widen<float, 8>(fetch<float, 8, ALIGNED>(p + k, K - k, stride), w);
    };
    NormRow<T> next[VECS];
    auto fetch_row = [&](int m) {
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = norm_column<ALIGNED>(c);
            next[c].y = next[c].h = next[c].g = zeros<T, 8>();
            if (k < K) {
                next[c].y = fetch<T, 8, ALIGNED>(static_cast<const T*>(a.y) + m * a.ld_y + k, K - k, stride);
                next[c].h = fetch<T, 8, ALIGNED>(static_cast<const T*>(a.h) + m * a.ld_h + k, K - k, stride);
                if (a.gate) next[c].g = fetch<T, 8, ALIGNED>(static_cast<const T*>(a.gate) + m * a.ld_gate + k, K - k, stride);
            }
        }
    };
    int m = blockIdx.x;
    if (m < a.rows) fetch_row(m);
    if (VECS == 1) {
        held.hold(0, a.post_weight, norm_column<ALIGNED>(0), K);
        held.hold(1, a.pre_weight, norm_column<ALIGNED>(0), K);
        if (a.scale) held.hold(2, a.scale, norm_column<ALIGNED>(0), K);
    }
    for (; m < a.rows; m += gridDim.x) {
        NormRow<T> row[VECS];
        f32x2 v[VECS][4];
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            row[c] = next[c];
            widen<T, 8>(row[c].y, v[c]);
            ss = dot(v[c], v[c], ss);
        }
        if (VECS == 1 && m + (int)gridDim.x < a.rows) fetch_row(m + gridDim.x);
        const float r1 = rms_inverse(block_sum(ss, red[0]), K, a.eps);
        ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = norm_column<ALIGNED>(c);
            if (k >= K) continue;
            f32x2 h[4], w[4], f[4];
            widen<T, 8>(row[c].h, h);
            weight(0, a.post_weight, k, w);
            if (a.gate) {
                widen<T, 8>(row[c].g, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], sigmoid2(f[i]));
            }
            if (a.scale) {
                weight(2, a.scale, k, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], f[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v[c][i] = fma2(w[i], mul2(v[c][i], both(r1)), h[i]);      // columns behind the row's end hold zeros
            ss = dot(v[c], v[c], ss);
            put<T, 8, ALIGNED>(static_cast<T*>(a.h_out) + (long long)m * K + k, K - k, stride, v[c]);
        }
        const float r2 = rms_inverse(block_sum(ss, red[1]), K, a.eps);
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = norm_column<ALIGNED>(c);
            if (k >= K) continue;
            f32x2 w[4];
            weight(1, a.pre_weight, k, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], mul2(v[c][i], both(r2)));
            put<T, 8, ALIGNED>(static_cast<T*>(a.normed) + (long long)m * K + k, K - k, stride, w);
        }
        if (a.rstd && threadIdx.x == 0) {
            a.rstd[2 * (long long)m] = r1;
            a.rstd[2 * (long long)m + 1] = r2;
        }
        if (VECS > 1 && m + (int)gridDim.x < a.rows) fetch_row(m + gridDim.x);
    }
}

// Backward, rows of up to 4096 columns: a row's values stay in registers, one vector of 16 bytes a thread, and so do the column sums of a block's
// rows, which go to `partial` [blocks][3][width]: dw1, dw2, ds.  The next row is on asynchronous copies into the threads' own slots in shared
// memory (one row ahead; two or three gain nothing); rows that no vector copy takes are fetched into registers.  4096 x 4096, bfloat16 67 us, float32 95.
template <typename T> constexpr int NORM_V = 16 / sizeof(T);
template <typename T> constexpr int NORM_THREADS = sizeof(T) == 2 ? 512 : 1024;        // of an SM: what its registers take
template <typename T> struct NormGrads { Vec<T, NORM_V<T>> v[5]; };              // dnormed, y, h, gate, dh_out

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(NORM_THREADS<T>, 1)
block_norm_backward_kernel(const el_block_norm_t a, float* __restrict__ partial) {
    __shared__ float red[2][3][NORM_MAX_WARPS];
    constexpr int V = NORM_V<T>, P = V / 2;
    const int K = a.width, stride = blockDim.x, k = ALIGNED ? threadIdx.x * V : threadIdx.x;
    const bool mine = k < K;
    f32x2 sums[3][P];
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 0; i < P; ++i) sums[q][i] = both(0.0f);
    extern __shared__ uint4 slots[];                          // [tensor][thread], then the weights
    const void* const from[5] = {a.dnormed, a.y, a.h, a.gate, a.dh_out};
    const long long pitch[5] = {a.ld_dnormed, a.ld_y, a.ld_h, a.ld_gate, a.ld_dh_out};
    uint4* const mine_ahead = slots + threadIdx.x;
    HeldWeights<V, ALIGNED> held{reinterpret_cast<float4*>(slots + (ALIGNED ? 5 * stride : 0)) + threadIdx.x};
    NormGrads<T> next;
    auto request = [&](int m) {
        if (m < a.rows && mine) {
#pragma unroll
            for (int q = 0; q < 5; ++q) {
                if (!from[q]) continue;
                const T* src = static_cast<const T*>(from[q]) + m * pitch[q] + k;
                if constexpr (ALIGNED) rowio::cp_async16(mine_ahead + q * stride, src);
                else next.v[q] = fetch<T, V, false>(src, K - k, stride);
            }
        }
        if (ALIGNED) rowio::cp_async_commit();
    };
    auto take = [&]() {                                       // zeros for a tensor that is not there
        NormGrads<T> row;
#pragma unroll
        for (int q = 0; q < 5; ++q) {
            row.v[q] = zeros<T, V>();
            if (!from[q] || !mine) continue;
            if constexpr (ALIGNED) {
                const uint4 x = mine_ahead[q * stride];
                row.v[q].w[0] = x.x; row.v[q].w[1] = x.y; row.v[q].w[2] = x.z; row.v[q].w[3] = x.w;
            } else {
                row.v[q] = next.v[q];
            }
        }
        return row;
    };
    auto out = [&](void* p, int m, const f32x2 v[P]) {
        if (p && mine) put<T, V, ALIGNED>(static_cast<T*>(p) + (long long)m * K + k, K - k, stride, v);
    };
    const int G = gridDim.x;
    request(blockIdx.x);
    held.hold(0, a.post_weight, k, K);
    held.hold(1, a.scale, k, K);
    held.hold(2, a.pre_weight, k, K);
    float r1_next = 0.0f, r2_next = 0.0f;
    auto rms = [&](int m) {                                   // one row ahead too: nothing of a row can start without them
        if (m < a.rows) {
            r1_next = a.rstd[2 * (long long)m];
            r2_next = a.rstd[2 * (long long)m + 1];
        }
    };
    rms(blockIdx.x);
    int turn = 0;
    for (int m = blockIdx.x; m < a.rows; m += G, turn ^= 1) {
        if (ALIGNED) rowio::cp_async_wait<0>();
        const NormGrads<T> row = take();
        const float r1 = r1_next, r2 = r2_next;
        rms(m + G);
        request(m + G);
        f32x2 yn[P], hn[P], sg[P], dt[P], w1[P], s[P], t[P], q[P];
        widen<T, V>(row.v[1], yn);
        widen<T, V>(row.v[2], hn);
        widen<T, V>(row.v[3], sg);
        widen<T, V>(row.v[0], dt);
        held.read(0, w1);
        held.read(1, s);
        held.read(2, t);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            yn[i] = mul2(yn[i], both(r1));
            sg[i] = a.gate ? sigmoid2(sg[i]) : both(1.0f);
            q[i] = mul2(mul2(sg[i], s[i]), mul2(yn[i], w1[i]));
            hn[i] = mul2(add2(q[i], hn[i]), both(r2));
            sums[1][i] = fma2(dt[i], hn[i], sums[1][i]);
            dt[i] = mul2(dt[i], t[i]);
        }
        widen<T, V>(row.v[4], t);
#pragma unroll
        for (int i = 0; i < P; ++i) t[i] = fma2(both(r2), dt[i], t[i]);
        float v[3] = {dot<P>(dt, hn, 0.0f), dot<P>(t, q, 0.0f), dot<P>(hn, q, 0.0f)};
        block_sums(v, red[turn]);
        const float c2 = __fdiv_rn(v[0], (float)K), c1 = __fdiv_rn(__fmaf_rn(-__fmul_rn(c2, r2), v[2], v[1]), (float)K);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            t[i] = fma2(hn[i], both(-__fmul_rn(c2, r2)), t[i]);            // dh
            const f32x2 p = mul2(yn[i], w1[i]), ds = mul2(t[i], sg[i]), dp = mul2(ds, s[i]);
            sums[2][i] = fma2(ds, p, sums[2][i]);
            hn[i] = mul2(mul2(dp, p), fma2(sg[i], both(-1.0f), both(1.0f)));      // of the gate
            sums[0][i] = fma2(dp, yn[i], sums[0][i]);
            dt[i] = mul2(both(r1), fma2(yn[i], both(-c1), mul2(dp, w1[i])));
        }
        out(a.dh, m, t);
        if (a.gate) out(a.dgate, m, hn);
        out(a.dy_in, m, dt);
    }
    if (mine && partial) {
#pragma unroll
        for (int q = 0; q < 3; ++q) put<float, V, ALIGNED>(partial + ((long long)blockIdx.x * 3 + q) * K + k, K - k, stride, sums[q]);
    }
}

// Wider rows: nothing is kept between the two passes over a row, the second one's values come from L2, and the column sums are in shared memory.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(512, 1)
block_norm_backward_wide_kernel(const el_block_norm_t a, float* __restrict__ partial) {
    __shared__ float red[2][3][NORM_MAX_WARPS];
    extern __shared__ float4 sums_[];                         // [3][padded width / 4]: a thread's own columns, as vectors
    float* sums = reinterpret_cast<float*>(sums_);
    const int K = a.width, stride = blockDim.x, vecs = (K + 8 * stride - 1) / (8 * stride), padded = vecs * 8 * stride;
    auto slot = [&](int q, int c, int half) -> float4& { return sums_[((q * vecs + c) * 2 + half) * stride + threadIdx.x]; };
    for (int i = threadIdx.x; i < 3 * padded; i += stride) sums[i] = 0.0f;
    __syncthreads();
    auto get = [&](const void* p, long long ld, int m, int k, f32x2 v[4]) {
        widen<T, 8>(p ? fetch<T, 8, ALIGNED>(static_cast<const T*>(p) + m * ld + k, K - k, stride) : zeros<T, 8>(), v);
    };
    auto weight = [&](const float* p, int k, f32x2 w[4]) {
        if (p) widen<float, 8>(fetch<float, 8, ALIGNED>(p + k, K - k, stride), w);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = both(1.0f);
    };
    auto add_to = [&](int q, int c, const f32x2 v[4]) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float4 s = slot(q, c, half);
            s.x += lo_of(v[2 * half]); s.y += hi_of(v[2 * half]); s.z += lo_of(v[2 * half + 1]); s.w += hi_of(v[2 * half + 1]);
            slot(q, c, half) = s;
        }
    };
    int turn = 0;
    for (int m = blockIdx.x; m < a.rows; m += gridDim.x, turn ^= 1) {
        const float r1 = a.rstd[2 * (long long)m], r2 = a.rstd[2 * (long long)m + 1];
        // of a vector: yn, sigmoid of the gate, w1, scale, q, hn, dn and dh' + r2 dn w2
        auto form = [&](int k, f32x2 yn[4], f32x2 sg[4], f32x2 w1[4], f32x2 s[4], f32x2 q[4], f32x2 hn[4], f32x2 dn[4], f32x2 d[4]) {
            f32x2 w2[4];
            get(a.y, a.ld_y, m, k, yn);
            get(a.h, a.ld_h, m, k, hn);
            get(a.gate, a.ld_gate, m, k, sg);
            get(a.dnormed, a.ld_dnormed, m, k, dn);
            get(a.dh_out, a.ld_dh_out, m, k, d);
            weight(a.post_weight, k, w1);
            weight(a.scale, k, s);
            weight(a.pre_weight, k, w2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                yn[i] = mul2(yn[i], both(r1));
                sg[i] = a.gate ? sigmoid2(sg[i]) : both(1.0f);
                q[i] = mul2(mul2(sg[i], s[i]), mul2(yn[i], w1[i]));
                hn[i] = mul2(add2(q[i], hn[i]), both(r2));
                w2[i] = mul2(w2[i], dn[i]);
                d[i] = fma2(both(r2), w2[i], d[i]);
                dn[i] = mul2(dn[i], hn[i]);                    // what the sum for w2 takes
                w2[i] = mul2(w2[i], hn[i]);
            }
            return lo_of(add2(add2(w2[0], w2[1]), add2(w2[2], w2[3]))) + hi_of(add2(add2(w2[0], w2[1]), add2(w2[2], w2[3])));
        };
        float v[3] = {};
        for (int c = 0; c < vecs; ++c) {
            const int k = norm_column<ALIGNED>(c);
            if (k >= K) continue;
            f32x2 yn[4], sg[4], w1[4], s[4], q[4], hn[4], dn[4], d[4];
            v[0] += form(k, yn, sg, w1, s, q, hn, dn, d);
            v[1] = dot(d, q, v[1]);
            v[2] = dot(hn, q, v[2]);
            add_to(1, c, dn);
        }
        block_sums(v, red[turn]);
        const float c2 = __fdiv_rn(v[0], (float)K), c1 = __fdiv_rn(__fmaf_rn(-__fmul_rn(c2, r2), v[2], v[1]), (float)K);
        for (int c = 0; c < vecs; ++c) {
            const int k = norm_column<ALIGNED>(c);
            if (k >= K) continue;
            f32x2 yn[4], sg[4], w1[4], s[4], q[4], hn[4], dn[4], d[4], ds[4], dw[4];
            form(k, yn, sg, w1, s, q, hn, dn, d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[i] = fma2(hn[i], both(-__fmul_rn(c2, r2)), d[i]);        // dh
                const f32x2 p = mul2(yn[i], w1[i]), g = mul2(d[i], sg[i]), dp = mul2(g, s[i]);
                ds[i] = mul2(g, p);
                dw[i] = mul2(dp, yn[i]);
                hn[i] = mul2(mul2(dp, p), fma2(sg[i], both(-1.0f), both(1.0f)));      // of the gate
                dn[i] = mul2(both(r1), fma2(yn[i], both(-c1), mul2(dp, w1[i])));      // of y
            }
            add_to(2, c, ds);
            add_to(0, c, dw);
            if (a.dh) put<T, 8, ALIGNED>(static_cast<T*>(a.dh) + (long long)m * K + k, K - k, stride, d);
            if (a.gate && a.dgate) put<T, 8, ALIGNED>(static_cast<T*>(a.dgate) + (long long)m * K + k, K - k, stride, hn);
            if (a.dy_in) put<T, 8, ALIGNED>(static_cast<T*>(a.dy_in) + (long long)m * K + k, K - k, stride, dn);
        }
    }
    if (partial == nullptr) return;
    for (int c = 0; c < vecs; ++c) {
        const int k = norm_column<ALIGNED>(c);
        if (k >= K) continue;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const float4 x = slot(q, c, 0), y = slot(q, c, 1);
            const f32x2 v[4] = {pair(x.x, x.y), pair(x.z, x.w), pair(y.x, y.y), pair(y.z, y.w)};
            put<float, 8, ALIGNED>(partial + ((long long)blockIdx.x * 3 + q) * K + k, K - k, stride, v);
        }
    }
}

struct NormSums {
    float *dw1, *dw2, *ds;
    int K;
    __device__ __forceinline__ void operator()(int i, float v) const {
        float* out = i < K ? dw1 : i < 2 * K ? dw2 : ds;
        if (out) out[i % K] = v;
    }
};

// ---- host side ----------------------------------------------------------------------------------------------------------

constexpr int NORM_HELD = 4096;       // columns of a row that the kernels hold, one vector a thread

static int norm_threads(int K, int vecs) { return ((K + 8 * vecs - 1) / (8 * vecs) + 31) / 32 * 32; }
static int norm_vectors(int K) { return K <= NORM_HELD ? 1 : K <= 2 * NORM_HELD ? 2 : 4; }
static int norm_blocks(int rows, int per_sm) {
    int sms = 148;
    device_sm_count(&sms);
    return rows < (long long)sms * per_sm ? rows : sms * per_sm;
}
static int norm_held_threads(const el_block_norm_t& a) {       // of a block of the backward kernel that holds its rows
    const int V = a.dtype == EL_F32 ? NORM_V<float> : NORM_V<__half>;
    return ((a.width + V - 1) / V + 31) / 32 * 32;
}
static int norm_backward_blocks(const el_block_norm_t& a) {
    if (a.width > NORM_HELD || a.width == 0) return norm_blocks(a.rows, 1);
    return norm_blocks(a.rows, (a.dtype == EL_F32 ? NORM_THREADS<float> : NORM_THREADS<__half>) / norm_held_threads(a));
}
static bool norm_wants_sums(const el_block_norm_t& a) { return a.dpost_weight || a.dpre_weight || a.dscale; }
size_t block_norm_backward_workspace_bytes(const el_block_norm_t& a) {
    if (!norm_wants_sums(a) && (a.dh || a.dy_in || a.dgate)) return 0;
    return (size_t)norm_backward_blocks(a) * 3 * a.width * sizeof(float);
}

static bool norm_aligned(const el_block_norm_t& a) {
    if (a.width % 8 != 0) return false;
    const void* io[] = {a.h, a.y, a.gate, a.h_out, a.normed, a.dh_out, a.dnormed, a.dh, a.dy_in, a.dgate, a.post_weight, a.pre_weight, a.scale};
    for (const void* p : io)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    const long long ld[] = {a.ld_h, a.ld_y, a.ld_gate, a.ld_dh_out, a.ld_dnormed};
    for (long long l : ld)
        if (l % 8 != 0) return false;
    return true;
}

// Allows a kernel the shared memory that its widest rows take, once per device.
template <typename K> static int norm_shared(K kernel, int bytes, DeviceOnce& once) {
    int dev = 0;
    EL_CUDA_TRY(cudaGetDevice(&dev));
    if (!once.is_done(dev)) {
        EL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        once.mark(dev);
    }
    return EL_OK;
}

template <typename F> static int norm_variant(const el_block_norm_t& a, F f) {
    auto typed = [&](auto t) { return norm_aligned(a) ? f(t, std::true_type()) : f(t, std::false_type()); };
    switch (a.dtype) {
        case EL_F16: return typed(__half());
        case EL_BF16: return typed(__nv_bfloat16());
        default: return typed(float());
    }
}

int launch_block_norm(const el_block_norm_t& a, cudaStream_t st) {
    const int vecs = norm_vectors(a.width), threads = norm_threads(a.width, vecs), blocks = norm_blocks(a.rows, vecs == 1 ? 1024 / threads : 1);
    return norm_variant(a, [&](auto t, auto al) {
        using T = decltype(t);
        constexpr bool AL = decltype(al)::value;
        if (vecs == 1) {
            static DeviceOnce once;
            const int rc = norm_shared(block_norm_kernel<T, 1, AL>, 3 * 8 * 512 * (int)sizeof(float), once);
            if (rc != EL_OK) return rc;
            block_norm_kernel<T, 1, AL><<<blocks, threads, 3 * 8 * threads * sizeof(float), st>>>(a);
        } else if (vecs == 2) {
            block_norm_kernel<T, 2, AL><<<blocks, threads, 0, st>>>(a);
        } else {
            block_norm_kernel<T, 4, AL><<<blocks, threads, 0, st>>>(a);
        }
        return check_launch();
    });
}

int launch_block_norm_backward(const el_block_norm_t& a, cudaStream_t st) {
    const int blocks = norm_backward_blocks(a);
    float* partial = norm_wants_sums(a) ? static_cast<float*>(a.workspace) : nullptr;
    if (blocks > 0) {
        const int rc = norm_variant(a, [&](auto t, auto al) {
            using T = decltype(t);
            constexpr bool AL = decltype(al)::value;
            static DeviceOnce once[2];
            if (a.width <= NORM_HELD) {
                const int threads = norm_held_threads(a), rc = norm_shared(block_norm_backward_kernel<T, AL>, NORM_THREADS<T> * (5 * 16 + 3 * NORM_V<T> * 4), once[0]);
                if (rc != EL_OK) return rc;
                block_norm_backward_kernel<T, AL><<<blocks, threads, threads * ((AL ? 5 * 16 : 0) + 3 * NORM_V<T> * sizeof(float)), st>>>(a, partial);
                return check_launch();
            }
            const int rc = norm_shared(block_norm_backward_wide_kernel<T, AL>, 3 * 16384 * 4, once[1]);
            if (rc != EL_OK) return rc;
            const int vecs = (a.width + 8 * 512 - 1) / (8 * 512);
            block_norm_backward_wide_kernel<T, AL><<<blocks, 512, 3 * vecs * 8 * 512 * sizeof(float), st>>>(a, partial);
            return check_launch();
        });
        if (rc != EL_OK) return rc;
    }
    if (!norm_wants_sums(a)) return EL_OK;
    return launch_column_sums(partial, blocks, 3 * a.width, NormSums{a.dpost_weight, a.dpre_weight, a.dscale, a.width}, st);
}

}  // namespace el
