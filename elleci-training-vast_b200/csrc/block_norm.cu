// The norm after a block, its gate and residual scale, the residual addition and the norm before the next block, in one pass.
//
//   p = w1 y r1,  r1 = 1/sqrt(mean y^2 + eps);   h' = h + s sigmoid(g) p;   n = w2 h' r2,  r2 = 1/sqrt(mean h'^2 + eps)
// backward (yn = y r1, hn = h' r2, both formed again from the inputs):
//   dh = dh' + r2 (dn w2 - hn mean(dn w2 hn));  dw2 = sum dn hn;  ds = sum dh sigmoid(g) p;  dg = dh s p sigmoid'(g)
//   dp = dh s sigmoid(g);  dw1 = sum dp yn;  dy = r1 (dp w1 - yn mean(dp w1 yn))
// Row sums in float32: a thread adds 8 or 16 squares, the block adds the threads' in a fixed order.
//
// A block walks over rows; a thread owns the same one or two vectors of 8 columns in each.
#include "mamba_common.cuh"

namespace el {
using namespace mamba;

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

template <typename T, int VECS, bool ALIGNED>
__global__ void __launch_bounds__(1024)
block_norm_kernel(const el_block_norm_t a) {
    __shared__ float red[2][NORM_MAX_WARPS];
    const int K = a.width;
    for (int m = blockIdx.x; m < a.rows; m += gridDim.x) {
        const T* h = static_cast<const T*>(a.h) + m * a.ld_h;
        const T* y = static_cast<const T*>(a.y) + m * a.ld_y;
        const T* g = a.gate ? static_cast<const T*>(a.gate) + m * a.ld_gate : nullptr;
        float v[VECS][8], ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
            if (k < K) load<T, 8, ALIGNED>(y + k, K - k, v[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = __fmaf_rn(v[c][j], v[c][j], ss);
        }
        const float r1 = __frsqrt_rn(__fadd_rn(__fdiv_rn(block_sum(ss, red[0]), (float)K), a.eps));
        ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = (c * blockDim.x + threadIdx.x) * 8;
            if (k < K) {
                float hv[8], gv[8], w[8], s[8];
                load<T, 8, ALIGNED>(h + k, K - k, hv);
                if (g) load<T, 8, ALIGNED>(g + k, K - k, gv);
                load<float, 8, ALIGNED>(a.post_weight + k, K - k, w);
                if (a.scale) load<float, 8, ALIGNED>(a.scale + k, K - k, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float f = g ? sigmoid(gv[j]) : 1.0f;
                    if (a.scale) f *= s[j];
                    v[c][j] = __fmaf_rn(f, v[c][j] * r1 * w[j], hv[j]);
                    ss = __fmaf_rn(v[c][j], v[c][j], ss);          // columns behind the row's end hold zeros
                }
                store<T, 8, ALIGNED>(static_cast<T*>(a.h_out) + (long long)m * K + k, K - k, v[c]);
            }
        }
        const float r2 = __frsqrt_rn(__fadd_rn(__fdiv_rn(block_sum(ss, red[1]), (float)K), a.eps));
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = (c * blockDim.x + threadIdx.x) * 8;
            if (k < K) {
                float w[8];
                load<float, 8, ALIGNED>(a.pre_weight + k, K - k, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * r2 * w[j];
                store<T, 8, ALIGNED>(static_cast<T*>(a.normed) + (long long)m * K + k, K - k, v[c]);
            }
        }
        if (a.rstd && threadIdx.x == 0) {
            a.rstd[2 * (long long)m] = r1;
            a.rstd[2 * (long long)m + 1] = r2;
        }
    }
}

// Column sums of a block's rows stay in registers and go to `partial` [blocks][3][width]: dw1, dw2, ds.
template <typename T, int VECS, bool ALIGNED>
__global__ void __launch_bounds__(1024)
block_norm_backward_kernel(const el_block_norm_t a, float* __restrict__ partial) {
    __shared__ float red[2][NORM_MAX_WARPS];
    const int K = a.width;
    float sums[VECS][3][8] = {};
    for (int m = blockIdx.x; m < a.rows; m += gridDim.x) {
        const float r1 = a.rstd[2 * (long long)m], r2 = a.rstd[2 * (long long)m + 1];
        const T* h = static_cast<const T*>(a.h) + m * a.ld_h;
        const T* y = static_cast<const T*>(a.y) + m * a.ld_y;
        const T* g = a.gate ? static_cast<const T*>(a.gate) + m * a.ld_gate : nullptr;
        const T* dh = a.dh_out ? static_cast<const T*>(a.dh_out) + m * a.ld_dh_out : nullptr;
        const T* dn = a.dnormed ? static_cast<const T*>(a.dnormed) + m * a.ld_dnormed : nullptr;
        float yn[VECS][8], hn[VECS][8], sg[VECS][8], dt[VECS][8], dot = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) yn[c][j] = hn[c][j] = sg[c][j] = dt[c][j] = 0.0f;
            if (k < K) {
                float w1[8], w2[8], s[8];
                load<T, 8, ALIGNED>(y + k, K - k, yn[c]);
                load<T, 8, ALIGNED>(h + k, K - k, hn[c]);
                if (g) load<T, 8, ALIGNED>(g + k, K - k, sg[c]);
                if (dn) load<T, 8, ALIGNED>(dn + k, K - k, dt[c]);
                load<float, 8, ALIGNED>(a.post_weight + k, K - k, w1);
                load<float, 8, ALIGNED>(a.pre_weight + k, K - k, w2);
                if (a.scale) load<float, 8, ALIGNED>(a.scale + k, K - k, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    yn[c][j] *= r1;
                    sg[c][j] = g ? sigmoid(sg[c][j]) : 1.0f;
                    const float f = a.scale ? sg[c][j] * s[j] : sg[c][j];
                    hn[c][j] = __fmaf_rn(f, yn[c][j] * w1[j], hn[c][j]) * r2;
                    sums[c][1][j] = __fmaf_rn(dt[c][j], hn[c][j], sums[c][1][j]);
                    dt[c][j] *= w2[j];
                    dot = __fmaf_rn(dt[c][j], hn[c][j], dot);
                }
            }
        }
        const float c2 = __fdiv_rn(block_sum(dot, red[0]), (float)K);
        dot = 0.0f;
#pragma unroll
        for (int c = 0; c < VECS; ++c) {
            const int k = (c * blockDim.x + threadIdx.x) * 8;
            if (k < K) {
                float w1[8], s[8], d[8] = {}, dg[8];
                if (dh) load<T, 8, ALIGNED>(dh + k, K - k, d);
                load<float, 8, ALIGNED>(a.post_weight + k, K - k, w1);
                if (a.scale) load<float, 8, ALIGNED>(a.scale + k, K - k, s);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    d[j] = __fmaf_rn(r2, __fmaf_rn(-hn[c][j], c2, dt[c][j]), d[j]);
                    const float p = yn[c][j] * w1[j], sc = a.scale ? s[j] : 1.0f, ds = d[j] * sg[c][j];
                    sums[c][2][j] = __fmaf_rn(ds, p, sums[c][2][j]);
                    dg[j] = ds * sc * p * (1.0f - sg[c][j]);
                    const float dp = ds * sc;
                    sums[c][0][j] = __fmaf_rn(dp, yn[c][j], sums[c][0][j]);
                    dt[c][j] = dp * w1[j];
                    dot = __fmaf_rn(dt[c][j], yn[c][j], dot);
                }
                if (a.dh) store<T, 8, ALIGNED>(static_cast<T*>(a.dh) + (long long)m * K + k, K - k, d);
                if (a.dgate && g) store<T, 8, ALIGNED>(static_cast<T*>(a.dgate) + (long long)m * K + k, K - k, dg);
            }
        }
        const float c1 = __fdiv_rn(block_sum(dot, red[1]), (float)K);
        if (a.dy_in) {
#pragma unroll
            for (int c = 0; c < VECS; ++c) {
                const int k = (c * blockDim.x + threadIdx.x) * 8;
                if (k < K) {
                    float d[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] = r1 * __fmaf_rn(-yn[c][j], c1, dt[c][j]);
                    store<T, 8, ALIGNED>(static_cast<T*>(a.dy_in) + (long long)m * K + k, K - k, d);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < VECS; ++c) {
        const int k = (c * blockDim.x + threadIdx.x) * 8;
        if (k < K) {
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j < K) partial[((long long)blockIdx.x * 3 + q) * K + k + j] = sums[c][q][j];
        }
    }
}

static __global__ void __launch_bounds__(256)
block_norm_sums_kernel(const float* __restrict__ partial, int n_parts, int K, float* __restrict__ dw1, float* __restrict__ dw2, float* __restrict__ ds) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= 3 * K) return;
    float s = 0.0f;
#pragma unroll 8
    for (int p = 0; p < n_parts; ++p) s += partial[(long long)p * 3 * K + i];
    float* out = i < K ? dw1 : i < 2 * K ? dw2 : ds;
    if (out) out[i % K] = s;
}

// ---- host side ----------------------------------------------------------------------------------------------------------

static int norm_threads(int K) {
    const int vecs = K > 8192 ? 2 : 1;
    const int t = (K + 8 * vecs - 1) / (8 * vecs);
    return (t + 31) / 32 * 32;
}
static int norm_backward_blocks(const el_block_norm_t& a) {
    int sms = 148;
    device_sm_count(&sms);
    return a.rows < sms ? a.rows : sms;
}
size_t block_norm_backward_workspace_bytes(const el_block_norm_t& a) { return (size_t)norm_backward_blocks(a) * 3 * a.width * sizeof(float); }

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

template <typename F> static int norm_variant(const el_block_norm_t& a, F f) {
    auto typed = [&](auto t) {
        const bool al = norm_aligned(a);
        if (a.width > 8192) return al ? f(t, std::integral_constant<int, 2>(), std::true_type()) : f(t, std::integral_constant<int, 2>(), std::false_type());
        return al ? f(t, std::integral_constant<int, 1>(), std::true_type()) : f(t, std::integral_constant<int, 1>(), std::false_type());
    };
    switch (a.dtype) {
        case EL_F16: return typed(__half());
        case EL_BF16: return typed(__nv_bfloat16());
        default: return typed(float());
    }
}

int launch_block_norm(const el_block_norm_t& a, cudaStream_t st) {
    return norm_variant(a, [&](auto t, auto vecs, auto al) {
        block_norm_kernel<decltype(t), decltype(vecs)::value, decltype(al)::value><<<a.rows, norm_threads(a.width), 0, st>>>(a);
        return check_launch();
    });
}

int launch_block_norm_backward(const el_block_norm_t& a, cudaStream_t st) {
    const int blocks = norm_backward_blocks(a);
    float* partial = static_cast<float*>(a.workspace);
    if (blocks > 0) {
        const int rc = norm_variant(a, [&](auto t, auto vecs, auto al) {
            block_norm_backward_kernel<decltype(t), decltype(vecs)::value, decltype(al)::value><<<blocks, norm_threads(a.width), 0, st>>>(a, partial);
            return check_launch();
        });
        if (rc != EL_OK) return rc;
    }
    if (a.dpost_weight || a.dpre_weight || a.dscale)
        block_norm_sums_kernel<<<(3 * a.width + 255) / 256, 256, 0, st>>>(partial, blocks, a.width, a.dpost_weight, a.dpre_weight, a.dscale);
    return check_launch();
}

}  // namespace el
