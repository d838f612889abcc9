// Depthwise causal convolution over the last 2 to 4 tokens of each channel, with bias and SiLU: forward, backward and single token.
//
//   pre[t] = bias + sum_j w[j] x[t - (W-1) + j],  y = pre * sigmoid(pre)
//   dpre = dy * slope(pre),  dx[t] = sum_i w[W-1-i] dpre[t + i],  dw[j] = sum_t dpre[t] x[t - (W-1) + j],  dbias = sum_t dpre[t]
//
// A thread owns a vector of channels and walks over a strip of tokens with the last W-1 inputs (backward: and W dpre) in registers, so
// every input is read once but for the W-1 tokens at a strip's ends.  Bound: memory, one read and one write per value (backward two and one).
#include "mamba_common.cuh"

namespace el {
using namespace mamba;

constexpr int CONV_LANES = 32;        // threads of a block along the channels; the others are strips of tokens

template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(128)
causal_conv_kernel(const el_conv_t a, int strip) {
    constexpr int V = 8, H = W - 1;
    const int d = (blockIdx.x * CONV_LANES + threadIdx.x) * V, b = blockIdx.z;
    if (d >= a.channels) return;
    const int valid = a.channels - d;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length;
    const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + d;
    T* y = static_cast<T*>(a.y) + (long long)b * a.length * a.channels + d;
    const T* first = a.initial_state ? static_cast<const T*>(a.initial_state) + (long long)b * H * a.channels + d : nullptr;
    auto input = [&](int t, float v[V]) {                     // x[t], the state before token 0; t < n
        if (t >= 0) load<T, V, ALIGNED>(x + t * a.x_stride_t, valid, v);
        else if (first) load<T, V, ALIGNED>(first + (long long)(t + H) * a.channels, valid, v);
        else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = 0.0f;
        }
    };
    const int s = blockIdx.y * blockDim.y + threadIdx.y;
    const int t0 = s * strip, t1 = min(t0 + strip, a.length);
    if (t0 < t1) {
        float w[W][V], bias[V], hist[H][V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = min(d + j, a.channels - 1);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][j] = a.weight[(long long)c * W + k];
            bias[j] = a.bias ? a.bias[c] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
            if (t0 - H + k < n) input(t0 - H + k, hist[k]);
        }
        const int tn = min(t1, n);
        int t = t0;
#pragma unroll 4
        for (; t < tn; ++t) {
            float v[V], o[V];
            load<T, V, ALIGNED>(x + t * a.x_stride_t, valid, v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float p = bias[j];
#pragma unroll
                for (int k = 0; k < H; ++k) p = __fmaf_rn(w[k][j], hist[k][j], p);
                p = __fmaf_rn(w[H][j], v[j], p);
                o[j] = a.silu ? __fmul_rn(p, sigmoid(p)) : p;
#pragma unroll
                for (int k = 0; k + 1 < H; ++k) hist[k][j] = hist[k + 1][j];
                hist[H - 1][j] = v[j];
            }
            store<T, V, ALIGNED>(y + (long long)t * a.channels, valid, o);
        }
        const float zero[V] = {};
        for (; t < t1; ++t) store<T, V, ALIGNED>(y + (long long)t * a.channels, valid, zero);
    }
    if (a.final_state && s == 0) {
        T* last = static_cast<T*>(a.final_state) + (long long)b * H * a.channels + d;
#pragma unroll
        for (int k = 0; k < H; ++k) {
            float v[V];
            input(n - H + k, v);
            store<T, V, ALIGNED>(last + (long long)k * a.channels, valid, v);
        }
    }
}

// dx and the partial sums of dweight and dbias: a block's strips are added in order and stored as one row [W+1][channels] of `partial`.
template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(256)
causal_conv_backward_kernel(const el_conv_t a, int strip, float* __restrict__ partial) {
    constexpr int V = 4, H = W - 1;
    extern __shared__ float red[];                            // [strips of the block][W+1][channels of the block]
    const int d = (blockIdx.x * CONV_LANES + threadIdx.x) * V, b = blockIdx.z;
    const int valid = a.channels - d;
    float dw[W][V] = {}, db[V] = {};
    const int s = blockIdx.y * blockDim.y + threadIdx.y;
    const int t0 = s * strip, t1 = min(t0 + strip, a.length);
    if (valid > 0 && (t0 < t1 || (s == 0 && a.d_initial_state))) {
        const int n = a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length;
        const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + d;
        const T* dy = static_cast<const T*>(a.dy) + b * a.dy_stride_b + d;
        T* dx = a.dx ? static_cast<T*>(a.dx) + (long long)b * a.length * a.channels + d : nullptr;
        const long long state_at = (long long)b * H * a.channels + d;
        const T* first = a.initial_state ? static_cast<const T*>(a.initial_state) + state_at : nullptr;
        const T* d_last = a.d_final_state ? static_cast<const T*>(a.d_final_state) + state_at : nullptr;
        T* d_first = a.d_initial_state ? static_cast<T*>(a.d_initial_state) + state_at : nullptr;
        float w[W][V], bias[V], hist[W][V], dp[W][V];         // hist: x[t-(W-1) .. t]; dp: dpre of the same tokens
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = min(d + j, a.channels - 1);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][j] = a.weight[(long long)c * W + k];
            bias[j] = a.bias ? a.bias[c] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const int t = t0 - W + k;
            float v[V] = {};
            if (t >= 0 && t < n) load<T, V, ALIGNED>(x + t * a.x_stride_t, valid, v);
            else if (t < 0 && t >= -H && first) load<T, V, ALIGNED>(first + (long long)(t + H) * a.channels, valid, v);
#pragma unroll
            for (int j = 0; j < V; ++j) { hist[k][j] = v[j]; dp[k][j] = 0.0f; }
        }
        // at token t the gradient of x[t-(W-1)] is complete; the strip's own x are t0 .. t1-1, for the first strip the state's before them too
        const int end = max(t1, t0) + H;
#pragma unroll 2
        for (int t = t0; t < end; ++t) {
            float v[V] = {}, g[V] = {};
            const bool live = t < n && a.dy;
            if (t < n) load<T, V, ALIGNED>(x + t * a.x_stride_t, valid, v);
            if (live) load<T, V, ALIGNED>(dy + t * a.dy_stride_t, valid, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
#pragma unroll
                for (int k = 0; k < H; ++k) { hist[k][j] = hist[k + 1][j]; dp[k][j] = dp[k + 1][j]; }
                hist[H][j] = v[j];
                float p = bias[j];
#pragma unroll
                for (int k = 0; k < W; ++k) p = __fmaf_rn(w[k][j], hist[k][j], p);
                if (a.silu) g[j] = live ? __fmul_rn(g[j], silu_slope(p, sigmoid(p))) : 0.0f;
                dp[H][j] = g[j];
            }
            if (t < t1) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    db[j] += g[j];
#pragma unroll
                    for (int k = 0; k < W; ++k) dw[k][j] = __fmaf_rn(g[j], hist[k][j], dw[k][j]);
                }
            }
            const int at = t - H;
            if (at >= t0 || s == 0) {
                float o[V] = {};
                if (at < n) {
#pragma unroll
                    for (int j = 0; j < V; ++j)
#pragma unroll
                        for (int k = 0; k < W; ++k) o[j] = __fmaf_rn(w[k][j], dp[H - k][j], o[j]);
                    if (d_last && at >= n - H) {              // x[at] is also part of the final state
                        float f[V];
                        load<T, V, ALIGNED>(d_last + (long long)(at - (n - H)) * a.channels, valid, f);
#pragma unroll
                        for (int j = 0; j < V; ++j) o[j] += f[j];
                    }
                }
                if (at >= 0) {
                    if (dx) store<T, V, ALIGNED>(dx + (long long)at * a.channels, valid, o);
                } else if (d_first) {
                    store<T, V, ALIGNED>(d_first + (long long)(at + H) * a.channels, valid, o);
                }
            }
        }
    }
    if (partial == nullptr) return;
    constexpr int COLS = CONV_LANES * V;
    float* mine = red + threadIdx.y * (W + 1) * COLS + threadIdx.x * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int k = 0; k < W; ++k) mine[k * COLS + j] = dw[k][j];
        mine[W * COLS + j] = db[j];
    }
    __syncthreads();
    float* row = partial + (long long)(blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * a.channels;
    for (int i = threadIdx.y * CONV_LANES + threadIdx.x; i < (W + 1) * COLS; i += blockDim.y * CONV_LANES) {
        const int c = blockIdx.x * COLS + i % COLS;
        float sum = 0.0f;
        for (int y = 0; y < (int)blockDim.y; ++y) sum += red[y * (W + 1) * COLS + i];
        if (c < a.channels) row[(long long)(i / COLS) * a.channels + c] = sum;
    }
}

// dweight [channels, W] and dbias from the rows of `partial`, added in order.
static __global__ void __launch_bounds__(256)
causal_conv_sums_kernel(const float* __restrict__ partial, int n_parts, int channels, int W, float* __restrict__ dweight, float* __restrict__ dbias) {
    const int i = blockIdx.x * 256 + threadIdx.x, all = (W + 1) * channels;
    if (i >= all) return;
    float sum = 0.0f;
#pragma unroll 8
    for (int p = 0; p < n_parts; ++p) sum += partial[(long long)p * all + i];
    const int k = i / channels, c = i - k * channels;
    if (k < W) {
        if (dweight) dweight[(long long)c * W + k] = sum;
    } else if (dbias) {
        dbias[c] = sum;
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(128)
causal_conv_step_kernel(const el_conv_t a) {
    constexpr int H = W - 1;
    const int d = blockIdx.x * 128 + threadIdx.x, b = blockIdx.y;
    if (d >= a.channels) return;
    const T* in = static_cast<const T*>(a.initial_state) + (long long)b * H * a.channels + d;
    T* out = static_cast<T*>(a.final_state) + (long long)b * H * a.channels + d;
    const T x = static_cast<const T*>(a.x)[b * a.x_stride_b + d];
    T rows[W];
#pragma unroll
    for (int k = 0; k < H; ++k) rows[k] = in[(long long)k * a.channels];
    rows[H] = x;
    float p = a.bias ? a.bias[d] : 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) p = __fmaf_rn(a.weight[(long long)d * W + k], to_float<T>(rows[k]), p);
    static_cast<T*>(a.y)[(long long)b * a.channels + d] = from_float<T>(a.silu ? __fmul_rn(p, sigmoid(p)) : p);
#pragma unroll
    for (int k = 0; k < H; ++k) out[(long long)k * a.channels] = rows[k + 1];
}

// ---- host side ----------------------------------------------------------------------------------------------------------

// Whether V channels at a time can be read as vectors: base and strides (in elements) are multiples of the vector.
static bool vectors(const void* p, long long s0, long long s1, int dtype, int V) {
    const int e = dtype == EL_F32 ? 4 : 2, bytes = V * e < 16 ? V * e : 16;
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && s0 % V == 0 && s1 % V == 0;
}

static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Tokens of a strip: long strips read fewer tokens twice, short ones give every SM work.
static int conv_strip(const el_conv_t& a, int vectors_per_token, int blocks_of) {
    int sms = 148;
    device_sm_count(&sms);
    const long long threads = (long long)a.batch * vectors_per_token * a.length;       // at one token a strip
    int strip = 32;
    while (strip > 4 && threads / strip < (long long)sms * blocks_of) strip >>= 1;
    return strip;
}

constexpr int FW_STRIPS = 4, BW_STRIPS = 8;

struct ConvBackwardPlan { int strip, blocks_t; };
static ConvBackwardPlan conv_backward_plan(const el_conv_t& a) {
    const int strip = conv_strip(a, (a.channels + 3) / 4, 1024);
    return {strip, ceil_div(a.length > 0 ? a.length : 1, (long long)strip * BW_STRIPS)};
}

size_t causal_conv_backward_workspace_bytes(const el_conv_t& a) {
    return (size_t)a.batch * conv_backward_plan(a).blocks_t * (a.width + 1) * a.channels * sizeof(float);
}

template <typename F> static int by_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}
template <typename F> static int by_width(int W, F f) {
    switch (W) {
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        default: return f(std::integral_constant<int, 4>());
    }
}

int launch_causal_conv(const el_conv_t& a, cudaStream_t st) {
    const int strip = conv_strip(a, (a.channels + 7) / 8, 512);
    const dim3 grid(ceil_div(a.channels, CONV_LANES * 8), ceil_div(a.length > 0 ? a.length : 1, (long long)strip * FW_STRIPS), a.batch);
    if (grid.y > 65535 || grid.z > 65535) return EL_ERR_TOO_LARGE;
    const dim3 block(CONV_LANES, FW_STRIPS);
    const bool al = a.channels % 8 == 0 && vectors(a.x, a.x_stride_b, a.x_stride_t, a.dtype, 8) && vectors(a.y, 0, 0, a.dtype, 8) &&
                    vectors(a.initial_state, 0, 0, a.dtype, 8) && vectors(a.final_state, 0, 0, a.dtype, 8);
    return by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            if (al) causal_conv_kernel<T, W, true><<<grid, block, 0, st>>>(a, strip);
            else causal_conv_kernel<T, W, false><<<grid, block, 0, st>>>(a, strip);
            return check_launch();
        });
    });
}

int launch_causal_conv_backward(const el_conv_t& a, cudaStream_t st) {
    const ConvBackwardPlan plan = conv_backward_plan(a);
    const dim3 grid(ceil_div(a.channels, CONV_LANES * 4), plan.blocks_t, a.batch), block(CONV_LANES, BW_STRIPS);
    if (grid.y > 65535 || grid.z > 65535) return EL_ERR_TOO_LARGE;
    const bool sums = a.dweight || a.dbias;
    float* partial = sums ? static_cast<float*>(a.workspace) : nullptr;
    const bool al = a.channels % 4 == 0 && vectors(a.x, a.x_stride_b, a.x_stride_t, a.dtype, 4) && vectors(a.dy, a.dy_stride_b, a.dy_stride_t, a.dtype, 4) &&
                    vectors(a.dx, 0, 0, a.dtype, 4) && vectors(a.initial_state, 0, 0, a.dtype, 4) && vectors(a.d_initial_state, 0, 0, a.dtype, 4) &&
                    vectors(a.d_final_state, 0, 0, a.dtype, 4);
    const size_t shared = (size_t)BW_STRIPS * (a.width + 1) * CONV_LANES * 4 * sizeof(float);       // 20 KB at most
    const int rc = a.batch == 0 ? EL_OK : by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            if (al) causal_conv_backward_kernel<T, W, true><<<grid, block, shared, st>>>(a, plan.strip, partial);
            else causal_conv_backward_kernel<T, W, false><<<grid, block, shared, st>>>(a, plan.strip, partial);
            return check_launch();
        });
    });
    if (rc != EL_OK || !sums) return rc;
    causal_conv_sums_kernel<<<ceil_div((long long)(a.width + 1) * a.channels, 256), 256, 0, st>>>(partial, a.batch * plan.blocks_t, a.channels, a.width,
                                                                                                 a.dweight, a.dbias);
    return check_launch();
}

int launch_causal_conv_step(const el_conv_t& a, cudaStream_t st) {
    const dim3 grid(ceil_div(a.channels, 128), a.batch);
    if (grid.y > 65535) return EL_ERR_TOO_LARGE;
    return by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            causal_conv_step_kernel<decltype(t), decltype(w)::value><<<grid, 128, 0, st>>>(a);
            return check_launch();
        });
    });
}

}  // namespace el
