// Depthwise causal convolution over the last 2 to 4 tokens of each channel, with bias and SiLU: forward, backward and single token.
//
//   pre[t] = bias + sum_j w[j] x[t - (W-1) + j],  y = pre * sigmoid(pre)
//   dpre = dy * slope(pre),  dx[t] = sum_i w[W-1-i] dpre[t + i],  dw[j] = sum_t dpre[t] x[t - (W-1) + j],  dbias = sum_t dpre[t]
//
// A thread owns a vector of channels and walks over a strip of tokens with the last W-1 inputs (backward: and W dpre) in registers, so
// every input is read once but for the W-1 tokens at a strip's ends.  Floor: memory, one read and one write per value
// (backward two and one).  4 x 1024 tokens of 8192 channels: forward 33 us in bfloat16 (floor 20), 49 in float32 (41); backward 68 (31) and 84 (61): in
// 16-bit types no unit is full, a copy, an address step and a store of 8 bytes carry two operands each.
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

constexpr int CONV_LANES = 32;        // threads of a block along the channels; the others are strips of tokens

constexpr int CONV_SLOTS = 8;         // tokens that are on their way to a thread's slots in shared memory
constexpr int CONV_V = 4;             // channels of a thread

// What a thread will read of later tokens it copies into its own slots with asynchronous copies, so that tokens ahead cost neither registers
// nor barriers.  Channels that no vector copy takes go through registers.
template <typename T, int TENSORS, bool ALIGNED> struct ConvRing {
    using Slot = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
    Slot* mine;
    int threads;
    __device__ __forceinline__ explicit ConvRing(void* shared) {
        threads = blockDim.x * blockDim.y;
        mine = static_cast<Slot*>(shared) + threadIdx.y * blockDim.x + threadIdx.x;
    }
    __device__ __forceinline__ Slot* at(int t, int tensor) const { return mine + ((t & (CONV_SLOTS - 1)) * TENSORS + tensor) * threads; }
    __device__ __forceinline__ void request(int t, int tensor, const T* src, int valid) const {
        Slot* to = at(t, tensor);
        if constexpr (ALIGNED) {
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
            if constexpr (sizeof(T) == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
            else asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        } else {
            const Vec<T, CONV_V> v = fetch<T, CONV_V, false>(src, valid, CONV_LANES);
            *to = *reinterpret_cast<const Slot*>(&v);
        }
    }
    __device__ __forceinline__ void read(int t, int tensor, f32x2 v[CONV_V / 2]) const {
        Vec<T, CONV_V> r;
        *reinterpret_cast<Slot*>(&r) = *at(t, tensor);
        widen<T, CONV_V>(r, v);
    }
};

// Where a thread's channels lie: V adjacent ones, or, where vectors are not possible, every 32nd.
template <int V, bool ALIGNED> struct ConvPlace {
    int d, valid;
    __device__ __forceinline__ explicit ConvPlace(int channels) {
        d = ALIGNED ? (blockIdx.x * CONV_LANES + threadIdx.x) * V : blockIdx.x * CONV_LANES * V + threadIdx.x;
        valid = channels - d;
    }
    __device__ __forceinline__ int channel(int j) const { return ALIGNED ? d + j : d + CONV_LANES * j; }
};

template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(128)
causal_conv_kernel(const el_conv_t a, int strip) {
    constexpr int V = CONV_V, P = V / 2, H = W - 1, U = 4;
    extern __shared__ uint4 slots[];
    const ConvRing<T, 1, ALIGNED> ring(slots);
    const ConvPlace<V, ALIGNED> at(a.channels);
    const int b = blockIdx.z;
    if (at.valid <= 0) return;
    const int n = a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length;
    const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + at.d;
    T* y = static_cast<T*>(a.y) + (long long)b * a.length * a.channels + at.d;
    const T* first = a.initial_state ? static_cast<const T*>(a.initial_state) + (long long)b * H * a.channels + at.d : nullptr;
    auto input = [&](int t) {                                 // x[t], the state before token 0, zeros from token n on
        if (t >= n) return zeros<T, V>();
        if (t >= 0) return fetch<T, V, ALIGNED>(x + t * a.x_stride_t, at.valid, CONV_LANES);
        return first ? fetch<T, V, ALIGNED>(first + (long long)(t + H) * a.channels, at.valid, CONV_LANES) : zeros<T, V>();
    };
    const int s = blockIdx.y * blockDim.y + threadIdx.y;
    const int t0 = s * strip, t1 = min(t0 + strip, a.length);
    if (t0 < t1) {
        f32x2 w[W][P], bias[P], win[H + U][P];                // win: x[t-H] .. x[t+U-1]
        const int tn = min(t1, n);
        const T* ask = x + t0 * a.x_stride_t;                 // of the token that is requested next
        T* to = y + (long long)t0 * a.channels;
        auto request = [&](int t) {                           // a group of tokens
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < tn) ring.request(t + u, 0, ask, at.valid);
                ask += a.x_stride_t;
            }
            rowio::cp_async_commit();
        };
        request(t0);
        request(t0 + U);
        static_assert(CONV_SLOTS == 2 * U, "");
#pragma unroll
        for (int k = 0; k < H; ++k) widen<T, V>(input(t0 - H + k), win[U + k]);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c0 = min(at.channel(2 * i), a.channels - 1), c1 = min(at.channel(2 * i + 1), a.channels - 1);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][i] = pair(a.weight[(long long)c0 * W + k], a.weight[(long long)c1 * W + k]);
            bias[i] = a.bias ? pair(a.bias[c0], a.bias[c1]) : both(0.0f);
        }
        auto group = [&](int t, auto edge) {                  // edge: some of the tokens are behind the strip or are padding
            constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
            for (int k = 0; k < H; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) win[k][i] = win[U + k][i];
            rowio::cp_async_wait<1>();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!EDGE || t + u < tn) ring.read(t + u, 0, win[H + u]);      // a slot that nothing was copied to is not looked at
                else
#pragma unroll
                    for (int i = 0; i < P; ++i) win[H + u][i] = both(0.0f);
            }
            request(t + 2 * U);
            f32x2 o[U][P];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    o[u][i] = bias[i];
#pragma unroll
                    for (int k = 0; k < W; ++k) o[u][i] = fma2(w[k][i], win[u + k][i], o[u][i]);
                }
            if (a.silu) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < P; ++i) o[u][i] = mul2(o[u][i], sigmoid2(o[u][i]));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (EDGE && t + u >= n) {
#pragma unroll
                    for (int i = 0; i < P; ++i) o[u][i] = both(0.0f);
                }
                if (!EDGE || t + u < t1) put<T, V, ALIGNED>(to, at.valid, CONV_LANES, o[u]);
                to += a.channels;
            }
        };
        int t = t0;
        for (; t + U <= tn; t += U) group(t, std::false_type());
        for (; t < t1; t += U) group(t, std::true_type());
    }
    if (a.final_state && s == 0) {
        T* last = static_cast<T*>(a.final_state) + (long long)b * H * a.channels + at.d;
#pragma unroll
        for (int k = 0; k < H; ++k) {
            f32x2 v[P];
            widen<T, V>(input(n - H + k), v);
            put<T, V, ALIGNED>(last + (long long)k * a.channels, at.valid, CONV_LANES, v);
        }
    }
}

// dx and the partial sums of dweight and dbias: a block's strips are added in order and stored as one row [W+1][channels] of `partial`.
template <typename T, int W, bool ALIGNED>
__global__ void __launch_bounds__(256, 2)
causal_conv_backward_kernel(const el_conv_t a, int strip, float* __restrict__ partial) {
    constexpr int V = CONV_V, P = V / 2, H = W - 1, U = 2, GROUPS = CONV_SLOTS / U;
    extern __shared__ uint4 slots[];                          // then the sums [strips of the block][W+1][channels of the block]
    const ConvRing<T, 2, ALIGNED> ring(slots);
    const ConvPlace<V, ALIGNED> at(a.channels);
    const int b = blockIdx.z;
    f32x2 dw[W][P], db[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        db[i] = both(0.0f);
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][i] = both(0.0f);
    }
    const int s = blockIdx.y * blockDim.y + threadIdx.y;
    const int t0 = s * strip, t1 = min(t0 + strip, a.length);
    if (at.valid > 0 && (t0 < t1 || (s == 0 && a.d_initial_state))) {
        const int n = a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length;
        const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + at.d;
        const T* dy = a.dy ? static_cast<const T*>(a.dy) + b * a.dy_stride_b + at.d : nullptr;
        T* dx = a.dx ? static_cast<T*>(a.dx) + (long long)b * a.length * a.channels + at.d : nullptr;
        const long long state_at = (long long)b * H * a.channels + at.d;
        const T* first = a.initial_state ? static_cast<const T*>(a.initial_state) + state_at : nullptr;
        const T* d_last = a.d_final_state ? static_cast<const T*>(a.d_final_state) + state_at : nullptr;
        T* d_first = a.d_initial_state ? static_cast<T*>(a.d_initial_state) + state_at : nullptr;
        auto input = [&](int t) {
            if (t >= n) return zeros<T, V>();
            if (t >= 0) return fetch<T, V, ALIGNED>(x + t * a.x_stride_t, at.valid, CONV_LANES);
            return first ? fetch<T, V, ALIGNED>(first + (long long)(t + H) * a.channels, at.valid, CONV_LANES) : zeros<T, V>();
        };
        // at token t the gradient of x[t-H] is complete; the strip's own x are t0 .. t1-1, for the first strip the state's before them too
        const int end = max(t1, t0) + H;
        f32x2 w[W][P], bias[P], win[H + U][P], dp[H + U][P];  // x and dpre of tokens t-H .. t+U-1
        const int tn = min(end, n);
        const T *ask_x = x + t0 * a.x_stride_t, *ask_g = dy + t0 * a.dy_stride_t;         // of the token that is requested next
        auto request = [&](int t) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < tn) {
                    ring.request(t + u, 0, ask_x, at.valid);
                    if (dy) ring.request(t + u, 1, ask_g, at.valid);
                }
                ask_x += a.x_stride_t;
                ask_g += a.dy_stride_t;
            }
            rowio::cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) request(t0 + i * U);
#pragma unroll
        for (int k = 0; k < H; ++k) {
            widen<T, V>(input(t0 - H + k), win[U + k]);
#pragma unroll
            for (int i = 0; i < P; ++i) dp[U + k][i] = both(0.0f);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c0 = min(at.channel(2 * i), a.channels - 1), c1 = min(at.channel(2 * i + 1), a.channels - 1);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][i] = pair(a.weight[(long long)c0 * W + k], a.weight[(long long)c1 * W + k]);
            bias[i] = a.bias ? pair(a.bias[c0], a.bias[c1]) : both(0.0f);
        }
        T* out = dx ? dx + (long long)(t0 - H) * a.channels : nullptr;        // of x[t-H]
        // edge: some of the tokens are padding or another strip's, or the x whose gradients they complete are, or these are the state's
        auto group = [&](int t, auto edge) {
            constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
            for (int k = 0; k < H; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    win[k][i] = win[U + k][i];
                    dp[k][i] = dp[U + k][i];
                }
            f32x2 g[U][P];
            rowio::cp_async_wait<GROUPS - 1>();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (EDGE || !dy) {
#pragma unroll
                    for (int i = 0; i < P; ++i) win[H + u][i] = g[u][i] = both(0.0f);
                }
                if (!EDGE || t + u < tn) {                    // a slot that nothing was copied to is not looked at
                    ring.read(t + u, 0, win[H + u]);
                    if (dy) ring.read(t + u, 1, g[u]);
                }
            }
            request(t + CONV_SLOTS);
            if (a.silu) {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        f32x2 p = bias[i];
#pragma unroll
                        for (int k = 0; k < W; ++k) p = fma2(w[k][i], win[u + k][i], p);
                        g[u][i] = mul2(g[u][i], silu_slope2(p, sigmoid2(p)));
                    }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool real = !EDGE || t + u < tn;        // not padding, whose slope may be anything if the bias is not finite
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    dp[H + u][i] = real ? g[u][i] : both(0.0f);
                    if (!EDGE || t + u < t1) {
                        db[i] = add2(db[i], dp[H + u][i]);
#pragma unroll
                        for (int k = 0; k < W; ++k) dw[k][i] = fma2(dp[H + u][i], win[u + k][i], dw[k][i]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int to = t + u - H;                     // whose gradient is complete
                T* here = out;
                if (dx) out += a.channels;
                if (EDGE && (t + u >= end || (to < t0 && s > 0))) continue;
                f32x2 o[P];
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    o[i] = both(0.0f);
                    if (!EDGE || to < n) {
                        o[i] = mul2(w[0][i], dp[u + H][i]);
#pragma unroll
                        for (int k = 1; k < W; ++k) o[i] = fma2(w[k][i], dp[u + H - k][i], o[i]);
                    }
                }
                if (EDGE && d_last && to < n && to >= n - H) {        // x[to] is also part of the final state
                    f32x2 f[P];
                    widen<T, V>(fetch<T, V, ALIGNED>(d_last + (long long)(to - (n - H)) * a.channels, at.valid, CONV_LANES), f);
#pragma unroll
                    for (int i = 0; i < P; ++i) o[i] = add2(o[i], f[i]);
                }
                if (!EDGE || to >= 0) {
                    if (dx) put<T, V, ALIGNED>(here, at.valid, CONV_LANES, o);
                } else if (d_first) {
                    put<T, V, ALIGNED>(d_first + (long long)(to + H) * a.channels, at.valid, CONV_LANES, o);
                }
            }
        };
        int t = t0;
        for (; t < t0 + H && t < end; t += U) group(t, std::true_type());
        for (; t + U <= t1 && t + U <= tn; t += U) group(t, std::false_type());
        for (; t < end; t += U) group(t, std::true_type());
    }
    rowio::cp_async_wait<0>();
    if (partial == nullptr) return;
    float* red = reinterpret_cast<float*>(slots) + 2 * CONV_SLOTS * V * blockDim.x * blockDim.y * sizeof(T) / sizeof(float);
    constexpr int COLS = CONV_LANES * V;
    float* mine = red + threadIdx.y * (W + 1) * COLS;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = ALIGNED ? threadIdx.x * V + j : threadIdx.x + CONV_LANES * j;
#pragma unroll
        for (int k = 0; k < W; ++k) mine[k * COLS + c] = j & 1 ? hi_of(dw[k][j / 2]) : lo_of(dw[k][j / 2]);
        mine[W * COLS + c] = j & 1 ? hi_of(db[j / 2]) : lo_of(db[j / 2]);
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

// Where column i of the sums belongs: dweight [channels, W], then dbias.
struct ConvSums {
    float *dweight, *dbias;
    int channels, W;
    __device__ __forceinline__ void operator()(int i, float v) const {
        const int k = i / channels, c = i - k * channels;
        if (k < W) {
            if (dweight) dweight[(long long)c * W + k] = v;
        } else if (dbias) {
            dbias[c] = v;
        }
    }
};

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

constexpr int FW_STRIPS = 4, BW_STRIPS = 8;

// Tokens of a strip, at most `longest`.  A strip costs its start (weights, the first tokens' latency, W-1 tokens read again) and its end, so it is long; but
// every SM is given 400 threads first.  Strips of up to 32 / 64 / 128 tokens, us: forward 4 x 1024 x 8192 35.7 / 33.4 / 36.1; backward 78.6 / 76.7 / 68.4.
// 1024 threads an SM instead: 3 x 1999 x 1504 forward 13.0 -> 19.0, backward 28.0 -> 35.0.
// Millions of tokens take longer strips, `strips` of them a block, so that a grid's 65535 rows hold them.
static int conv_strip(const el_conv_t& a, int longest, int strips) {
    int sms = 148;
    device_sm_count(&sms);
    const long long threads = (long long)a.batch * ((a.channels + CONV_V - 1) / CONV_V) * a.length;        // at one token a strip
    int strip = longest;
    while (strip > 8 && threads / strip < (long long)sms * 400) strip >>= 1;
    while (ceil_div(a.length, (long long)strip * strips) > 65535) strip <<= 1;
    return strip;
}

struct ConvBackwardPlan { int strip, blocks_t; };
static ConvBackwardPlan conv_backward_plan(const el_conv_t& a) {
    const int strip = conv_strip(a, 128, BW_STRIPS);
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

// n sequences of a call from number b0 on, as a call of their own.
static el_conv_t conv_sequences(const el_conv_t& a, int b0, int n) {
    const int e = a.dtype == EL_F32 ? 4 : 2;
    const long long tokens = (long long)a.length * a.channels, state = (long long)(a.width - 1) * a.channels;
    auto from = [&](auto* p, long long pitch) { return p ? reinterpret_cast<decltype(p)>(reinterpret_cast<uintptr_t>(p) + (uintptr_t)(b0 * pitch * e)) : p; };
    el_conv_t s = a;
    s.batch = n;
    s.x = from(a.x, a.x_stride_b);
    s.dy = from(a.dy, a.dy_stride_b);
    s.y = from(a.y, tokens);
    s.dx = from(a.dx, tokens);
    s.initial_state = from(a.initial_state, state);
    s.final_state = from(a.final_state, state);
    s.d_initial_state = from(a.d_initial_state, state);
    s.d_final_state = from(a.d_final_state, state);
    if (a.lengths) s.lengths = a.lengths + b0;
    return s;
}
// launch(call, first sequence) of as many sequences at a time as a grid has rows
template <typename F> static int by_sequences(const el_conv_t& a, F launch) {
    constexpr int ROWS = 65535;
    if (a.batch <= ROWS) return launch(a, 0);
    for (long long b0 = 0; b0 < a.batch; b0 += ROWS) {
        const int rc = launch(conv_sequences(a, (int)b0, (int)(a.batch - b0 < ROWS ? a.batch - b0 : ROWS)), (int)b0);
        if (rc != EL_OK) return rc;
    }
    return EL_OK;
}

int launch_causal_conv(const el_conv_t& a, cudaStream_t st) {
    constexpr int V = CONV_V;
    const int strip = conv_strip(a, 64, FW_STRIPS);
    const unsigned blocks_t = ceil_div(a.length > 0 ? a.length : 1, (long long)strip * FW_STRIPS);
    const dim3 block(CONV_LANES, FW_STRIPS);
    const size_t shared = (size_t)CONV_SLOTS * CONV_LANES * FW_STRIPS * V * (a.dtype == EL_F32 ? 4 : 2);        // 16 KB at most
    const bool al = a.channels % V == 0 && vectors(a.x, a.x_stride_b, a.x_stride_t, a.dtype, V) && vectors(a.y, 0, 0, a.dtype, V) &&
                    vectors(a.initial_state, 0, 0, a.dtype, V) && vectors(a.final_state, 0, 0, a.dtype, V);
    return by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            return by_sequences(a, [&](const el_conv_t& part, int) {
                const dim3 grid(ceil_div(a.channels, CONV_LANES * V), blocks_t, part.batch);
                if (al) causal_conv_kernel<T, W, true><<<grid, block, shared, st>>>(part, strip);
                else causal_conv_kernel<T, W, false><<<grid, block, shared, st>>>(part, strip);
                return check_launch();
            });
        });
    });
}

int launch_causal_conv_backward(const el_conv_t& a, cudaStream_t st) {
    const ConvBackwardPlan plan = conv_backward_plan(a);
    const dim3 block(CONV_LANES, BW_STRIPS);
    const bool sums = a.dweight || a.dbias;
    float* partial = sums ? static_cast<float*>(a.workspace) : nullptr;
    const bool al = a.channels % 4 == 0 && vectors(a.x, a.x_stride_b, a.x_stride_t, a.dtype, 4) && vectors(a.dy, a.dy_stride_b, a.dy_stride_t, a.dtype, 4) &&
                    vectors(a.dx, 0, 0, a.dtype, 4) && vectors(a.initial_state, 0, 0, a.dtype, 4) && vectors(a.d_initial_state, 0, 0, a.dtype, 4) &&
                    vectors(a.d_final_state, 0, 0, a.dtype, 4);
    // slots and sums: 84 KB at most (float32)
    const size_t shared = (size_t)2 * CONV_SLOTS * CONV_LANES * BW_STRIPS * CONV_V * (a.dtype == EL_F32 ? 4 : 2) +
                          (size_t)BW_STRIPS * (a.width + 1) * CONV_LANES * CONV_V * sizeof(float);
    const int rc = a.batch == 0 ? EL_OK : by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            auto launch = [&](auto kernel, DeviceOnce& once) {
                int dev = 0;
                EL_CUDA_TRY(cudaGetDevice(&dev));
                if (!once.is_done(dev)) {
                    EL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024));
                    once.mark(dev);
                }
                return by_sequences(a, [&](const el_conv_t& part, int b0) {
                    const dim3 grid(ceil_div(a.channels, CONV_LANES * 4), plan.blocks_t, part.batch);
                    kernel<<<grid, block, shared, st>>>(part, plan.strip, partial ? partial + (size_t)b0 * plan.blocks_t * (a.width + 1) * a.channels : nullptr);
                    return check_launch();
                });
            };
            static DeviceOnce once[2];
            return al ? launch(causal_conv_backward_kernel<T, W, true>, once[0]) : launch(causal_conv_backward_kernel<T, W, false>, once[1]);
        });
    });
    if (rc != EL_OK || !sums) return rc;
    return launch_column_sums(partial, a.batch * plan.blocks_t, (a.width + 1) * a.channels, ConvSums{a.dweight, a.dbias, a.channels, a.width}, st);
}

int launch_causal_conv_step(const el_conv_t& a, cudaStream_t st) {
    return by_type(a.dtype, [&](auto t) {
        return by_width(a.width, [&](auto w) {
            return by_sequences(a, [&](const el_conv_t& part, int) {
                causal_conv_step_kernel<decltype(t), decltype(w)::value><<<dim3(ceil_div(a.channels, 128), part.batch), 128, 0, st>>>(part);
                return check_launch();
            });
        });
    });
}

}  // namespace el
