// Selective state space scan: forward, backward and single token.
//
//   delta = softplus(dt + bias),  h[t] = exp(delta A[n]) h[t-1] + delta u B[n],  y = (sum_n C[n] h[t] + D u) z sigmoid(z)
//
// backward, with dyg = dy z sigmoid(z) and g[t] = C[t] dyg[t] + a[t+1] g[t+1] (a = exp(delta A)), the gradient of the state after token t:
//   dA = sum_t delta w,  w = g a h[t-1];   ddelta = sum_n A w + u sum_n g B;   ddt = ddelta sigmoid(dt + bias)
//   du = D dyg + delta sum_n g B;   dB = sum_d g delta u;   dC = sum_d dyg h;   dz = dy yn slope(z) for the ungated yn
// The states before every TILE-th token are kept by the forward pass; backward forms the states of a tile again from them.
//
// A thread owns one channel of one sequence and all its states, and walks over the tokens.
#include "mamba_common.cuh"

namespace el {
using namespace mamba;

constexpr int TILE = 16;              // tokens from one kept state to the next

struct Token { float delta, raw, u, z; };

template <typename T>
__device__ __forceinline__ Token scan_token(const el_scan_t& a, int b, int t, int d, float bias) {
    Token k;
    k.u = to_float<T>(static_cast<const T*>(a.u)[b * a.u_stride_b + t * a.u_stride_t + d]);
    k.raw = to_float<T>(static_cast<const T*>(a.dt)[b * a.dt_stride_b + t * a.dt_stride_t + d]) + bias;
    k.delta = a.softplus ? softplus_of(k.raw, exp_minus_abs(k.raw)) : k.raw;
    k.z = a.z ? to_float<T>(static_cast<const T*>(a.z)[b * a.z_stride_b + t * a.z_stride_t + d]) : 0.0f;
    return k;
}
__device__ __forceinline__ int live_tokens(const el_scan_t& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length; }

template <typename T, int NS>
__global__ void __launch_bounds__(64)
selective_scan_kernel(const el_scan_t a) {
    const int d = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y, N = a.states;
    if (d >= a.channels) return;
    const int g = d / (a.channels / a.groups), n_live = live_tokens(a, b);
    const long long state_at = ((long long)b * a.channels + d) * N;
    float h[NS], A[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        h[n] = a.initial_state && n < N ? a.initial_state[state_at + n] : 0.0f;
        A[n] = n < N ? a.A[(long long)d * N + n] * LOG2E : 0.0f;
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, D = a.D ? a.D[d] : 0.0f;
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_stride_b + g * a.B_stride_g;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_stride_b + g * a.C_stride_g;
    T* y = static_cast<T*>(a.y) + (long long)b * a.length * a.channels + d;
    const int tiles = (a.length + TILE - 1) / TILE;
    for (int t = 0; t < a.length; ++t) {
        if (a.checkpoints && t % TILE == 0) {
            float* c = a.checkpoints + (((long long)b * tiles + t / TILE) * a.channels + d) * N;
            for (int n = 0; n < NS; ++n)
                if (n < N) c[n] = h[n];
        }
        float out = 0.0f;
        if (t < n_live) {
            const Token k = scan_token<T>(a, b, t, d, bias);
            out = D * k.u;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (n < N) {
                    const float B = to_float<T>(Bp[t * a.B_stride_t + n]), C = to_float<T>(Cp[t * a.C_stride_t + n]);
                    h[n] = __fmaf_rn(ex2(k.delta * A[n]), h[n], k.delta * k.u * B);
                    out = __fmaf_rn(C, h[n], out);
                }
            }
            if (a.z) out *= k.z * sigmoid(k.z);
        }
        y[(long long)t * a.channels] = from_float<T>(out);
    }
    if (a.final_state) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n < N) a.final_state[state_at + n] = h[n];
    }
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A warp: 32 channels of one group.  partial_bc: [warps of a group][2][batch][length][groups][states]; partial_a: [batch][channels][states + 2]
template <typename T, int NS>
__global__ void __launch_bounds__(32)
selective_scan_backward_kernel(const el_scan_t a, float* __restrict__ partial_bc, float* __restrict__ partial_a) {
    const int per_group = a.channels / a.groups, parts = (per_group + 31) / 32, N = a.states;
    const int g = blockIdx.x / parts, part = blockIdx.x % parts, b = blockIdx.y;
    const int in_group = part * 32 + threadIdx.x;
    const bool real = in_group < per_group;
    const int d = g * per_group + min(in_group, per_group - 1);
    const int n_live = live_tokens(a, b);
    const long long state_at = ((long long)b * a.channels + d) * N;
    float A[NS], adj[NS], dA[NS] = {}, dD = 0.0f, dbias = 0.0f;
    for (int n = 0; n < NS; ++n) {
        A[n] = n < N ? a.A[(long long)d * N + n] : 0.0f;
        adj[n] = a.d_final_state && n < N ? a.d_final_state[state_at + n] : 0.0f;
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, D = a.D ? a.D[d] : 0.0f;
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_stride_b + g * a.B_stride_g;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_stride_b + g * a.C_stride_g;
    const long long out_at = (long long)b * a.length * a.channels + d;
    const int tiles = (a.length + TILE - 1) / TILE;
    const long long bc_all = (long long)a.batch * a.length * a.groups * N;
    float* pb = partial_bc + (long long)part * 2 * bc_all + ((long long)b * a.length * a.groups + g) * N;
    for (int tile = tiles - 1; tile >= 0; --tile) {
        float hs[TILE + 1][NS];
        const float* c = a.checkpoints + (((long long)b * tiles + tile) * a.channels + d) * N;
        for (int n = 0; n < N; ++n) hs[0][n] = c[n];
        for (int i = 0; i < TILE; ++i) {
            const int t = tile * TILE + i;
            if (t < n_live) {
                const Token k = scan_token<T>(a, b, t, d, bias);
                for (int n = 0; n < N; ++n)
                    hs[i + 1][n] = __fmaf_rn(ex2(k.delta * (A[n] * LOG2E)), hs[i][n], k.delta * k.u * to_float<T>(Bp[t * a.B_stride_t + n]));
            }
        }
        for (int i = TILE - 1; i >= 0; --i) {
            const int t = tile * TILE + i;
            if (t >= a.length) continue;
            float du = 0.0f, ddt = 0.0f, dz = 0.0f;
            if (t < n_live) {
                const Token k = scan_token<T>(a, b, t, d, bias);
                const float dy = a.dy ? to_float<T>(static_cast<const T*>(a.dy)[b * a.dy_stride_b + t * a.dy_stride_t + d]) : 0.0f;
                const float s = sigmoid(k.z), dyg = a.z ? dy * k.z * s : dy;
                float y = D * k.u, gb = 0.0f, wa = 0.0f;
                for (int n = 0; n < N; ++n) {
                    const float B = to_float<T>(Bp[t * a.B_stride_t + n]), C = to_float<T>(Cp[t * a.C_stride_t + n]);
                    y = __fmaf_rn(C, hs[i + 1][n], y);
                    const float gn = __fmaf_rn(C, dyg, adj[n]), ag = ex2(k.delta * (A[n] * LOG2E)) * gn, w = ag * hs[i][n];
                    gb = __fmaf_rn(gn, B, gb);
                    wa = __fmaf_rn(w, A[n], wa);
                    dA[n] = __fmaf_rn(w, k.delta, dA[n]);
                    adj[n] = ag;
                    const float dB = warp_sum_f(real ? gn * (k.delta * k.u) : 0.0f), dC = warp_sum_f(real ? dyg * hs[i + 1][n] : 0.0f);
                    if (threadIdx.x == 0) {
                        pb[(long long)t * a.groups * N + n] = dB;
                        pb[bc_all + (long long)t * a.groups * N + n] = dC;
                    }
                }
                du = __fmaf_rn(D, dyg, k.delta * gb);
                ddt = __fmaf_rn(k.u, gb, wa);
                if (a.softplus) ddt *= sigmoid(k.raw);
                if (a.z) dz = dy * y * silu_slope(k.z, s);
                dD = __fmaf_rn(dyg, k.u, dD);
                dbias += ddt;
            } else if (threadIdx.x == 0) {
                for (int n = 0; n < N; ++n) pb[(long long)t * a.groups * N + n] = pb[bc_all + (long long)t * a.groups * N + n] = 0.0f;
            }
            if (real) {
                const long long at = out_at + (long long)t * a.channels;
                if (a.du) static_cast<T*>(a.du)[at] = from_float<T>(du);
                if (a.ddt) static_cast<T*>(a.ddt)[at] = from_float<T>(ddt);
                if (a.dz && a.z) static_cast<T*>(a.dz)[at] = from_float<T>(dz);
            }
        }
    }
    if (!real) return;
    float* pa = partial_a + ((long long)b * a.channels + d) * (N + 2);
    for (int n = 0; n < N; ++n) {
        pa[n] = dA[n];
        if (a.d_initial_state) a.d_initial_state[state_at + n] = adj[n];
    }
    pa[N] = dD;
    pa[N + 1] = dbias;
}

template <typename T>
__global__ void __launch_bounds__(256)
scan_bc_sums_kernel(const float* __restrict__ partial, int parts, long long all, T* __restrict__ dB, T* __restrict__ dC) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= all) return;
    float b = 0.0f, c = 0.0f;
    for (int p = 0; p < parts; ++p) {
        b += partial[2 * p * all + i];
        c += partial[(2 * p + 1) * all + i];
    }
    if (dB) dB[i] = from_float<T>(b);
    if (dC) dC[i] = from_float<T>(c);
}

static __global__ void __launch_bounds__(256)
scan_a_sums_kernel(const float* __restrict__ partial, int batch, int channels, int N, float* __restrict__ dA, float* __restrict__ dD,
                   float* __restrict__ dbias) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)channels * (N + 2);
    if (i >= all) return;
    float s = 0.0f;
    for (int b = 0; b < batch; ++b) s += partial[b * all + i];
    const int d = (int)(i / (N + 2)), n = (int)(i % (N + 2));
    if (n < N) { if (dA) dA[(long long)d * N + n] = s; }
    else if (n == N) { if (dD) dD[d] = s; }
    else if (dbias) dbias[d] = s;
}

// One token: a thread owns a channel's state.
template <typename T>
__global__ void __launch_bounds__(128)
selective_scan_step_kernel(const el_scan_t a) {
    const int d = blockIdx.x * 128 + threadIdx.x, b = blockIdx.y, N = a.states;
    if (d >= a.channels) return;
    const int g = d / (a.channels / a.groups);
    const long long state_at = ((long long)b * a.channels + d) * N;
    const Token k = scan_token<T>(a, b, 0, d, a.dt_bias ? a.dt_bias[d] : 0.0f);
    const T* Bp = static_cast<const T*>(a.B) + b * a.B_stride_b + g * a.B_stride_g;
    const T* Cp = static_cast<const T*>(a.C) + b * a.C_stride_b + g * a.C_stride_g;
    float out = a.D ? a.D[d] * k.u : 0.0f;
    for (int n = 0; n < N; ++n) {
        const float h = __fmaf_rn(ex2(k.delta * (a.A[(long long)d * N + n] * LOG2E)), a.initial_state[state_at + n], k.delta * k.u * to_float<T>(Bp[n]));
        out = __fmaf_rn(to_float<T>(Cp[n]), h, out);
        a.final_state[state_at + n] = h;
    }
    if (a.z) out *= k.z * sigmoid(k.z);
    static_cast<T*>(a.y)[(long long)b * a.channels + d] = from_float<T>(out);
}

// ---- host side ----------------------------------------------------------------------------------------------------------

template <typename F> static int scan_by_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}
template <typename F> static int scan_by_states(int N, F f) {
    if (N <= 16) return f(std::integral_constant<int, 16>());
    return f(std::integral_constant<int, 64>());
}

size_t selective_scan_checkpoint_bytes(const el_scan_t& a) {
    return (size_t)a.batch * ((a.length + TILE - 1) / TILE) * a.channels * a.states * sizeof(float);
}
size_t selective_scan_workspace_bytes(const el_scan_t&) { return 0; }
static int scan_parts(const el_scan_t& a) { return (a.channels / a.groups + 31) / 32; }
size_t selective_scan_backward_workspace_bytes(const el_scan_t& a) {
    return ((size_t)2 * scan_parts(a) * a.batch * a.length * a.groups * a.states + (size_t)a.batch * a.channels * (a.states + 2)) * sizeof(float);
}

int launch_selective_scan(const el_scan_t& a, cudaStream_t st) {
    if (a.batch > 65535) return EL_ERR_TOO_LARGE;
    return scan_by_type(a.dtype, [&](auto t) {
        return scan_by_states(a.states, [&](auto n) {
            selective_scan_kernel<decltype(t), decltype(n)::value><<<dim3((a.channels + 63) / 64, a.batch), 64, 0, st>>>(a);
            return check_launch();
        });
    });
}

int launch_selective_scan_backward(const el_scan_t& a, cudaStream_t st) {
    if (a.batch > 65535) return EL_ERR_TOO_LARGE;
    const long long all = (long long)a.batch * a.length * a.groups * a.states;
    const int parts = scan_parts(a);
    float* partial_bc = static_cast<float*>(a.workspace);
    float* partial_a = partial_bc + 2 * parts * all;
    return scan_by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const int rc = a.batch == 0 ? EL_OK : scan_by_states(a.states, [&](auto n) {
            selective_scan_backward_kernel<T, decltype(n)::value><<<dim3(a.groups * parts, a.batch), 32, 0, st>>>(a, partial_bc, partial_a);
            return check_launch();
        });
        if (rc != EL_OK) return rc;
        if ((a.dB || a.dC) && all > 0)
            scan_bc_sums_kernel<T><<<(unsigned)((all + 255) / 256), 256, 0, st>>>(partial_bc, parts, all, static_cast<T*>(a.dB), static_cast<T*>(a.dC));
        const long long cols = (long long)a.channels * (a.states + 2);
        if (a.dA || a.dD || a.ddt_bias)
            scan_a_sums_kernel<<<(unsigned)((cols + 255) / 256), 256, 0, st>>>(partial_a, a.batch, a.channels, a.states, a.dA, a.dD, a.ddt_bias);
        return check_launch();
    });
}

int launch_selective_scan_step(const el_scan_t& a, cudaStream_t st) {
    if (a.batch > 65535) return EL_ERR_TOO_LARGE;
    return scan_by_type(a.dtype, [&](auto t) {
        selective_scan_step_kernel<decltype(t)><<<dim3((a.channels + 127) / 128, a.batch), 128, 0, st>>>(a);
        return check_launch();
    });
}

}  // namespace el
