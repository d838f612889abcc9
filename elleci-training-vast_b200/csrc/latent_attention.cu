// Attention in the expanded form of latent attention, forward and backward, for every type and head size up to 256: float32 on the CUDA cores.
//
//   s[i,j] = scale * (q[i] . k[j] + q_rot[i] . k_rot[j]),  p[i,:] = softmax of s[i,:] over the keys that query i sees,  out[i] = sum_j p[i,j] v[j]
//   dv[j] = sum_i p[i,j] dout[i],  ds[i,j] = p[i,j] (dout[i] . v[j] - delta[i]) scale,  delta[i] = dout[i] . out[i]
//   dq[i] = sum_j ds[i,j] k[j],  dk[j] = sum_i ds[i,j] q[i]  (the rotated parts alike; dk_rot is the sum over the heads)
//
// The forward pass keeps lse[i] = log2(sum_j 2^(s[i,j] log2 e)), from which the backward kernels form p again (+inf for a query that sees nothing:
// p = 0).  The tcgen05 kernels (latent_attention_tc.cu) take 16-bit types whose head sizes are multiples of 16; this file's take float32
// and the other sizes.  A block holds 64 rows (queries, or keys for dk and dv) and walks over tiles of the other side.  Bound: shared-memory reads,
// 8 for 16 multiply-adds.
#include "latent_common.cuh"

namespace el {

int launch_attention_tc(const el_attention_t& a, cudaStream_t st);
int launch_attention_backward_tc(const el_attention_t& a, const float* delta, float* rot_parts, cudaStream_t st);
bool attention_tc_takes(const el_attention_t& a, bool backward);
size_t attention_tc_workspace_bytes(const el_attention_t& a);

using namespace latent;

namespace {

constexpr int ROWS = 64;              // rows that a block holds
constexpr int THREADS = 256;
constexpr int MOST_DIM = 256;         // channels of a key (both parts) and of a value

// rows `first` .. of a matrix of two parts (content, rotated) into dst [rows][pitch], zeros from row `valid` on
template <typename T>
__device__ void load_rows(float* dst, int pitch, int rows, const T* x, long long stride, int dim, const T* rot, long long rot_stride, int rot_dim, int first, int valid) {
    const int all = dim + rot_dim;
    for (int i = threadIdx.x; i < rows * all; i += THREADS) {
        const int r = i / all, c = i - r * all;
        float v = 0.0f;
        if (first + r < valid) v = c < dim ? to_float(x[(first + r) * stride + c]) : to_float(rot[(first + r) * rot_stride + c - dim]);
        dst[r * pitch + c] = v;
    }
}

template <typename T> struct Heads {       // one head of one sequence
    const T *q, *q_rot, *k, *k_rot, *v;
    __device__ Heads(const el_attention_t& a, int b, int h) {
        q = static_cast<const T*>(a.q) + b * a.q_stride_b + h * a.q_stride_h;
        q_rot = static_cast<const T*>(a.q_rot) + b * a.q_rot_stride_b + h * a.q_rot_stride_h;
        k = static_cast<const T*>(a.k) + b * a.k_stride_b + h * a.k_stride_h;
        k_rot = static_cast<const T*>(a.k_rot) + b * a.k_rot_stride_b;
        v = static_cast<const T*>(a.v) + b * a.v_stride_b + h * a.v_stride_h;
    }
};

// A thread holds rows 4 ty .. 4 ty + 3; columns of the score tile and of the output are tx + 16 n.  Bound: the FMA pipes and shared memory's loads (float32, 2 x 1024
// tokens, 8 heads of 128 and 128 channels, causal: 620 us, the gradients 2040; 16-bit types that the tensor cores take: 30 and 67).
template <typename T>
__global__ void __launch_bounds__(THREADS) attention_rows_kernel(const el_attention_t a) {
    extern __shared__ float sm[];
    const int D = a.key_dim + a.rot_dim, V = a.value_dim, DP = D | 1, VP = V | 1;
    float* Q = sm;
    float* K = Q + ROWS * DP;
    float* Vs = K + ROWS * DP;
    float* P = Vs + ROWS * VP;                      // [64][65]
    const Place at(a);                              // the longest rows first
    const int b = at.batch, h = at.head, i0 = ((int)(lse_pitch(a.length) / ROWS) - 1 - at.tile) * ROWS;
    const Sequence seq(a, b);
    const Heads<T> in(a, b, h);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float to_log2 = a.scale * mamba::LOG2E;
    load_rows<T>(Q, DP, ROWS, in.q, a.q_stride_t, a.key_dim, in.q_rot, a.q_rot_stride_t, a.rot_dim, i0, seq.queries);
    float top[4], sum[4], o[4][MOST_DIM / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        top[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < MOST_DIM / 16; ++c) o[r][c] = 0.0f;
    }
    const int end = seq.key_end(i0 + ROWS);
    for (int j0 = 0; j0 < end; j0 += ROWS) {
        __syncthreads();
        load_rows<T>(K, DP, ROWS, in.k, a.k_stride_t, a.key_dim, in.k_rot, a.k_rot_stride_t, a.rot_dim, j0, seq.keys);
        load_rows<T>(Vs, VP, ROWS, in.v, a.v_stride_t, V, in.v, 0, 0, j0, seq.keys);
        __syncthreads();
        float s[4][4] = {};
        for (int d = 0; d < D; ++d) {
            float x[4], y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = Q[(4 * ty + r) * DP + d];
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = K[(tx + 16 * c) * DP + d];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[r][c] = fmaf(x[r], y[c], s[r][c]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 4 * ty + r;
            float m = top[r];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = seq.sees(i, j0 + tx + 16 * c) ? s[r][c] * to_log2 : -INFINITY;
                m = mamba::max_nan(m, s[r][c]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) m = mamba::max_nan(m, __shfl_xor_sync(0xffffffffu, m, w));
            const float from = m == -INFINITY ? 0.0f : m, old = exp2_neg(top[r] - from);
            top[r] = m;
            float t = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = exp2_neg(s[r][c] - from);
                t += p;
                P[(4 * ty + r) * 65 + tx + 16 * c] = p;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) t += __shfl_xor_sync(0xffffffffu, t, w);
            sum[r] = fmaf(sum[r], old, t);
#pragma unroll
            for (int c = 0; c < MOST_DIM / 16; ++c) o[r][c] *= old;
        }
        __syncwarp();                               // a row of P is written and read by the same half warp
        const int n = seq.keys - j0 < ROWS ? seq.keys - j0 : ROWS;
        for (int j = 0; j < n; ++j) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) p[r] = P[(4 * ty + r) * 65 + j];
#pragma unroll
            for (int c = 0; c < MOST_DIM / 16; ++c) {
                if (16 * c >= V) break;
                const float v = tx + 16 * c < V ? Vs[j * VP + tx + 16 * c] : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r][c] = fmaf(p[r], v, o[r][c]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * ty + r;
        const bool empty = top[r] == -INFINITY;      // also the padding
        const float inv = 1.0f / sum[r];
        if (a.lse && tx == 0) a.lse[((long long)b * a.heads + h) * lse_pitch(a.length) + i] = empty ? INFINITY : top[r] + log2f(sum[r]);
        if (i >= a.length) continue;
        T* out = static_cast<T*>(a.out) + (((long long)b * a.length + i) * a.heads + h) * V;
#pragma unroll
        for (int c = 0; c < MOST_DIM / 16; ++c)
            if (tx + 16 * c < V) {
                const float x = empty ? 0.0f : o[r][c] * inv;
                out[tx + 16 * c] = mamba::from_float<T>(x);
                if constexpr (sizeof(T) == 2)
                    if (a.out_rest) a.out_rest[out - static_cast<T*>(a.out) + tx + 16 * c] = (int8_t)(rest_of<T>(x, to_float(mamba::from_float<T>(x))) >> 8);
            }
    }
}

// delta[b,h,i] = dout[i] . out[i] (with what rounding took from out, where it is kept: an error of delta goes to all of a row's ds alike), zeros for padding.  A block takes 8 tokens of up to 32 heads, whose values lie side by side (15.5 us; rows of one head, 256 bytes
// of every 8 KB, took 26), and writes 8 tokens of a head at a time.  `lanes` threads (a power of two from 2 to 32, 8 values each) take a row, and 4 rows
// are on their way at once.  VEC: 8 values are vectors on 16 bytes.  Bound: memory (4 x 1024 tokens, 32 heads of 128: 67 MB and 17 MB of rests, 19 us with cold caches).
constexpr int DELTA_TOKENS = 8, DELTA_HEADS = 32;
template <typename T, bool VEC, bool REST>
__global__ void __launch_bounds__(THREADS) attention_delta_kernel(const el_attention_t a, float* __restrict__ delta, int lanes, int head_bits) {
    __shared__ float sums[DELTA_TOKENS * DELTA_HEADS];
    const int groups = THREADS / lanes, part = threadIdx.x & (lanes - 1), heads = 1 << head_bits, rows = DELTA_TOKENS << head_bits, c = part * 8, V = a.value_dim;
    const long long pitch = lse_pitch(a.length);
    const unsigned per = (unsigned)(pitch / DELTA_TOKENS), groups_of_heads = (a.heads + heads - 1) >> head_bits, tile = blockIdx.x / groups_of_heads, b = tile / per;
    const int t0 = (int)(tile - b * per) * DELTA_TOKENS, h0 = (int)(blockIdx.x - tile * groups_of_heads) * heads, live = length_of(a.lengths, b, a.length, a.length);
    const T *out0 = static_cast<const T*>(a.out), *dout0 = static_cast<const T*>(a.dout);
    const T *out = out0 + ((long long)b * a.length + t0) * a.heads * V, *dout = dout0 + b * a.dout_stride_b + t0 * a.dout_stride_t;
    if (V == 0 || t0 >= live) {
        for (int i = threadIdx.x; i < rows; i += THREADS)
            if (h0 + i / DELTA_TOKENS < a.heads) delta[((long long)b * a.heads + h0 + i / DELTA_TOKENS) * pitch + t0 + i % DELTA_TOKENS] = 0.0f;
        return;
    }
    for (int r0 = threadIdx.x / lanes; r0 - (int)threadIdx.x / lanes < rows; r0 += 4 * groups) {
        float s[4];
        bool there[4];
        const T *o[4], *g[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {                                  // (a row that is not there reads the first one)
            const int r = r0 + k * groups, t = r >> head_bits, h = h0 + (r & (heads - 1));
            there[k] = r < rows && t0 + t < live && h < a.heads && c < V;
            o[k] = there[k] ? out + ((long long)t * a.heads + h) * V + c : out0;
            g[k] = there[k] ? dout + t * a.dout_stride_t + h * a.dout_stride_h + c : dout0;
        }
        if constexpr (VEC) {
            constexpr int WORDS = sizeof(T) * 8 / 16;
            uint4 x[4][WORDS], y[4][WORDS];
            uint2 z[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int w = 0; w < WORDS; ++w) {
                    x[k][w] = reinterpret_cast<const uint4*>(o[k])[w];
                    y[k][w] = reinterpret_cast<const uint4*>(g[k])[w];
                }
                if constexpr (REST) z[k] = *reinterpret_cast<const uint2*>(a.out_rest + (o[k] - out0));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const T *xs = reinterpret_cast<const T*>(x[k]), *ys = reinterpret_cast<const T*>(y[k]);
                s[k] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float v = to_float(xs[e]);
                    if constexpr (REST) v = with_rest<T>(v, e < 4 ? z[k].x : z[k].y, e & 3);
                    s[k] = fmaf(v, to_float(ys[e]), s[k]);
                }
            }
        } else {
            for (int k = 0; k < 4; ++k) {
                s[k] = 0.0f;
                for (int e = 0; e < 8 && c + e < V; ++e) {
                    float v = to_float(o[k][e]);
                    if constexpr (REST) v = with_rest<T>(v, (uint8_t)a.out_rest[o[k] - out0 + e], 0);
                    s[k] = fmaf(v, to_float(g[k][e]), s[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (!there[k]) s[k] = 0.0f;
        for (int w = lanes / 2; w > 0; w >>= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + k * groups;
            if (part == 0 && r < rows) sums[(r & (heads - 1)) * DELTA_TOKENS + (r >> head_bits)] = s[k];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows; i += THREADS) {
        const int h = h0 + i / DELTA_TOKENS;
        if (h < a.heads) delta[((long long)b * a.heads + h) * pitch + t0 + i % DELTA_TOKENS] = sums[i];
    }
}

// KEYS: the block holds 64 keys, walks over the queries and forms dk and dv; otherwise it holds 64 queries, walks over the keys and forms dq.
// The held side's two matrices (k and v, or q and dout) are A1 and A2, the other side's B1 and B2: s = A1 B1', dp = A2 B2'.
template <typename T, bool KEYS>
__global__ void __launch_bounds__(THREADS) attention_backward_rows_kernel(const el_attention_t a, const float* __restrict__ delta, float* __restrict__ rot_parts) {
    constexpr int STEP = 32;
    extern __shared__ float sm[];
    const int D = a.key_dim + a.rot_dim, V = a.value_dim, DP = D | 1, VP = V | 1;
    float* A1 = sm;
    float* A2 = A1 + ROWS * DP;
    float* B1 = A2 + ROWS * VP;
    float* B2 = B1 + STEP * DP;
    float* P = B2 + STEP * VP;                      // [64][33]
    float* G = P + ROWS * 33;
    const Place at(a);
    const int b = at.batch, h = at.head, r0 = at.tile * ROWS;
    const Sequence seq(a, b);
    const Heads<T> in(a, b, h);
    const T* g = static_cast<const T*>(a.dout) + b * a.dout_stride_b + h * a.dout_stride_h;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const float to_log2 = a.scale * mamba::LOG2E;
    const long long stats = ((long long)b * a.heads + h) * lse_pitch(a.length);
    if (KEYS) {
        load_rows<T>(A1, DP, ROWS, in.k, a.k_stride_t, a.key_dim, in.k_rot, a.k_rot_stride_t, a.rot_dim, r0, seq.keys);
        load_rows<T>(A2, VP, ROWS, in.v, a.v_stride_t, V, in.v, 0, 0, r0, seq.keys);
    } else {
        load_rows<T>(A1, DP, ROWS, in.q, a.q_stride_t, a.key_dim, in.q_rot, a.q_rot_stride_t, a.rot_dim, r0, seq.queries);
        load_rows<T>(A2, VP, ROWS, g, a.dout_stride_t, V, g, 0, 0, r0, seq.queries);
    }
    float d1[4][MOST_DIM / 16], d2[4][KEYS ? MOST_DIM / 16 : 1];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int c = 0; c < MOST_DIM / 16; ++c) d1[r][c] = 0.0f;
#pragma unroll
        for (int c = 0; c < (KEYS ? MOST_DIM / 16 : 1); ++c) d2[r][c] = 0.0f;
    }
    const int begin = KEYS ? (r0 < seq.keys ? seq.query_begin(r0) / STEP * STEP : seq.queries) : 0, end = KEYS ? seq.queries : seq.key_end(r0 + ROWS);
    for (int c0 = begin; c0 < end; c0 += STEP) {
        __syncthreads();
        if (KEYS) {
            load_rows<T>(B1, DP, STEP, in.q, a.q_stride_t, a.key_dim, in.q_rot, a.q_rot_stride_t, a.rot_dim, c0, seq.queries);
            load_rows<T>(B2, VP, STEP, g, a.dout_stride_t, V, g, 0, 0, c0, seq.queries);
        } else {
            load_rows<T>(B1, DP, STEP, in.k, a.k_stride_t, a.key_dim, in.k_rot, a.k_rot_stride_t, a.rot_dim, c0, seq.keys);
            load_rows<T>(B2, VP, STEP, in.v, a.v_stride_t, V, in.v, 0, 0, c0, seq.keys);
        }
        __syncthreads();
        float s[4][2] = {}, dp[4][2] = {};
        for (int d = 0; d < D; ++d) {
            const float y0 = B1[tx * DP + d], y1 = B1[(tx + 16) * DP + d];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = A1[(4 * ty + r) * DP + d];
                s[r][0] = fmaf(x, y0, s[r][0]);
                s[r][1] = fmaf(x, y1, s[r][1]);
            }
        }
        for (int d = 0; d < V; ++d) {
            const float y0 = B2[tx * VP + d], y1 = B2[(tx + 16) * VP + d];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = A2[(4 * ty + r) * VP + d];
                dp[r][0] = fmaf(x, y0, dp[r][0]);
                dp[r][1] = fmaf(x, y1, dp[r][1]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = r0 + 4 * ty + r, col = c0 + tx + 16 * c, i = KEYS ? col : row, j = KEYS ? row : col;
                float p = 0.0f, ds = 0.0f;
                if (seq.sees(i, j)) {
                    p = exp2_neg(fmaf(s[r][c], to_log2, -a.lse[stats + i]));
                    ds = p * (dp[r][c] - delta[stats + i]) * a.scale;
                }
                if (KEYS) P[(4 * ty + r) * 33 + tx + 16 * c] = p;
                G[(4 * ty + r) * 33 + tx + 16 * c] = ds;
            }
        __syncwarp();
        for (int c = 0; c < STEP; ++c) {
            float x[4], y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = G[(4 * ty + r) * 33 + c];
                y[r] = KEYS ? P[(4 * ty + r) * 33 + c] : 0.0f;
            }
#pragma unroll
            for (int n = 0; n < MOST_DIM / 16; ++n) {
                if (16 * n >= D) break;
                const float z = tx + 16 * n < D ? B1[c * DP + tx + 16 * n] : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) d1[r][n] = fmaf(x[r], z, d1[r][n]);
            }
            if (KEYS) {
#pragma unroll
                for (int n = 0; n < (KEYS ? MOST_DIM / 16 : 1); ++n) {
                    if (16 * n >= V) break;
                    const float z = tx + 16 * n < V ? B2[c * VP + tx + 16 * n] : 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) d2[r][n] = fmaf(y[r], z, d2[r][n]);
                }
            }
        }
    }
    const int all = KEYS ? a.keys : a.length, live = KEYS ? seq.keys : seq.queries;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const long long row = r0 + 4 * ty + r;
        if (row >= all) continue;
#pragma unroll
        for (int n = 0; n < MOST_DIM / 16; ++n) {
            const int c = tx + 16 * n;
            if (c >= D) continue;
            const float v = row < live ? d1[r][n] : 0.0f;
            if (KEYS) {
                if (c < a.key_dim) {
                    if (a.dk) static_cast<T*>(a.dk)[b * a.dk_stride_b + row * a.dk_stride_t + h * a.dk_stride_h + c] = mamba::from_float<T>(v);
                } else if (rot_parts) {
                    rot_parts[((b * (long long)a.heads + h) * a.keys + row) * a.rot_dim + c - a.key_dim] = v;
                }
            } else {
                const long long to = (b * (long long)a.length + row) * a.heads + h;
                if (c < a.key_dim) {
                    if (a.dq) static_cast<T*>(a.dq)[to * a.key_dim + c] = mamba::from_float<T>(v);
                } else if (a.dq_rot) {
                    static_cast<T*>(a.dq_rot)[to * a.rot_dim + c - a.key_dim] = mamba::from_float<T>(v);
                }
            }
        }
        if (KEYS && a.dv) {
#pragma unroll
            for (int n = 0; n < (KEYS ? MOST_DIM / 16 : 1); ++n) {
                const int c = tx + 16 * n;
                if (c < V) static_cast<T*>(a.dv)[b * a.dv_stride_b + row * a.dv_stride_t + h * a.dv_stride_h + c] = mamba::from_float<T>(row < live ? d2[r][n] : 0.0f);
            }
        }
    }
}

// dk_rot[b,j,c] = sum over the heads of parts[b,h,j,c], in their order.  A value a thread: 4 values a thread leave too few loads on their way (12 us and 9.3 us
// for 32 heads' parts of 4 x 1024 x 64).
template <typename T>
__global__ void __launch_bounds__(THREADS) attention_rot_sum_kernel(const float* __restrict__ parts, T* __restrict__ out, int heads, long long per_head, long long n) {
    const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (i >= n) return;
    const long long b = i / per_head, at = i - b * per_head;
    const float* p = parts + b * heads * per_head + at;
    float s = 0.0f;
#pragma unroll 8
    for (int h = 0; h < heads; ++h) s += p[h * per_head];
    out[i] = mamba::from_float<T>(s);
}

template <typename F> int of_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}

template <typename K> int allow_shared(K kernel, int bytes, DeviceOnce& once) {
    int dev = 0;
    EL_CUDA_TRY(cudaGetDevice(&dev));
    if (!once.is_done(dev)) {
        EL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        once.mark(dev);
    }
    return EL_OK;
}

int forward_bytes(int D, int V) { return 4 * (2 * ROWS * (D | 1) + ROWS * (V | 1) + ROWS * 65); }
int backward_bytes(int D, int V) { return 4 * ((ROWS + 32) * ((D | 1) + (V | 1)) + 2 * ROWS * 33); }

size_t align16(size_t n) { return (n + 15) / 16 * 16; }
size_t delta_bytes(const el_attention_t& a) { return align16((size_t)a.batch * a.heads * lse_pitch(a.length) * 4); }

}  // namespace

size_t attention_lse_bytes(const el_attention_t& a) { return (size_t)a.batch * a.heads * lse_pitch(a.length) * 4; }
size_t attention_workspace_bytes(const el_attention_t& a) { return attention_tc_takes(a, false) ? attention_tc_workspace_bytes(a) : 0; }
size_t attention_backward_workspace_bytes(const el_attention_t& a) {
    return delta_bytes(a) + (a.dk_rot ? align16((size_t)a.batch * a.heads * a.keys * a.rot_dim * 4) : 0);
}

int launch_attention(const el_attention_t& a, cudaStream_t st) {
    if (attention_tc_takes(a, false)) return launch_attention_tc(a, st);
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        static DeviceOnce once;
        const int rc = allow_shared(attention_rows_kernel<T>, forward_bytes(MOST_DIM, MOST_DIM), once);
        if (rc != EL_OK) return rc;
        // every row of the padded log sums is written
        attention_rows_kernel<T><<<blocks_of(a, (int)lse_pitch(a.length), ROWS), THREADS, forward_bytes(a.key_dim + a.rot_dim, a.value_dim), st>>>(a);
        return check_launch();
    });
}

int launch_attention_backward(const el_attention_t& a, cudaStream_t st) {
    float* delta = static_cast<float*>(a.workspace);
    float* rot_parts = a.dk_rot ? reinterpret_cast<float*>(static_cast<char*>(a.workspace) + delta_bytes(a)) : nullptr;
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.length > 0) {
            int lanes = 2;
            while (lanes < 32 && lanes * 8 < a.value_dim) lanes *= 2;
            const long long e = 16 / (int)sizeof(T);
            const bool vec = a.value_dim % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && reinterpret_cast<uintptr_t>(a.dout) % 16 == 0 &&
                             a.dout_stride_b % e == 0 && a.dout_stride_t % e == 0 && a.dout_stride_h % e == 0;
            int head_bits = 0;
            while (1 << head_bits < a.heads && 1 << head_bits < DELTA_HEADS) ++head_bits;
            const unsigned grid = (unsigned)(a.batch * (lse_pitch(a.length) / DELTA_TOKENS) * ((a.heads + (1 << head_bits) - 1) >> head_bits));
            auto run = [&](auto v, auto rest) {
                attention_delta_kernel<T, decltype(v)::value, decltype(rest)::value><<<grid, THREADS, 0, st>>>(a, delta, lanes, head_bits);
            };
            auto form = [&](auto rest) { vec ? run(std::true_type(), rest) : run(std::false_type(), rest); };
            if constexpr (sizeof(T) == 2) a.out_rest ? form(std::true_type()) : form(std::false_type());
            else form(std::false_type());
            int rc = check_launch();
            if (rc != EL_OK) return rc;
        }
        int rc = EL_OK;
        if (attention_tc_takes(a, true)) {
            rc = launch_attention_backward_tc(a, delta, rot_parts, st);
            if (rc != EL_OK) return rc;
        } else {
            const int bytes = backward_bytes(a.key_dim + a.rot_dim, a.value_dim);
            static DeviceOnce once[2];
            if ((a.dk || a.dv || a.dk_rot) && a.keys > 0) {
                rc = allow_shared(attention_backward_rows_kernel<T, true>, backward_bytes(MOST_DIM, MOST_DIM), once[0]);
                if (rc != EL_OK) return rc;
                attention_backward_rows_kernel<T, true><<<blocks_of(a, a.keys, ROWS), THREADS, bytes, st>>>(a, delta, rot_parts);
                if ((rc = check_launch()) != EL_OK) return rc;
            }
            if ((a.dq || a.dq_rot) && a.length > 0) {
                rc = allow_shared(attention_backward_rows_kernel<T, false>, backward_bytes(MOST_DIM, MOST_DIM), once[1]);
                if (rc != EL_OK) return rc;
                attention_backward_rows_kernel<T, false><<<blocks_of(a, a.length, ROWS), THREADS, bytes, st>>>(a, delta, rot_parts);
                if ((rc = check_launch()) != EL_OK) return rc;
            }
        }
        if (!a.dk_rot || a.keys == 0) return rc;
        const long long per_head = (long long)a.keys * a.rot_dim, n = a.batch * per_head;
        attention_rot_sum_kernel<T><<<(unsigned)((n + THREADS - 1) / THREADS), THREADS, 0, st>>>(rot_parts, static_cast<T*>(a.dk_rot), a.heads, per_head, n);
        return check_launch();
    });
}

}  // namespace el
