// One token for every sequence against the cache of latent vectors (the absorbed form of latent attention).
//
// A key is k[j] = gamma W_k c[j] with the latent vector c[j] = absmax[j] / 127 * row[j], so q . k[j] = (gamma W_k' q) . c[j]: the query goes into the
// latent space once, the keys and values are never formed, and a token costs its own row and rotated part, read once for all heads.
//
//   query   u[h] = scale gamma log2(e) W_k[h]' q[h]  (rank), w[h] = scale log2(e) rotated q_rot[h]
//   scores  s[h,j] = absmax[j] / 127 * (u[h] . row[j]) + w[h] . key[j],  p = 2^(s - max)
//   sum     o[h] = sum_j p[h,j] absmax[j] / 127 * row[j]
//   join    out[h] = gamma W_v[h] (sum over the parts of 2^(max' - max) o[h]) / (sum of p)
//
// Three launches: query, scores and sums of the workers' parts (latent_step.cuh says how tokens are divided), join.  The kernel of this file
// holds everything in float32; latent_step_tc.cu takes 16-bit activations.
#include "latent_step.cuh"

namespace el {

bool latent_step_tc_takes(const el_latent_step_t& a);
int latent_step_tc_groups(const el_latent_step_t& a);
int launch_latent_step_tc(const el_latent_step_t& a, const int8_t* digits, const float* steps, const void* rotated, const latent::StepParts& parts, int workers,
                          cudaStream_t st);

using namespace latent;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int GROUP = 32;             // heads of a block
constexpr int MOST_RANK = 512, MOST_ROT = 64;

// four 2-bit codes as float: 0 -> -1, 1 -> 0, 2 -> 1, 3 -> 0
__device__ __forceinline__ float weight_of(uint32_t w, int i) { return (float)decode2(w >> (2 * i)); }

// u and w of one head for PER sequences.  Thread (x, y): column words x of the weights (16 columns each), rows y, y + 8 ..
// DIGITS: for the tensor cores, u as two 8-bit digits of 1 / 32512 of its largest magnitude (digits [.., 2, rank padded to 32], steps) and w as T [.., 64].
template <typename T, bool DIGITS, int PER>
__global__ void __launch_bounds__(THREADS) step_query_kernel(const el_latent_step_t a, float* __restrict__ query, int8_t* __restrict__ digits, float* __restrict__ steps, T* __restrict__ rotated) {
    __shared__ float q[PER][256];
    __shared__ float part[WARPS][32][17];
    __shared__ float most[WARPS];
    const int h = blockIdx.x, b0 = blockIdx.y * PER, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int words = a.rank / 16, width = a.rank + a.rot_dim;
    const float by = a.scale * mamba::LOG2E;
    for (int i = threadIdx.x; i < PER * a.key_dim; i += THREADS) {
        const int n = i / a.key_dim, d = i - n * a.key_dim;
        q[n][d] = b0 + n < a.batch ? to_float(static_cast<const T*>(a.q)[(b0 + n) * a.q_stride_b + h * a.q_stride_h + d]) : 0.0f;
    }
    __syncthreads();
    float sum[PER][16] = {};
    if (lane < words) {
        const uint32_t* W = reinterpret_cast<const uint32_t*>(a.W_packed + (long long)h * a.key_dim * (a.rank / 4)) + lane;
#pragma unroll 4
        for (int d = warp; d < a.key_dim; d += WARPS) {
            const uint32_t w = W[(long long)d * words];
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = weight_of(w, i);
#pragma unroll
            for (int n = 0; n < PER; ++n) {
                const float v = q[n][d];
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[n][i] = fmaf(v, f[i], sum[n][i]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        if (b0 + n >= a.batch) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[warp][lane][i] = sum[n][i];
        __syncthreads();
        const long long bh = (long long)(b0 + n) * a.heads + h;
        float* out = query + bh * width;
        float u[MOST_RANK / THREADS], top = 0.0f;
#pragma unroll
        for (int i = 0; i < MOST_RANK / THREADS; ++i) {
            const int c = threadIdx.x + i * THREADS;
            u[i] = 0.0f;
            if (c < a.rank) {
#pragma unroll
                for (int w = 0; w < WARPS; ++w) u[i] += part[w][c / 16][c % 16];
                u[i] *= a.gamma * by;
                if (!DIGITS) out[c] = u[i];
            }
            top = mamba::max_nan(top, fabsf(u[i]));
        }
        if constexpr (DIGITS) {
            const int rp = (a.rank + 31) / 32 * 32;
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) top = mamba::max_nan(top, __shfl_xor_sync(0xffffffffu, top, x));
            if (lane == 0) most[warp] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = mamba::max_nan(top, most[w]);
            const float step = top * (1.0f / 32512.0f), inv = step > 0.0f ? 32512.0f / top : 0.0f;
            if (threadIdx.x == 0) steps[bh] = step;                  // a NaN or infinity makes the scores NaN
#pragma unroll
            for (int i = 0; i < MOST_RANK / THREADS; ++i) {
                const int c = threadIdx.x + i * THREADS;
                if (c >= rp) continue;
                const int v = __float2int_rn(u[i] * inv), hi = (v + 128) >> 8;
                digits[bh * 2 * rp + c] = (int8_t)hi;
                digits[bh * 2 * rp + rp + c] = (int8_t)(v - hi * 256);
            }
            for (int c = a.rot_dim + threadIdx.x; c < 64; c += THREADS) rotated[bh * 64 + c] = mamba::from_float<T>(0.0f);
        }
        auto put = [&](int c, float v) {
            if constexpr (DIGITS) rotated[bh * 64 + c] = mamba::from_float<T>(v);
            else out[a.rank + c] = v;
        };
        if (a.rot_dim == 0) continue;
        const T* x = static_cast<const T*>(a.q_rot) + (b0 + n) * a.q_rot_stride_b + h * a.q_rot_stride_h;
        if (!a.table) {
            for (int c = threadIdx.x; c < a.rot_dim; c += THREADS) put(c, to_float(x[c]) * by);
            continue;
        }
        const int half = a.rot_dim / 2, at = step_tokens(a, b0 + n) - 1;      // the token itself is the cache's last one
        const float* cs = a.table + (long long)(at < 0 ? 0 : at >= a.table_rows ? a.table_rows - 1 : at) * a.rot_dim;
        for (int c = threadIdx.x; c < half; c += THREADS) {
            const int i0 = a.neighbours ? 2 * c : c, i1 = a.neighbours ? 2 * c + 1 : c + half;
            const float u = to_float(x[i0]), v = to_float(x[i1]), co = cs[c], si = cs[c + half];
            put(i0, fmaf(u, co, -__fmul_rn(v, si)) * by);
            put(i1, fmaf(v, co, __fmul_rn(u, si)) * by);
        }
    }
}

// A block takes 32 heads of a worker's tokens, 32 at a time; a warp takes 4 heads: a lane is a token for the scores, a column in every 32 for the sums.
template <typename K>
__global__ void __launch_bounds__(THREADS) step_rows_kernel(const el_latent_step_t a, const float* __restrict__ query, const StepParts parts, int workers) {
    extern __shared__ float sm[];
    constexpr int TILE = 32, CP = MOST_RANK + MOST_ROT + 1;
    const int R = a.rank, width = R + a.rot_dim;
    float* C = sm;                                   // [32 tokens][CP]: row, rotated part
    float* U = C + TILE * CP;                        // [32 heads][width]
    __shared__ float scale_of[TILE];
    __shared__ int seen[TILE];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h0 = blockIdx.y * GROUP, w = blockIdx.x;
    const long long tiles = step_tiles_before(a, a.batch);
    workers = step_active(workers, tiles);
    if (w >= workers) return;
    const long long first = w * tiles / workers, last = (w + 1) * tiles / workers;
    int b;
    long long before;
    step_find(a, first, b, before);
    for (long long t = first; t < last; ++b) {
        const int n = step_tokens(a, b);
        const long long here = (n + STEP_TILE - 1) / STEP_TILE, stop = before + here < last ? before + here : last;
        if (here == 0) continue;
        const int p0 = (int)(t - before) * STEP_TILE, p1 = (int)min((stop - before) * STEP_TILE, (long long)n);
        __syncthreads();
        for (int i = threadIdx.x; i < GROUP * width; i += THREADS) {
            const int h = i / width;
            U[i] = h0 + h < a.heads ? query[((long long)b * a.heads + h0 + h) * width + i - h * width] : 0.0f;
        }
        float top[4], sum[4], o[4][MOST_RANK / 32];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            top[g] = -INFINITY;
            sum[g] = 0.0f;
#pragma unroll
            for (int c = 0; c < MOST_RANK / 32; ++c) o[g][c] = 0.0f;
        }
        for (int p = p0; p < p1; p += TILE) {
            __syncthreads();
            for (int j = warp; j < TILE; j += WARPS) {
                const long long row = p + j < p1 ? step_row(a, b, p + j) : -1;
                if (lane == 0) {
                    seen[j] = row >= 0;
                    scale_of[j] = row >= 0 ? __fdiv_rn(a.absmax[row], 127.0f) : 0.0f;
                }
                for (int c = lane; c < R; c += 32) C[j * CP + c] = row >= 0 ? (float)a.latents[row * R + c] : 0.0f;
                for (int c = lane; c < a.rot_dim; c += 32) C[j * CP + R + c] = row >= 0 ? to_float(static_cast<const K*>(a.cache_keys)[row * a.rot_dim + c]) : 0.0f;
            }
            __syncthreads();
            float s[4] = {}, r[4] = {};
            const float* u = U + 4 * warp * width;
            for (int c = 0; c < R; ++c) {
                const float v = C[lane * CP + c];
#pragma unroll
                for (int g = 0; g < 4; ++g) s[g] = fmaf(v, u[g * width + c], s[g]);
            }
            for (int c = R; c < width; ++c) {
                const float v = C[lane * CP + c];
#pragma unroll
                for (int g = 0; g < 4; ++g) r[g] = fmaf(v, u[g * width + c], r[g]);
            }
            float prob[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                s[g] = seen[lane] ? fmaf(s[g], scale_of[lane], r[g]) : -INFINITY;
                float m = mamba::max_nan(top[g], s[g]);
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) m = mamba::max_nan(m, __shfl_xor_sync(0xffffffffu, m, x));
                const float from = m == -INFINITY ? 0.0f : m, old = exp2_neg(top[g] - from);
                prob[g] = exp2_neg(s[g] - from);
                top[g] = m;
                float e = prob[g];
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) e += __shfl_xor_sync(0xffffffffu, e, x);
                sum[g] = fmaf(sum[g], old, e);
                prob[g] *= scale_of[lane];
#pragma unroll
                for (int c = 0; c < MOST_RANK / 32; ++c) o[g][c] *= old;
            }
            for (int j = 0; j < TILE; ++j) {
                float e[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) e[g] = __shfl_sync(0xffffffffu, prob[g], j);
#pragma unroll
                for (int c = 0; c < MOST_RANK / 32; ++c) {
                    if (32 * c >= R) break;
                    const float v = lane + 32 * c < R ? C[j * CP + lane + 32 * c] : 0.0f;
#pragma unroll
                    for (int g = 0; g < 4; ++g) o[g][c] = fmaf(e[g], v, o[g][c]);
                }
            }
        }
        const long long slot = (long long)w + b;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int h = h0 + 4 * warp + g;
            if (h >= a.heads) break;
            if (lane == 0) {
                parts.stats(slot)[2 * h] = top[g];
                parts.stats(slot)[2 * h + 1] = sum[g];
            }
#pragma unroll
            for (int c = 0; c < MOST_RANK / 32; ++c)
                if (lane + 32 * c < R) parts.vectors(slot)[(long long)h * R + lane + 32 * c] = o[g][c];
        }
        t = stop;
        before += here;
    }
}

// A block joins the parts of one head of one sequence and takes the result through the head's value rows.
template <typename T>
__global__ void __launch_bounds__(THREADS) step_join_kernel(const el_latent_step_t a, const StepParts parts, int workers) {
    __shared__ float o[MOST_RANK];
    __shared__ int range[2];
    const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.rank;
    if (warp == 0) {
        const long long tiles = step_tiles_before(a, a.batch), before = step_tiles_before(a, b);
        const int here = step_tiles(a, b);
        workers = step_active(workers, tiles);
        if (lane == 0) {
            range[0] = here ? step_worker(before, workers, tiles) : 0;
            range[1] = here ? step_worker(before + here - 1, workers, tiles) : -1;
        }
    }
    __syncthreads();
    const int w0 = range[0], w1 = range[1];
    float top = -INFINITY, sum = 0.0f;
    for (int w = w0; w <= w1; ++w) top = mamba::max_nan(top, parts.stats((long long)w + b)[2 * h]);
    for (int w = w0; w <= w1; ++w) {
        const float m = parts.stats((long long)w + b)[2 * h];
        if (m != -INFINITY) sum += exp2_neg(m - top) * parts.stats((long long)w + b)[2 * h + 1];
    }
    const float by = top == -INFINITY ? 0.0f : a.gamma / sum;
    for (int c = threadIdx.x; c < R; c += THREADS) {
        float s = 0.0f;
        for (int w = w0; w <= w1; ++w) {
            const float m = parts.stats((long long)w + b)[2 * h];
            if (m != -INFINITY) s = fmaf(exp2_neg(m - top), parts.vectors((long long)w + b)[(long long)h * R + c], s);
        }
        o[c] = s * by;
    }
    __syncthreads();
    const int words = R / 16;
    const uint32_t* W = reinterpret_cast<const uint32_t*>(a.W_packed + ((long long)a.heads * a.key_dim + (long long)h * a.value_dim) * (R / 4));
    T* out = static_cast<T*>(a.out) + ((long long)b * a.heads + h) * a.value_dim;
    for (int v = warp; v < a.value_dim; v += WARPS) {
        float s = 0.0f;
        if (lane < words) {
            const uint32_t w = W[(long long)v * words + lane];
#pragma unroll
            for (int i = 0; i < 16; ++i) s = fmaf(weight_of(w, i), o[lane * 16 + i], s);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (lane == 0) out[v] = mamba::from_float<T>(s);
    }
}

template <typename F> int of_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}

// Blocks that share the tokens: one for every SM, but no more than there can be tiles.
int step_workers(const el_latent_step_t& a, int groups) {
    int sms = 148;
    device_sm_count(&sms);
    const long long tiles = (((long long)a.pages_per_sequence * a.page_size + STEP_TILE - 1) / STEP_TILE) * a.batch;
    const int most = sms / groups > 0 ? sms / groups : 1;
    return (int)(tiles < most ? tiles : most);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }
size_t digits_bytes(const el_latent_step_t& a) { return align256((size_t)a.batch * a.heads * 2 * ((a.rank + 31) / 32 * 32)); }
size_t steps_bytes(const el_latent_step_t& a) { return align256((size_t)a.batch * a.heads * 4); }
size_t rotated_bytes(const el_latent_step_t& a) { return align256((size_t)a.batch * a.heads * 64 * 2); }
size_t query_bytes(const el_latent_step_t& a) {
    return latent_step_tc_takes(a) ? digits_bytes(a) + steps_bytes(a) + rotated_bytes(a) : align256((size_t)a.batch * a.heads * (a.rank + a.rot_dim) * 4);
}
int groups_of(const el_latent_step_t& a) { return latent_step_tc_takes(a) ? latent_step_tc_groups(a) : 1; }

}  // namespace

size_t latent_step_workspace_bytes(const el_latent_step_t& a) {
    return query_bytes(a) + (size_t)(step_workers(a, groups_of(a)) + a.batch) * a.heads * (2 + (size_t)a.rank) * 4;
}

int launch_latent_step(const el_latent_step_t& a, cudaStream_t st) {
    const int workers = step_workers(a, groups_of(a));
    char* ws = static_cast<char*>(a.workspace);
    const StepParts parts{reinterpret_cast<float*>(ws + query_bytes(a)), a.heads, a.rank};
    constexpr int PER = 4;
    const dim3 grid(a.heads, (a.batch + PER - 1) / PER);
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        int rc = EL_OK;
        if (latent_step_tc_takes(a)) {
            int8_t* digits = reinterpret_cast<int8_t*>(ws);
            float* steps = reinterpret_cast<float*>(ws + digits_bytes(a));
            T* rotated = reinterpret_cast<T*>(ws + digits_bytes(a) + steps_bytes(a));
            step_query_kernel<T, true, PER><<<grid, THREADS, 0, st>>>(a, nullptr, digits, steps, rotated);
            if ((rc = check_launch()) != EL_OK) return rc;
            if (workers > 0) rc = launch_latent_step_tc(a, digits, steps, rotated, parts, workers, st);
        } else {
            float* query = reinterpret_cast<float*>(ws);
            step_query_kernel<T, false, PER><<<grid, THREADS, 0, st>>>(a, query, nullptr, nullptr, nullptr);
            if ((rc = check_launch()) != EL_OK) return rc;
            if (workers > 0) {
                static DeviceOnce once;
                int dev = 0;
                constexpr int most = 4 * (32 * (MOST_RANK + MOST_ROT + 1) + GROUP * (MOST_RANK + MOST_ROT));
                EL_CUDA_TRY(cudaGetDevice(&dev));
                if (!once.is_done(dev)) {
                    EL_CUDA_TRY(cudaFuncSetAttribute(step_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
                    once.mark(dev);
                }
                step_rows_kernel<T><<<dim3(workers, (a.heads + GROUP - 1) / GROUP), THREADS, most, st>>>(a, query, parts, workers);
                rc = check_launch();
            }
        }
        if (rc != EL_OK) return rc;
        step_join_kernel<T><<<(unsigned)(a.batch * a.heads), THREADS, 0, st>>>(a, parts, workers);
        return check_launch();
    });
}

}  // namespace el
