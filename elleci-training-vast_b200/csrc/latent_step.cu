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
int launch_latent_step_tc(const el_latent_step_t& a, const uint8_t* images, const float* steps, const latent::StepParts& parts, int workers, cudaStream_t st);

using namespace latent;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int GROUP = 32;             // heads of a block
constexpr int MOST_RANK = 512, MOST_ROT = 64;
constexpr float STEPS = 32512.0f;     // 127 * 256: the largest value of two digits whose high one is at most 127

// Two neighbouring 2-bit codes (the low four bits of x) as two 16-bit floats: 0 -> -1, 1 -> 0, 2 -> 1, 3 -> 0, by a byte permutation of their tables.
template <typename T> __device__ __forceinline__ uint32_t weight_pair(uint32_t first, uint32_t second) {
    constexpr uint32_t high = std::is_same<T, __half>::value ? 0x003C00BCu : 0x003F00BFu, low = std::is_same<T, __half>::value ? 0u : 0x00800080u;
    return prmt(high, low, first * 0x11u + (second * 0x1100u + 0x0404u));
}
// d += a b on the warp: a 16 x 16 (rows lane / 4 and 8 more), b 16 x 8 of T, sums in float32.  The products here are small next to what is read for them.
template <typename T> __device__ __forceinline__ void warp_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// pair c (of rot_dim / 2) of w of one head of one sequence: put(channel, value)
template <typename T, typename F> __device__ __forceinline__ void rotated_query(const el_latent_step_t& a, int b, int h, int c, F put) {
    const float by = a.scale * mamba::LOG2E;
    const T* x = static_cast<const T*>(a.q_rot) + b * a.q_rot_stride_b + h * a.q_rot_stride_h;
    const int half = a.rot_dim / 2, i0 = a.neighbours ? 2 * c : c, i1 = a.neighbours ? 2 * c + 1 : c + half;
    float u = to_float(x[i0]), v = to_float(x[i1]);
    if (a.table) {
        const int at = step_tokens(a, b) - 1;        // the token itself is the cache's last one
        const float* cs = a.table + (long long)(at < 0 ? 0 : at >= a.table_rows ? a.table_rows - 1 : at) * a.rot_dim;
        const float co = cs[c], si = cs[c + half], t = fmaf(u, co, -__fmul_rn(v, si));
        v = fmaf(v, co, __fmul_rn(u, si));
        u = t;
    }
    put(i0, u * by);
    put(i1, v * by);
}

// u and w of one head for 4 sequences, in float32.  Thread (x, y): column words x of the weights (16 columns each), rows y, y + 8 ..
template <typename T>
__global__ void __launch_bounds__(THREADS) step_query_kernel(const el_latent_step_t a, float* __restrict__ query) {
    constexpr int PER = 4;
    __shared__ float q[PER][256];
    __shared__ float part[WARPS][32][17];
    const int h = blockIdx.x, b0 = blockIdx.y * PER, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int words = a.rank / 16, width = a.rank + a.rot_dim;
    for (int i = threadIdx.x; i < PER * a.key_dim; i += THREADS) {
        const int n = i / a.key_dim, d = i - n * a.key_dim;
        q[n][d] = b0 + n < a.batch ? to_float(static_cast<const T*>(a.q)[(b0 + n) * a.q_stride_b + h * a.q_stride_h + d]) : 0.0f;
    }
    __syncthreads();
    float sum[PER][16] = {};
    if (lane < words) {
        const uint32_t* W = reinterpret_cast<const uint32_t*>(a.W_packed + (long long)h * a.key_dim * (a.rank / 4)) + lane;
        for (int d = warp; d < a.key_dim; d += WARPS) {
            const uint32_t w = W[(long long)d * words];
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = (float)decode2(w >> (2 * i));
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
        float* out = query + ((long long)(b0 + n) * a.heads + h) * width;
        for (int c = threadIdx.x; c < a.rank; c += THREADS) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) s += part[w][c / 16][c % 16];
            out[c] = s * (a.gamma * a.scale * mamba::LOG2E);
        }
        auto put = [&](int c, float v) { out[a.rank + c] = v; };
        for (int c = threadIdx.x; c < a.rot_dim / 2; c += THREADS) rotated_query<T>(a, b0 + n, h, c, put);
        // an odd last channel has no partner and is not turned (there is no table then)
        if (a.rot_dim % 2 && threadIdx.x == 0)
            put(a.rot_dim - 1, to_float(static_cast<const T*>(a.q_rot)[(b0 + n) * a.q_rot_stride_b + h * a.q_rot_stride_h + a.rot_dim - 1]) * a.scale * mamba::LOG2E);
    }
}

// u and w for the tensor cores: of one head, 128 columns of u for 16 sequences, into the images of latent_step.cuh.  u = gamma scale log2(e) q W is held in
// two 8-bit digits of 1 / 32512 of gamma scale log2(e) sum |q|, which it cannot exceed whatever the weights are: no block has to know another's columns.
// (For weights of random signs that is 3 to 4 times the largest u, 14 bits of it.)  steps [batch, groups, 32].  A warp takes 16 columns, which are one
// word of every row of the weights (32: 94 us for the whole step of 64 sequences instead of 87).  Operands go from memory to the threads' registers as the products take them (a lane has 8 neighbouring channels of
// every 32, in the query and in the weights, whatever the order of a product's own reduction), 64 channels at a time: shared memory in between, and its
// barriers, made the kernel 13000 cycles long where there are 64 sequences of 32 heads of 128 channels.
constexpr int QUERY_ROWS = 16, QUERY_COLS = 128;
template <typename T>
__global__ void __launch_bounds__(THREADS, 4) step_query_digits_kernel(const el_latent_step_t a, uint8_t* __restrict__ images, float* __restrict__ steps, const bool vectors) {
    const StepImage image(a);
    asm volatile("griddepcontrol.launch_dependents;");
    const int h = blockIdx.x, c0 = blockIdx.y * QUERY_COLS, b0 = blockIdx.z * QUERY_ROWS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int nb = min(QUERY_ROWS, a.batch - b0), D = h < a.heads ? a.key_dim : 0, words = a.rank / 16, rp = (a.rank + 31) / 32 * 32;
    const int group = h / 32, hg = h % 32, r = lane >> 2, own = (lane & 3) * 8, word = c0 / 16 + warp;
    const float by = a.gamma * a.scale * mamba::LOG2E;
    const uint32_t* weights = reinterpret_cast<const uint32_t*>(a.W_packed) + (long long)h * a.key_dim * words + word;
    float sum[2][4] = {}, total[2] = {};             // of columns t * 8 ..; of |q| of rows r, r + 8
#pragma unroll 1
    for (int k0 = 0; k0 < D; k0 += 64) {
        uint32_t q[2][2][4], w[2][8];                // [32 channels][row][pairs of 8], [32 channels][8]
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int d0 = k0 + 32 * x + own;
#pragma unroll
            for (int d = 0; d < 8; ++d) w[x][d] = d0 + d < D && word < words ? weights[(long long)(d0 + d) * words] : 0x55555555u;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int n = r + 8 * m;
                const T* from = static_cast<const T*>(a.q) + (b0 + n) * a.q_stride_b + h * a.q_stride_h + d0;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (vectors) {                       // rows of 8 values on 16 bytes
                    if (n < nb && d0 < D) v = *reinterpret_cast<const uint4*>(from);
                } else {
                    T one[8];
#pragma unroll
                    for (int d = 0; d < 8; ++d) one[d] = n < nb && d0 + d < D ? from[d] : mamba::from_float<T>(0.0f);
                    memcpy(&v, one, 16);
                }
                q[x][m][0] = v.x; q[x][m][1] = v.y; q[x][m][2] = v.z; q[x][m][3] = v.w;
            }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                T one[8];
                memcpy(one, q[x][m], 16);
#pragma unroll
                for (int d = 0; d < 8; ++d) total[m] += fabsf(to_float(one[d]));
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {            // 16 channels: four of each lane's eight
                const uint32_t f[4] = {q[x][0][2 * y], q[x][1][2 * y], q[x][0][2 * y + 1], q[x][1][2 * y + 1]};
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int at = 2 * (t * 8 + r);
                    warp_mma<T>(sum[t], f, weight_pair<T>((w[x][4 * y] >> at) & 3u, (w[x][4 * y + 1] >> at) & 3u),
                                weight_pair<T>((w[x][4 * y + 2] >> at) & 3u, (w[x][4 * y + 3] >> at) & 3u));
                }
            }
        }
    }
    if (a.rot_dim) {                                 // the column blocks share the rows
        const int pairs = 32;                        // of the 64 places of w; those behind rot_dim are zeros
        for (int i = blockIdx.y * THREADS + threadIdx.x; i < nb * pairs; i += gridDim.y * THREADS) {
            const int n = i / pairs, c = i % pairs, half = a.rot_dim / 2;
            uint8_t* out = images + ((long long)(b0 + n) * image.groups + group) * image.bytes();
            auto put = [&](int x, float v) { *reinterpret_cast<T*>(out + image.w(2 * x, hg)) = mamba::from_float<T>(v); };
            if (h < a.heads && c < half) rotated_query<T>(a, b0 + n, h, c, put);
            for (int x = a.rot_dim + c; x < 64; x += pairs) put(x, 0.0f);
            if (h >= a.heads)
                for (int x = c; x < a.rot_dim; x += pairs) put(x, 0.0f);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        const int n = r + 8 * m;
        float s = total[m];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (n >= nb) continue;
        if (c0 == 0 && warp == 0 && (lane & 3) == 0) steps[((long long)(b0 + n) * image.groups + group) * 32 + hg] = by * s * (1.0f / STEPS);      // a NaN or infinity makes the scores NaN
        const float inv = s > 0.0f ? STEPS / s : 0.0f;
        uint8_t* out = images + ((long long)(b0 + n) * image.groups + group) * image.bytes();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int c = c0 + warp * 16 + t * 8 + (lane & 3) * 2;
            if (c >= rp) continue;
            int v[2], hi[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                v[e] = min(max(__float2int_rn(sum[t][2 * m + e] * inv), -(int)STEPS), (int)STEPS);
                hi[e] = (v[e] + 128) >> 8;
            }
            *reinterpret_cast<char2*>(out + image.digit(c, 0, hg)) = make_char2((signed char)hi[0], (signed char)hi[1]);
            *reinterpret_cast<char2*>(out + image.digit(c, 1, hg)) = make_char2((signed char)(v[0] - hi[0] * 256), (signed char)(v[1] - hi[1] * 256));
        }
    }
}

// A block takes 32 heads of a worker's tokens, 32 at a time; a warp takes 4 heads: a lane is a token for the scores, a column in every 32 for the sums.  Bound: the FMA pipes
// (float32, 8 sequences of 8000 tokens, 32 heads: the step takes 474 us, 38 on the tensor cores in bfloat16).
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
    const long long tiles = step_all_tiles(a);
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// a word to the same place of shared memory in block `rank` of the cluster
__device__ __forceinline__ void store_cluster(uint32_t addr, int rank, uint32_t v) {
    asm volatile("{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %0, %1;\n\tst.shared::cluster.u32 [at], %2;\n\t}" ::"r"(addr), "r"(rank), "r"(v) : "memory");
}

// BLOCKS blocks (a cluster of four, or one) join the parts of one head of up to 16 sequences and take the results through the head's value rows: each block
// joins its share of the latent channels, all write theirs into all blocks' shared memory, and each forms its share of the values.  Sequences are spread over
// a block's 16 warps; where there are fewer, several warps share a sequence's parts, and the warps share the reduction of the product.  The product
// runs on the warps' matrix instructions, the float32 vectors split into two bfloat16 terms (16 bits of each), three for float32 outputs.
// Four blocks for up to 16 sequences, where each has many parts and there would be few blocks: the whole step of 1 sequence of 32768 tokens, 32 heads, takes 35.3 us
// with one block and 31.0 with four, of 64 sequences 89 and 107.
constexpr int JOIN_THREADS = 512, JOIN_WARPS = 16, JOIN_ROWS = 16, JOIN_PITCH = MOST_RANK + 8;
template <typename T> constexpr int JOIN_TERMS = sizeof(T) == 4 ? 3 : 2;
template <int BLOCKS> constexpr int JOIN_FLOATS = JOIN_WARPS * (MOST_RANK / BLOCKS > 256 ? MOST_RANK / BLOCKS : 256);          // sums by warp; of 16 x 16 results by warp
template <typename T, int BLOCKS> constexpr int JOIN_BYTES = JOIN_FLOATS<BLOCKS> * 4 + JOIN_TERMS<T> * JOIN_ROWS * JOIN_PITCH * 2;

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(JOIN_THREADS) step_join_kernel(const el_latent_step_t a, const StepParts parts, int workers) {
    constexpr int COLS = MOST_RANK / BLOCKS, WORDS = BLOCKS == 1 ? 16 : 8, AT_ONCE = BLOCKS == 1 ? 4 : 10;
    extern __shared__ float4 join_smem[];
    float* o = reinterpret_cast<float*>(join_smem);                                            // [16 warps][COLS]
    __nv_bfloat16* terms = reinterpret_cast<__nv_bfloat16*>(o + JOIN_FLOATS<BLOCKS>);            // [terms][16 sequences][JOIN_PITCH]
    const int h = blockIdx.x / BLOCKS, quarter = blockIdx.x % BLOCKS, b0 = blockIdx.y * JOIN_ROWS, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = a.rank;
    const int nb = min(JOIN_ROWS, a.batch - b0);
    int spread = 1;                                  // sequences side by side, a power of two; 16 / spread warps share one
    while (spread < nb) spread *= 2;
    const int shares = JOIN_WARPS / spread, share = warp / spread, b = b0 + warp % spread;
    const int c0 = quarter * COLS, cols = min(COLS, R - c0);                                   // this block's channels (none: 0 or less)
    // the value rows of this block, 16 for a warp at a time (its operand of the sequences serves both eights); warps that have the same ones take every
    // `depth`-th word (16 channels) of them
    const int words = R / 16, r = lane >> 2, k2 = (lane & 3) * 2, per = (a.value_dim + 8 * BLOCKS - 1) / (8 * BLOCKS) * 8, v_begin = quarter * per;
    int groups = 1;                                  // of 16 rows, a power of two and 8 at most: depth is 2 or more, with four blocks (64 rows) 4 or more
    while (groups * 16 < per && groups < JOIN_WARPS / 2) groups *= 2;
    const int depth = JOIN_WARPS / groups, first = warp / groups, mine = (warp % groups) * 16;
    uint32_t w[2][WORDS];
    auto load_weights = [&](int v0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int v = v0 + mine + 8 * e + r, row = v_begin + v;
            const uint32_t* W = reinterpret_cast<const uint32_t*>(a.W_packed) + ((long long)a.heads * a.key_dim + (long long)h * a.value_dim + row) * words;
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[e][k] = v < per && row < a.value_dim && first + k * depth < words ? W[first + k * depth] : 0x55555555u;
        }
    };
    load_weights(0);                                 // before anything that the kernels before leave is there
    float acc[COLS / 32] = {};
    int w0 = 0, w1 = -1;
    if (warp % spread < nb) {
        long long tiles = 0, before = 0;
        int here = 0;
#pragma unroll 4
        for (int x = lane; x < a.batch; x += 32) {
            const int n = step_tiles(a, x);
            tiles += n;
            before += x < b ? n : 0;
            here += x == b ? n : 0;
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            tiles += __shfl_xor_sync(0xffffffffu, tiles, x);
            before += __shfl_xor_sync(0xffffffffu, before, x);
            here += __shfl_xor_sync(0xffffffffu, here, x);
        }
        if (here > 0) {
            const int active = step_active(workers, tiles);
            w0 = step_worker(before, active, tiles);
            w1 = step_worker(before + here - 1, active, tiles);
        }
    }
    for (int i = threadIdx.x; i < JOIN_TERMS<T> * (JOIN_ROWS - nb) * (JOIN_PITCH / 2); i += JOIN_THREADS) {      // rows of no sequence
        const int t = i / ((JOIN_ROWS - nb) * (JOIN_PITCH / 2));
        reinterpret_cast<uint32_t*>(terms + (t * JOIN_ROWS + nb) * JOIN_PITCH)[i - t * (JOIN_ROWS - nb) * (JOIN_PITCH / 2)] = 0u;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (w0 <= w1) {
        // A load here takes some 1000 cycles (other SMs have just written what it reads), so all loads that a warp's first parts need are on their way at once.
        float4 y[AT_ONCE][COLS / 128];
        float own;                                   // lane l: the maximum of the l-th of them
        auto fetch = [&](int i0) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int p = w0 + share + (i0 + i) * shares;
                const float4* v = reinterpret_cast<const float4*>(parts.vectors((long long)p + b) + (long long)h * R + c0) + lane;
#pragma unroll
                for (int c = 0; c < COLS / 128; ++c) y[i][c] = p <= w1 && (c * 32 + lane) * 4 < cols ? v[c * 32] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            const int p = w0 + share + (i0 + lane) * shares;
            own = lane < AT_ONCE && p <= w1 ? parts.stats((long long)p + b)[2 * h] : -INFINITY;
        };
        fetch(0);
        float top = -INFINITY, sum = 0.0f;
        for (int p0 = w0; p0 <= w1; p0 += 160) {
            float2 st[5];
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                const int p = p0 + lane + 32 * k;
                st[k] = p <= w1 ? *reinterpret_cast<const float2*>(parts.stats((long long)p + b) + 2 * h) : make_float2(-INFINITY, 0.0f);
            }
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                const float m = mamba::max_nan(top, st[k].x), from = m == -INFINITY ? 0.0f : m;
                sum = fmaf(sum, exp2_neg(top - from), exp2_neg(st[k].x - from) * st[k].y);
                top = m;
            }
        }
        float all = top;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) all = mamba::max_nan(all, __shfl_xor_sync(0xffffffffu, all, x));
        const float from = all == -INFINITY ? 0.0f : all;
        sum *= exp2_neg(top - from);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const float by = all == -INFINITY ? 0.0f : a.gamma / sum;
        for (int i0 = 0; w0 + share + i0 * shares <= w1; i0 += AT_ONCE) {
            if (i0 > 0) fetch(i0);
            const float f = exp2_neg(own - from) * by;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float x = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
                for (int c = 0; c < COLS / 128; ++c) {
                    acc[4 * c] = fmaf(x, y[i][c].x, acc[4 * c]);
                    acc[4 * c + 1] = fmaf(x, y[i][c].y, acc[4 * c + 1]);
                    acc[4 * c + 2] = fmaf(x, y[i][c].z, acc[4 * c + 2]);
                    acc[4 * c + 3] = fmaf(x, y[i][c].w, acc[4 * c + 3]);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < COLS / 128; ++c)
        reinterpret_cast<float4*>(o + warp * COLS)[c * 32 + lane] = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
    auto meet = [&]() {
        if (BLOCKS > 1) {
            cluster_arrive();
            cluster_wait();
        } else {
            __syncthreads();
        }
    };
    meet();                                          // the other blocks have begun, too: their shared memory may be written
#pragma unroll 1
    for (int i = threadIdx.x; i < nb * COLS / 2; i += JOIN_THREADS) {
        const int n = i / (COLS / 2), c = i % (COLS / 2) * 2;
        if (c >= cols) continue;
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int s = 0; s < shares; ++s) {
            const float2 x = *reinterpret_cast<const float2*>(o + (s * spread + n) * COLS + c);
            v.x += x.x;
            v.y += x.y;
        }
#pragma unroll
        for (int t = 0; t < JOIN_TERMS<T>; ++t) {
            const uint32_t x = pack_bf16x2(v.x, v.y);
            __nv_bfloat16* to = terms + (t * JOIN_ROWS + n) * JOIN_PITCH + c0 + c;
            if (BLOCKS > 1) {
#pragma unroll
                for (int q = 0; q < BLOCKS; ++q) store_cluster((uint32_t)__cvta_generic_to_shared(to), q, x);
            } else {
                *reinterpret_cast<uint32_t*>(to) = x;
            }
            v.x -= __uint_as_float(x << 16);
            v.y -= __uint_as_float(x & 0xFFFF0000u);
        }
    }
    meet();
    for (int v0 = 0; v0 < per; v0 += groups * 16) {
        if (v0 > 0) {
            __syncthreads();                         // the results before have been read
            load_weights(v0);
        }
        // four words in a row of code: the kernel is short and its code is not in the instruction cache when it begins
        float d[2][4] = {}, low[2][4] = {};
#pragma unroll 1
        for (int k0 = 0; first + k0 * depth < words; k0 += 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int word = first + (k0 + k) * depth;
                if (word >= words) break;
                uint32_t x[2][2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t y = w[e][k] >> (2 * k2);
                    x[e][0] = weight_pair<__nv_bfloat16>(y & 3u, (y >> 2) & 3u);
                    x[e][1] = weight_pair<__nv_bfloat16>((y >> 16) & 3u, (y >> 18) & 3u);
                }
#pragma unroll
                for (int t = JOIN_TERMS<T> - 1; t >= 0; --t) {
                    const __nv_bfloat16* p = terms + (t * JOIN_ROWS + r) * JOIN_PITCH + word * 16 + k2;
                    const uint32_t y[4] = {*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(p + 8 * JOIN_PITCH), *reinterpret_cast<const uint32_t*>(p + 8),
                                           *reinterpret_cast<const uint32_t*>(p + 8 * JOIN_PITCH + 8)};
#pragma unroll
                    for (int e = 0; e < 2; ++e) warp_mma<__nv_bfloat16>(t == 0 ? d[e] : low[e], y, x[e][0], x[e][1]);
                }
            }
#pragma unroll
            for (int k = 0; k + 4 < WORDS; ++k) {
                w[0][k] = w[0][k + 4];
                w[1][k] = w[1][k + 4];
            }
        }
        // the warps' shares of the reduction: [warp][16 sequences][16 rows]
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float* to = o + warp * 256 + r * 16 + 8 * e + k2;
            *reinterpret_cast<float2*>(to) = make_float2(d[e][0] + low[e][0], d[e][1] + low[e][1]);
            *reinterpret_cast<float2*>(to + 128) = make_float2(d[e][2] + low[e][2], d[e][3] + low[e][3]);
        }
        __syncthreads();
        const int here = min(groups * 16, per - v0);
        for (int i = threadIdx.x; i < nb * here; i += JOIN_THREADS) {
            const int n = i / here, v = i - n * here;
            if (v_begin + v0 + v >= a.value_dim) continue;
            float x = 0.0f;
#pragma unroll 2
            for (int s = 0; s < depth; ++s) x += o[(s * groups + v / 16) * 256 + n * 16 + v % 16];
            static_cast<T*>(a.out)[((long long)(b0 + n) * a.heads + h) * a.value_dim + v_begin + v0 + v] = mamba::from_float<T>(x);
        }
    }
}

// A launch that may begin before the one in front of it has ended; what that one leaves is read behind griddepcontrol.wait.
template <typename K, typename... A> int launch_dependent(K kernel, dim3 grid, int cluster, int threads, int bytes, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    EL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
    return check_launch();
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

// Blocks that share the tokens: one for every SM, but no more than there can be tiles.
int step_workers(const el_latent_step_t& a, int groups) {
    int sms = 148;
    device_sm_count(&sms);
    const long long tiles = (((long long)a.pages_per_sequence * a.page_size + STEP_TILE - 1) / STEP_TILE) * a.batch;
    const int most = sms / groups > 0 ? sms / groups : 1;
    return (int)(tiles < most ? tiles : most);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }
size_t images_bytes(const el_latent_step_t& a) { return align256((size_t)a.batch * StepImage(a).groups * StepImage(a).bytes()); }
size_t query_bytes(const el_latent_step_t& a) {
    return latent_step_tc_takes(a) ? images_bytes(a) + align256((size_t)a.batch * StepImage(a).groups * 32 * 4) : align256((size_t)a.batch * a.heads * (a.rank + a.rot_dim) * 4);
}
int groups_of(const el_latent_step_t& a) { return latent_step_tc_takes(a) ? StepImage(a).groups : 1; }

}  // namespace

size_t latent_step_workspace_bytes(const el_latent_step_t& a) {
    return query_bytes(a) + (size_t)(step_workers(a, groups_of(a)) + a.batch) * a.heads * (2 + (size_t)a.rank) * 4;
}

int launch_latent_step(const el_latent_step_t& a, cudaStream_t st) {
    const int workers = step_workers(a, groups_of(a));
    char* ws = static_cast<char*>(a.workspace);
    float* vectors = reinterpret_cast<float*>(ws + query_bytes(a));
    const StepParts parts{vectors, vectors + (size_t)(workers + a.batch) * a.heads * a.rank, a.heads, a.rank};
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        int rc = EL_OK;
        if (!latent_step_tc_takes(a)) {
            float* query = reinterpret_cast<float*>(ws);
            step_query_kernel<T><<<dim3(a.heads, (a.batch + 3) / 4), THREADS, 0, st>>>(a, query);
            constexpr int bytes = 4 * (32 * (MOST_RANK + MOST_ROT + 1) + GROUP * (MOST_RANK + MOST_ROT));
            static DeviceOnce once;
            if ((rc = check_launch()) == EL_OK) rc = allow_shared(step_rows_kernel<T>, bytes, once);
            if (rc == EL_OK && workers > 0) {
                step_rows_kernel<T><<<dim3(workers, (a.heads + GROUP - 1) / GROUP), THREADS, bytes, st>>>(a, query, parts, workers);
                rc = check_launch();
            }
        } else if constexpr (!std::is_same<T, float>::value) {
            uint8_t* images = reinterpret_cast<uint8_t*>(ws);
            float* steps = reinterpret_cast<float*>(ws + images_bytes(a));
            const StepImage image(a);
            const bool vectors = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride_b % 8 == 0 && a.q_stride_h % 8 == 0 && a.key_dim % 8 == 0;
            const dim3 grid((image.groups - 1) * 32 + image.hp, (a.rank + QUERY_COLS - 1) / QUERY_COLS, (a.batch + QUERY_ROWS - 1) / QUERY_ROWS);
            step_query_digits_kernel<T><<<grid, THREADS, 0, st>>>(a, images, steps, vectors);
            if ((rc = check_launch()) == EL_OK && workers > 0) rc = launch_latent_step_tc(a, images, steps, parts, workers, st);
        }
        if (rc != EL_OK) return rc;
        auto join = [&](auto blocks) {
            constexpr int BLOCKS = decltype(blocks)::value;
            static DeviceOnce once;
            const int rc = allow_shared(step_join_kernel<T, BLOCKS>, JOIN_BYTES<T, BLOCKS>, once);
            if (rc != EL_OK) return rc;
            const dim3 grid(a.heads * BLOCKS, (a.batch + JOIN_ROWS - 1) / JOIN_ROWS);
            return launch_dependent(step_join_kernel<T, BLOCKS>, grid, BLOCKS, JOIN_THREADS, JOIN_BYTES<T, BLOCKS>, st, a, parts, workers);
        };
        return a.batch <= JOIN_ROWS ? join(std::integral_constant<int, 4>()) : join(std::integral_constant<int, 1>());
    });
}

}  // namespace el
