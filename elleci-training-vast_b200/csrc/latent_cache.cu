// Rotation by position, and the cache of latent vectors: pages of tokens, each an int8 row with its largest magnitude (what the up projection's
// quantiser makes of it) and a rotated key part shared by all heads.
//
//   rotary   (x[i], x[i + d/2]) (or neighbours x[2 i], x[2 i + 1]) turned by the angle whose cosine and sine the table holds for the token's position
//   write    norm and quantisation of new tokens as rmsnorm.cu does them, rotation of their key part, both into the tokens' places
//   read     a window of each sequence's tokens out of its pages: the rows and magnitudes as they are (what el_gemm_fwd takes), or the values
//            that they stand for
//
// Bound: memory.  Position p of sequence b lies in page block_table[b][p / page_size]; an entry outside the pool is not followed (nothing is
// written there, zeros are read).
#include "latent_common.cuh"

namespace el {

using namespace latent;
using rowio::Io;

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;

// position of token t of sequence b, within the table
__device__ __forceinline__ int table_row(const int32_t* positions, bool each, int b, int t, int length, int rows) {
    const long long p = positions ? (each ? positions[(long long)b * length + t] : positions[b] + (long long)t) : t;
    return (int)(p < 0 ? 0 : p >= rows ? rows - 1 : p);
}

// VEC pairs a thread: 8 where halves are multiples of 8 and everything lies on 16 bytes, else one.  Bound: memory (4 x 1024 tokens, 32 heads of 64 in bfloat16:
// 34 MB in 9.7 us, 53 % of the HBM's rate with the launch).
template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const el_rotary_t a) {
    const int half = a.dim / 2, per = half / VEC;
    const long long n = (long long)a.batch * a.length * a.heads * per;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < n; i += (long long)gridDim.x * THREADS) {
        const long long row = i / per, token = row / a.heads;
        const int c = (int)(i - row * per) * VEC, h = (int)(row - token * a.heads), b = (int)(token / a.length), t = (int)(token - (long long)b * a.length);
        const float* cs = a.table + (long long)table_row(a.positions, a.position_each != 0, b, t, a.length, a.table_rows) * a.dim + c;
        const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + t * a.x_stride_t + h * a.x_stride_h;
        T* y = static_cast<T*>(a.y) + row * a.dim;
        if constexpr (VEC == 8) {
            float u[8], v[8], co[8], si[8], p[8], q[8];
            rowio::load8_w(cs, co);
            rowio::load8_w(cs + half, si);
            if (a.neighbours) {
                float w[16];
                Io<T>::load8(x + 2 * c, w);
                Io<T>::load8(x + 2 * c + 8, w + 8);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = w[2 * j], v[j] = w[2 * j + 1];
            } else {
                Io<T>::load8(x + c, u);
                Io<T>::load8(x + c + half, v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float s = a.inverse ? -si[j] : si[j];
                p[j] = fmaf(u[j], co[j], -__fmul_rn(v[j], s));
                q[j] = fmaf(v[j], co[j], __fmul_rn(u[j], s));
            }
            if (a.neighbours) {
                float w[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[2 * j] = p[j], w[2 * j + 1] = q[j];
                Io<T>::store8(y + 2 * c, w);
                Io<T>::store8(y + 2 * c + 8, w + 8);
            } else {
                Io<T>::store8(y + c, p);
                Io<T>::store8(y + c + half, q);
            }
        } else {
            const int i0 = a.neighbours ? 2 * c : c, i1 = a.neighbours ? 2 * c + 1 : c + half;
            const float u = to_float(x[i0]), v = to_float(x[i1]), co = cs[0], si = a.inverse ? -cs[half] : cs[half];
            y[i0] = mamba::from_float<T>(fmaf(u, co, -__fmul_rn(v, si)));
            y[i1] = mamba::from_float<T>(fmaf(v, co, __fmul_rn(u, si)));
        }
    }
}

// the pool's row of position p of sequence b, or -1
__device__ __forceinline__ long long pool_row(const int32_t* block_table, int per, int pages, int page_size, int b, long long p) {
    if (p < 0 || p >= (long long)per * page_size) return -1;
    const int page = block_table[(long long)b * per + (int)(p / page_size)];
    return page < 0 || page >= pages ? -1 : (long long)page * page_size + p % page_size;
}

// A warp takes a token; lane l holds columns 8 l .. 8 l + 7 of every 256.  Bound: latency (a page lookup, a row, two reductions, one wave of warps): 4 x 1024 tokens of
// rank 512 with norm and rotation 8 us; asking for the weights and the rotated part before the lookup cost registers and 2 us.
constexpr int ROW_VECS = 2;           // ranks up to 512
template <typename T>
__global__ void __launch_bounds__(THREADS) cache_write_kernel(const el_latent_cache_t a) {
    const long long token = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (token >= (long long)a.batch * a.length) return;
    const int b = (int)(token / a.length), t = (int)(token - (long long)b * a.length);
    if (t >= length_of(a.lengths, b, a.length, a.length)) return;
    const long long p = (a.starts ? a.starts[b] : 0) + (long long)t, row = pool_row(a.block_table, a.pages_per_sequence, a.pages, a.page_size, b, p);
    if (row < 0) return;
    const T* x = static_cast<const T*>(a.x) + b * a.x_stride_b + t * a.x_stride_t;
    const int R = a.rank;
    float v[ROW_VECS][8];
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < ROW_VECS; ++c) {
        const int k = c * 256 + lane * 8;
        if (k < R) {
            if (a.x_aligned) {
                Io<T>::load8(x + k, v[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] = to_float(x[k + i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += (double)__fmul_rn(v[c][i], v[c][i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
        }
    }
    if (a.norm_weight) {              // y = io(io(x * r) * io(w)), the layer's own order of roundings
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn((float)ss, (float)R), a.norm_eps)));
#pragma unroll
        for (int c = 0; c < ROW_VECS; ++c) {
            const int k = c * 256 + lane * 8;
            if (k >= R) continue;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = Io<T>::round(__fmul_rn(Io<T>::round(__fmul_rn(v[c][i], r)), Io<T>::round(a.norm_weight[k + i])));
        }
    }
    float top = 0.0f;                 // of the finite values; the others become zeros
#pragma unroll
    for (int c = 0; c < ROW_VECS; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(finite_or_zero(v[c][i])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(top, a.quant_eps);
    const float s = __fdiv_rn(127.0f, top);
    int8_t* q = a.latents + row * R;
#pragma unroll
    for (int c = 0; c < ROW_VECS; ++c) {
        const int k = c * 256 + lane * 8;
        if (k >= R) continue;
        int n[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = q8_sat(__fmul_rn(finite_or_nan(v[c][i]), s));
        *reinterpret_cast<uint2*>(q + k) = make_uint2(pack4_s8(n[0], n[1], n[2], n[3]), pack4_s8(n[4], n[5], n[6], n[7]));
    }
    if (lane == 0) a.absmax[row] = top;
    if (a.rot_dim == 0) return;
    const T* kx = static_cast<const T*>(a.k_rot) + b * a.k_rot_stride_b + t * a.k_rot_stride_t;
    T* ky = static_cast<T*>(a.cache_keys) + row * a.rot_dim;
    if (!a.table) {
        for (int c = lane; c < a.rot_dim; c += 32) ky[c] = kx[c];
        return;
    }
    const int half = a.rot_dim / 2;
    const float* cs = a.table + (p >= a.table_rows ? a.table_rows - 1 : p) * a.rot_dim;
    for (int c = lane; c < half; c += 32) {
        const int i0 = a.neighbours ? 2 * c : c, i1 = a.neighbours ? 2 * c + 1 : c + half;
        const float u = to_float(kx[i0]), w = to_float(kx[i1]), co = cs[c], si = cs[c + half];
        ky[i0] = mamba::from_float<T>(fmaf(u, co, -__fmul_rn(w, si)));
        ky[i1] = mamba::from_float<T>(fmaf(w, co, __fmul_rn(u, si)));
    }
}

// A warp takes READ_TOKENS tokens; VALUES: the rows come out as values of type T.  All 16-byte pieces of the rows are on their way before the first is written.
// 8 tokens where that leaves two blocks for every SM, else one: 8 x 8192 tokens of rank 512 15.4 and 20.3 us, 4 x 1024 8.9 and 6.2.
template <typename K, typename T, bool VALUES, int READ_TOKENS>
__global__ void __launch_bounds__(THREADS) cache_read_kernel(const el_latent_cache_t a) {
    const long long all = (long long)a.batch * a.length, first = ((long long)blockIdx.x * WARPS + (threadIdx.x >> 5)) * READ_TOKENS;
    if (first >= all) return;
    const int lane = threadIdx.x & 31, R = a.rank;
    // lane l (and l + 8 ..) looks token l up
    long long row = -1;
    float top = 0.0f;
    const long long own = first + (lane & (READ_TOKENS - 1));
    if (own < all) {
        const int b = (int)(own / a.length), t = (int)(own - (long long)b * a.length);
        if (t < length_of(a.lengths, b, a.length, a.length))
            row = pool_row(a.block_table, a.pages_per_sequence, a.pages, a.page_size, b, (a.starts ? a.starts[b] : 0) + (long long)t);
        if (row >= 0) top = a.absmax[row];
    }
    if (!VALUES && lane < READ_TOKENS && own < all) a.out_absmax[own] = top;
    const float scale = VALUES ? __fdiv_rn(top, 127.0f) : 0.0f;
    const int per = R / 16, pieces = READ_TOKENS * per;              // 16-byte pieces of a row, of all
    for (int i0 = 0; i0 < pieces; i0 += 32 * READ_TOKENS) {
        uint4 w[READ_TOKENS];
        int at[READ_TOKENS];
#pragma unroll
        for (int k = 0; k < READ_TOKENS; ++k) {
            const int i = i0 + k * 32 + lane, n = i < pieces ? i / per : 0;
            const long long r = __shfl_sync(0xffffffffu, row, n);
            at[k] = i < pieces && first + n < all ? i : -1;
            w[k] = make_uint4(0u, 0u, 0u, 0u);
            if (at[k] >= 0 && r >= 0) w[k] = *reinterpret_cast<const uint4*>(a.latents + r * R + (i - n * per) * 16);
        }
#pragma unroll
        for (int k = 0; k < READ_TOKENS; ++k) {
            const float s = VALUES ? __shfl_sync(0xffffffffu, scale, at[k] < 0 ? 0 : at[k] / per) : 0.0f;
            if (at[k] < 0) continue;
            if constexpr (!VALUES) {
                *reinterpret_cast<uint4*>(static_cast<int8_t*>(a.out) + first * R + at[k] * 16) = w[k];
            } else {
                const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __fmul_rn((float)(int8_t)(u[i / 4] >> (8 * (i & 3))), s);
                T* out = static_cast<T*>(a.out) + first * R + at[k] * 16;
                Io<T>::store8(out, v);
                Io<T>::store8(out + 8, v + 8);
            }
        }
    }
    if (a.rot_dim == 0) return;
    const K* kx = static_cast<const K*>(a.cache_keys);
    K* ky = static_cast<K*>(a.out_keys) + first * a.rot_dim;
    constexpr int E = 16 / (int)sizeof(K);
    const bool vec = a.rot_dim % E == 0 && reinterpret_cast<uintptr_t>(a.cache_keys) % 16 == 0;
    const int width = vec ? a.rot_dim / E : a.rot_dim, count = READ_TOKENS * width;
    for (int i0 = 0; i0 < count; i0 += 32) {
        const int i = i0 + lane, n = i < count ? i / width : 0, c = i - n * width;
        const long long r = __shfl_sync(0xffffffffu, row, n);
        if (i >= count || first + n >= all) continue;
        if (vec) reinterpret_cast<uint4*>(ky)[i] = r < 0 ? make_uint4(0u, 0u, 0u, 0u) : reinterpret_cast<const uint4*>(kx + r * a.rot_dim)[c];
        else ky[i] = r < 0 ? mamba::from_float<K>(0.0f) : kx[r * a.rot_dim + c];
    }
}

template <typename F> int of_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

int launch_rotary(const el_rotary_t& a, cudaStream_t st) {
    const long long pairs = (long long)a.batch * a.length * a.heads * (a.dim / 2);
    int sms = 148;
    device_sm_count(&sms);
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const long long e = 16 / (int)sizeof(T);
        const bool vec = a.dim % 16 == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.table) && a.x_stride_b % e == 0 && a.x_stride_t % e == 0 && a.x_stride_h % e == 0;
        const long long blocks = (pairs / (vec ? 8 : 1) + THREADS - 1) / THREADS, most = (long long)sms * 64;
        const unsigned grid = (unsigned)(blocks < most ? blocks : most);
        if (vec) rotary_kernel<T, 8><<<grid, THREADS, 0, st>>>(a);
        else rotary_kernel<T, 1><<<grid, THREADS, 0, st>>>(a);
        return check_launch();
    });
}

int launch_latent_cache_write(el_latent_cache_t a, cudaStream_t st) {
    const unsigned grid = (unsigned)(((long long)a.batch * a.length + WARPS - 1) / WARPS);
    return of_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const long long e = 16 / (int)sizeof(T);
        a.x_aligned = aligned16(a.x) && a.x_stride_b % e == 0 && a.x_stride_t % e == 0;
        cache_write_kernel<T><<<grid, THREADS, 0, st>>>(a);
        return check_launch();
    });
}

int launch_latent_cache_read(const el_latent_cache_t& a, cudaStream_t st) {
    const long long tokens = (long long)a.batch * a.length;
    int sms = 148;
    device_sm_count(&sms);
    const bool many = tokens >= 2LL * sms * WARPS * 8;
    const unsigned grid = (unsigned)(many ? (tokens + WARPS * 8 - 1) / (WARPS * 8) : (tokens + WARPS - 1) / WARPS);
    return of_type(a.dtype, [&](auto k) {
        using K = decltype(k);
        if (a.out_dtype < 0) {
            if (many) cache_read_kernel<K, K, false, 8><<<grid, THREADS, 0, st>>>(a);
            else cache_read_kernel<K, K, false, 1><<<grid, THREADS, 0, st>>>(a);
            return check_launch();
        }
        return of_type(a.out_dtype, [&](auto t) {
            using T = decltype(t);
            if (many) cache_read_kernel<K, T, true, 8><<<grid, THREADS, 0, st>>>(a);
            else cache_read_kernel<K, T, true, 1><<<grid, THREADS, 0, st>>>(a);
            return check_launch();
        });
    });
}

}  // namespace el
