// Selective state space scan: forward, backward and single token.
//
//   delta = softplus(dt + bias),  h[t] = exp(delta A[n]) h[t-1] + delta u B[n],  y = (sum_n C[n] h[t] + D u) z sigmoid(z)
//
// backward, with dyg = dy z sigmoid(z) and g[t] = C[t] dyg[t] + a[t+1] g[t+1] (a = exp(delta A)), the gradient of the state after token t:
//   dA = sum_t delta w,  w = g a h[t-1];   ddelta = sum_n A w + u sum_n g B;   ddt = ddelta sigmoid(dt + bias)
//   du = D dyg + delta sum_n g B;   dB = sum_d g delta u;   dC = sum_d dyg h;   dz = dy yn slope(z) for the ungated yn
// The states before every KEEP-th token are kept by the forward pass; backward forms the states of a tile again from them.
//
// Floor: the exponentials.  16 states are 16 of them per token and channel (backward: twice), softplus and SiLU four more special functions, at
// 16 a clock and SM; the memory traffic of a bfloat16 call (forward 8 bytes per token and channel) takes less than a third of that time.  What binds
// beside them: wavefronts of shared memory, 19 per token and 16 channels forward, 76 backward, each worth a clock of the SM.  4 x 1024 tokens of
// 8192 channels, 16 states, bfloat16: forward 246 us (floor 144), backward 874.
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
using rowio::Quad;

constexpr int TILE = 16;              // tokens that the forward kernel takes at a time
constexpr int KEEP = 8;               // tokens from one kept state to the next, and of a tile of the backward kernel
constexpr int COUPLES = 4;            // forward: pairs of warps in a block, one on each of the SM's schedulers
constexpr int BACK_WARPS = 8;         // backward: warps of a block

// 2^x of ex2 lies 2e-8 of its value too low on average where x is -1 .. 0 (measured; each value within 1.5e-7).  In a state that decays
// by d per token such an error piles up to 2e-8 / d, a hundred times the scatter's, so the argument is shifted by 2.1e-8 / ln 2.  2^DECAY_SHIFT is 1:
// a token with delta = 0 leaves the state as it is.
constexpr float DECAY_SHIFT = 3.0e-8f;

__device__ __forceinline__ int live_tokens(const el_scan_t& a, int b) { return a.lengths ? min(max(a.lengths[b], 0), a.length) : a.length; }

// The lanes of a warp over the states and channels of its tile.  4 states x 2 channels a lane: B and C are read once for two channels, and 16
// channels a warp are still 512 warps for a layer of 8192.  Forward, 4096 tokens of 8192 channels / 4 x 1024 tokens, 16 states, bfloat16, when the
// shapes were compared: this 349 / 251 us (319 / 246 now); 4 channels a lane 567 / 289; 2 states a lane 464 / 435.
template <int NS_>
struct Shape {
    static constexpr int NS = NS_, SPL = 4, CPL = 2;
    static constexpr int SG = NS / SPL;               // lanes of a channel
    static constexpr int CG = 32 / SG;                // channel pairs side by side
    static constexpr int CW = CG * CPL;               // channels of a warp
    static constexpr int QUADS = CW / 4;
    static constexpr int PAIRS = (QUADS * TILE + 31) / 32;                            // quads of (token, 4 channels) per lane
    static constexpr int BCS = NS / 4 * TILE / 32;                                    // quads of B (and of C) per lane
    static constexpr int GROUP = 2;                   // tokens whose exponentials are in flight together; 4 cost registers and gain nothing
    static constexpr int PER_SM = NS > 32 ? 8 : 16;   // warps of an SM that the registers have to suffice for: what fits in shared memory
    static constexpr int BACK_PER_SM = NS > 16 ? 8 : 16;                              // the same of the backward kernel
    static_assert(CW % 4 == 0 && 32 % QUADS == 0 && BCS >= 1, "");
};

// Where a warp works: its channels d0 .. d0 + n - 1 of group g in sequence b.
struct WarpPlace { int b, g, d0, n; };

// Four states of a channel that has N, from number n0 on; `whole`: all channels' states lie on 16-byte boundaries and N is a multiple of 4.
__device__ __forceinline__ bool whole_states(const float* p, int N) { return N % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }
__device__ __forceinline__ void load_states(const float* p, int n0, int N, bool whole, float v[4]) {
    if (whole) {
        const float4 x = n0 < N ? *reinterpret_cast<const float4*>(p + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n0 + j < N ? p[n0 + j] : 0.0f;
}
__device__ __forceinline__ void store_states(float* p, int n0, int N, bool whole, const float v[4]) {
    if (whole) {
        if (n0 < N) *reinterpret_cast<float4*>(p + n0) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n0 + j < N) p[n0 + j] = v[j];
}
// The same of two adjacent channels, as far as they exist, each pair of values one operand.
__device__ __forceinline__ void load_states2(const float* p, int channels, int n0, int N, bool whole, f32x2 v[4]) {
    float x[2][4] = {};
    if (channels > 0) load_states(p, n0, N, whole, x[0]);
    if (channels > 1) load_states(p + N, n0, N, whole, x[1]);
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = pair(x[0][n], x[1][n]);
}
__device__ __forceinline__ void store_states2(float* p, int channels, int n0, int N, bool whole, const f32x2 v[4]) {
    const float lo[4] = {lo_of(v[0]), lo_of(v[1]), lo_of(v[2]), lo_of(v[3])}, hi[4] = {hi_of(v[0]), hi_of(v[1]), hi_of(v[2]), hi_of(v[3])};
    if (channels > 0) store_states(p, n0, N, whole, lo);
    if (channels > 1) store_states(p + N, n0, N, whole, hi);
}
// The four values of lane group sg as operands for two channels, from token t of a tile's b or c.
template <int TOKENS, int QN> __device__ __forceinline__ void load_twice(const float4 (&m)[TOKENS][QN], int t, int sg, f32x2 v[4]) {
    const float4 x = m[t][sg];
    v[0] = both(x.x); v[1] = both(x.y); v[2] = both(x.z); v[3] = both(x.w);
}
__device__ __forceinline__ f32x2 decay_of(f32x2 A, f32x2 delta) {         // A is already times log2(e)
    const f32x2 x = fma2(A, delta, both(DECAY_SHIFT));
    return pair(ex2(lo_of(x)), ex2(hi_of(x)));
}// Decay rates times log2(e).  Infinite ones (a state that forgets at once; A log2(e) may overflow too) become the largest finite value, which decays as
// much for any step size above 1e-36: 0 times infinity would be NaN for the tokens behind a tile's last one, whose delta is 0 and which leave the
// state as it is.
__device__ __forceinline__ float rate_of(float A) {
    const float x = __fmul_rn(A, LOG2E);
    return isinf(x) ? copysignf(3.402823466e38f, x) : x;
}
__device__ __forceinline__ f32x2 rates_of(f32x2 A) { return pair(rate_of(lo_of(A)), rate_of(hi_of(A))); }

// The state behind a chunk: h before it, decayed over the whole chunk, and what the chunk adds.  A token's decay may be far from 0 and infinity while
// the product over a chunk is not: 0 times infinity would turn a state (or gradient) of zero into a NaN that token by token never arises.  So large
// powers are applied in three steps, each of them finite; beyond 2^300 every state other than zero leaves float32 anyway.
__device__ __forceinline__ f32x2 after_chunk(f32x2 A, f32x2 delta, f32x2 h, f32x2 own) {
    const f32x2 x = fma2(A, delta, both(DECAY_SHIFT));
    float f[2] = {lo_of(x), hi_of(x)}, g[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const bool far = fabsf(f[k]) > 120.0f;                // not a NaN, which stays one
        f[k] = ex2(far ? fminf(fmaxf(f[k], -300.0f), 300.0f) * (1.0f / 3.0f) : f[k]);
        g[k] = far ? f[k] : 1.0f;
    }
    const f32x2 rest = pair(g[0], g[1]);
    return fma2(pair(f[0], f[1]), mul2(rest, mul2(rest, h)), own);
}

// A sequence in chunks: `states` [batch][chunks][channels][states] and `deltas` [batch][chunks][channels] take what each adds on its own.
struct ScanSplit { int chunks, tokens; float* states; float* deltas; };

// ---- forward ------------------------------------------------------------------------------------------------------------
// Warps work in pairs.  A pair owns CW channels and walks over the tokens in tiles.  One warp forms delta and delta u of a tile's (token, channel)
// pairs, four channels of a token at a time as they lie in memory, and puts them into shared memory beside B and C; the other holds the
// states in registers and walks over the tile's tokens; the first one adds its sums over the states' lanes, gates and writes y, while the next
// tile is already in the other's hands.  Both kinds of work are bound by special functions and latencies; on one scheduler each, one's fill the
// other's gaps: 4096 tokens of 8192 channels 437 -> 349 us, 4 x 1024 tokens 270 -> 251 us against warps that do both in turn.

template <typename S>
__device__ __forceinline__ bool warp_place(const el_scan_t& a, WarpPlace& p) {
    const int per_group = a.channels / a.groups, parts = (per_group + S::CW - 1) / S::CW;
    const int w = blockIdx.x * COUPLES + (threadIdx.x >> 5) % COUPLES;
    if (w >= a.batch * a.groups * parts) return false;
    const int part = w % parts, bg = w / parts;
    p.g = bg % a.groups;
    p.b = bg / a.groups;
    p.d0 = p.g * per_group + part * S::CW;
    p.n = min(S::CW, per_group - part * S::CW);
    return true;
}

// What a pair of warps keeps of a tile in shared memory.
template <typename S>
struct Tile {
    // Of channels 2 i, 2 i + 1: delta, delta, delta u, delta u.  Even i lie before odd ones, 64 bytes apart modulo the banks: neither a
    // quad's two stores nor the loads meet a bank twice.
    float4 steps[2][TILE * S::CW / 4 + 4];
    // Each value once: in shared memory twice, as operands for two channels, they save moves but cost wavefronts (256 us forward, 893 backward; so 245 and 871).
    float4 b[TILE][S::NS / 4], c[TILE][S::NS / 4];
    // C h of a lane's states; the lane that writes y adds them.  The rows are 16 floats longer than they need: its vector reads then meet no
    // bank twice.
    float y[TILE][S::SG * S::CW + 16];
};

// Barrier `id` of the two warps of a pair: one arrives and goes on, the other waits for it.
__device__ __forceinline__ void couple_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void couple_wait(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// Tiles go through two buffers.  Barriers of a pair: 2 (tile % 2) says that a tile's inputs are there, 2 (tile % 2) + 1 that its sums are
// and its inputs have been read.  The warp that prepares waits for a tile's sums after it has prepared the next tile.
template <typename T, typename S, bool LOCAL>
struct ScanInputs {
    static constexpr int PAIRS = S::PAIRS, BCS = S::BCS, ROWS = 32 / S::QUADS;
    static constexpr bool FULL = S::QUADS * TILE >= 32;        // every lane has pairs

    static __device__ __forceinline__ void run(const el_scan_t& a, const WarpPlace& p, Tile<S>* tiles, int barrier, int begin, int end, int stop,
                                               bool aligned, bool aligned_bc) {
        const int lane = threadIdx.x & 31, N = a.states;
        const int quad = lane % S::QUADS * 4, row = lane / S::QUADS;          // tokens row, row + 32 / QUADS, ..
        const int valid = p.n - quad;
        float bias[4], D[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bias[j] = a.dt_bias && j < valid ? a.dt_bias[p.d0 + quad + j] : 0.0f;
            D[j] = a.D && j < valid ? a.D[p.d0 + quad + j] : 0.0f;
        }
        const T* up = static_cast<const T*>(a.u) + p.b * a.u_stride_b + p.d0 + quad;
        const T* dtp = static_cast<const T*>(a.dt) + p.b * a.dt_stride_b + p.d0 + quad;
        const T* zp = a.z ? static_cast<const T*>(a.z) + p.b * a.z_stride_b + p.d0 + quad : nullptr;
        const T* Bp = static_cast<const T*>(a.B) + p.b * a.B_stride_b + p.g * a.B_stride_g;
        const T* Cp = static_cast<const T*>(a.C) + p.b * a.C_stride_b + p.g * a.C_stride_g;
        T* yp = static_cast<T*>(a.y) + (long long)p.b * a.length * a.channels + p.d0 + quad;

        Quad<T> u[PAIRS], z[PAIRS], u_next[PAIRS], dt_next[PAIRS], z_next[PAIRS], b_next[BCS], c_next[BCS];
        auto fetch = [&](int t0) {                            // a tile's inputs; zeros behind the sequence's end
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int r = row + i * ROWS, t = t0 + r, v = (FULL || r < TILE) && t < stop ? valid : 0;
                u_next[i] = fetch_quad<T>(up + t * a.u_stride_t, v, aligned);
                dt_next[i] = fetch_quad<T>(dtp + t * a.dt_stride_t, v, aligned);
                if (!LOCAL && zp) z_next[i] = fetch_quad<T>(zp + t * a.z_stride_t, v, aligned);
            }
#pragma unroll
            for (int i = 0; i < BCS; ++i) {
                const int q = lane + 32 * i, t = t0 + q / (S::NS / 4), n = q % (S::NS / 4) * 4, v = t < stop ? N - n : 0;
                b_next[i] = fetch_quad<T>(Bp + t * a.B_stride_t + n, v, aligned_bc);
                if (!LOCAL) c_next[i] = fetch_quad<T>(Cp + t * a.C_stride_t + n, v, aligned_bc);
            }
        };
        auto prepare = [&](int t0, Tile<S>& tile) {           // the fetched tile goes to shared memory, delta formed
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int r = row + i * ROWS;
                const float4 uv = widen<T>(u_next[i]), dv = widen<T>(dt_next[i]);
                const float uu[4] = {uv.x, uv.y, uv.z, uv.w}, dd[4] = {dv.x, dv.y, dv.z, dv.w};
                float delta[4];
                const uint32_t live = t0 + r < stop ? 0xffffffffu : 0u;   // as a mask: a branch here would keep the pairs apart
#pragma unroll
                for (int j = 0; j < 4; ++j) delta[j] = dd[j] + bias[j];
                if (a.softplus) {
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const f32x2 sp = softplus2(delta[j], delta[j + 1], exp_minus_abs(delta[j]), exp_minus_abs(delta[j + 1]));
                        delta[j] = lo_of(sp);
                        delta[j + 1] = hi_of(sp);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) delta[j] = __uint_as_float(__float_as_uint(delta[j]) & live);
                if (FULL || r < TILE) {
                    const int at = r * S::QUADS + quad / 4;
                    tile.steps[0][at] = make_float4(delta[0], delta[1], __fmul_rn(delta[0], uu[0]), __fmul_rn(delta[1], uu[1]));
                    tile.steps[1][at] = make_float4(delta[2], delta[3], __fmul_rn(delta[2], uu[2]), __fmul_rn(delta[3], uu[3]));
                }
            }
#pragma unroll
            for (int i = 0; i < BCS; ++i) {
                const int q = lane + 32 * i, r = q / (S::NS / 4), n = q % (S::NS / 4);
                const float4 bv = widen<T>(b_next[i]);
                tile.b[r][n] = bv;
                if (!LOCAL) {
                    const float4 cv = widen<T>(c_next[i]);
                    tile.c[r][n] = cv;
                }
            }
        };
        auto finish = [&](int t0, const Tile<S>& tile) {      // y of the tile whose u and z are held
            float4 out[PAIRS];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int r = row + i * ROWS;
                const float4 uv = widen<T>(u[i]);
                f32x2 y0 = pair(__fmul_rn(D[0], uv.x), __fmul_rn(D[1], uv.y)), y1 = pair(__fmul_rn(D[2], uv.z), __fmul_rn(D[3], uv.w));
#pragma unroll
                for (int k = 0; k < S::SG; ++k) {
                    const float4 v = *reinterpret_cast<const float4*>(&tile.y[r & (TILE - 1)][k * S::CW + quad]);
                    y0 = add2(y0, pair(v.x, v.y));
                    y1 = add2(y1, pair(v.z, v.w));
                }
                out[i] = make_float4(lo_of(y0), hi_of(y0), lo_of(y1), hi_of(y1));
            }
            if (zp) {
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    const float4 zv = widen<T>(z[i]);
                    out[i].x = __fmul_rn(out[i].x, __fmul_rn(zv.x, sigmoid(zv.x)));
                    out[i].y = __fmul_rn(out[i].y, __fmul_rn(zv.y, sigmoid(zv.y)));
                    out[i].z = __fmul_rn(out[i].z, __fmul_rn(zv.z, sigmoid(zv.z)));
                    out[i].w = __fmul_rn(out[i].w, __fmul_rn(zv.w, sigmoid(zv.w)));
                }
            }
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int r = row + i * ROWS, t = t0 + r;
                if (t >= stop) out[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if ((FULL || r < TILE) && t < end) store_quad<T>(yp + (long long)t * a.channels, valid, aligned, out[i]);
            }
        };
        if (begin < stop) fetch(begin);
        int k = 0;                                            // the tile's number
        for (int t0 = begin; t0 < stop; t0 += TILE, ++k) {
            prepare(t0, tiles[k & 1]);
            couple_arrive(barrier + 2 * (k & 1));
            Quad<T> u_now[PAIRS], z_now[PAIRS];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                u_now[i] = u_next[i];
                if (!LOCAL && zp) z_now[i] = z_next[i];
            }
            if (t0 + TILE < stop) fetch(t0 + TILE);
            if (k > 0) {
                couple_wait(barrier + 2 * ((k - 1) & 1) + 1);
                if (!LOCAL) finish(t0 - TILE, tiles[(k - 1) & 1]);
            }
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                u[i] = u_now[i];
                if (!LOCAL && zp) z[i] = z_now[i];
            }
        }
        if (k > 0) {
            couple_wait(barrier + 2 * ((k - 1) & 1) + 1);
            if (!LOCAL) finish(begin + (k - 1) * TILE, tiles[(k - 1) & 1]);
        }
        if (!LOCAL) {                                         // padding of whole tiles
            for (int t = begin + k * TILE + row; t < end; t += ROWS)
                store_quad<T>(yp + (long long)t * a.channels, valid, aligned, make_float4(0.f, 0.f, 0.f, 0.f));
        }
    }
};

// LOCAL: the state at the chunk's end from zeros at its start, and the sum of delta, for a sequence that is cut into chunks.
template <typename T, typename S, bool LOCAL>
__global__ void __launch_bounds__(64 * COUPLES, S::PER_SM / (2 * COUPLES))
selective_scan_kernel(const el_scan_t a, const ScanSplit split, bool aligned, bool aligned_bc) {
    constexpr int GROUP = S::GROUP, GROUPS = TILE / GROUP;
    extern __shared__ float4 shared_[];
    WarpPlace p;
    if (!warp_place<S>(a, p)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunk = blockIdx.y, barrier = warp % COUPLES * 4;
    Tile<S>* tiles = reinterpret_cast<Tile<S>*>(shared_) + 2 * (warp % COUPLES);
    const int N = a.states, n_live = live_tokens(a, p.b);
    const int begin = chunk * split.tokens, end = min(begin + split.tokens, a.length), stop = min(end, n_live);
    if (warp >= COUPLES) {
        ScanInputs<T, S, LOCAL>::run(a, p, tiles, barrier, begin, end, stop, aligned, aligned_bc);
        return;
    }
    const int sg = lane / S::CG, cg = lane % S::CG;           // lanes of the same states side by side read B and C at once
    const int d0 = p.d0 + 2 * cg, channels = p.n - 2 * cg;    // the lane's: d0, d0 + 1, as far as they exist
    f32x2 A[4], h[4];                                         // the two channels' values
    float dsum[2] = {};
    load_states2(a.A + (long long)d0 * N, channels, sg * 4, N, whole_states(a.A, N), A);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        A[n] = rates_of(A[n]);
        h[n] = both(0.0f);
    }
    if (!LOCAL) {
        if (a.initial_state) load_states2(a.initial_state + ((long long)p.b * a.channels + d0) * N, channels, sg * 4, N, whole_states(a.initial_state, N), h);
        for (int j = 0; j < chunk; ++j) {                     // the chunks before this one, each a state of its own and a decay
            const long long at = ((long long)p.b * split.chunks + j) * a.channels + d0;
            f32x2 own[4];
            load_states2(split.states + at * N, channels, sg * 4, N, whole_states(split.states, N), own);
            const f32x2 delta = pair(channels > 0 ? split.deltas[at] : 0.0f, channels > 1 ? split.deltas[at + 1] : 0.0f);
#pragma unroll
            for (int n = 0; n < 4; ++n) h[n] = after_chunk(A[n], delta, h[n], own[n]);
        }
    }
    const int kept = (a.length + KEEP - 1) / KEEP;
    const bool whole_kept = whole_states(a.checkpoints, N);
    int k = 0;
    for (int t0 = begin; t0 < stop; t0 += TILE, ++k) {
        Tile<S>& tile = tiles[k & 1];
        float* keep = !LOCAL && a.checkpoints ? a.checkpoints + (((long long)p.b * kept + t0 / KEEP) * a.channels + d0) * N : nullptr;
        if (keep) store_states2(keep, channels, sg * 4, N, whole_kept, h);
        couple_wait(barrier + 2 * (k & 1));
        // The tile's tokens in groups: while one group's states are formed, the exponentials of the next are on their way.  Tokens behind
        // the sequence's end have delta = B = C = 0 and leave the states as they are.
        f32x2 decay[2][GROUP][4], add[2][GROUP][4];
        auto prepare = [&](int g, int at) {
#pragma unroll
            for (int k = 0; k < GROUP; ++k) {
                const int t = g * GROUP + k;
                f32x2 B[4];
                load_twice(tile.b, t, sg, B);
                const float4 s = tile.steps[cg & 1][t * S::QUADS + (cg >> 1)];
                if (LOCAL) {
                    dsum[0] += s.x;
                    dsum[1] += s.y;
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    decay[at][k][n] = decay_of(A[n], pair(s.x, s.y));
                    add[at][k][n] = mul2(pair(s.z, s.w), B[n]);
                }
            }
        };
        prepare(0, 0);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (g + 1 < GROUPS) prepare(g + 1, (g + 1) & 1);
            if (g * GROUP == KEEP && keep && t0 + KEEP < stop) store_states2(keep + (long long)a.channels * N, channels, sg * 4, N, whole_kept, h);
#pragma unroll
            for (int k = 0; k < GROUP; ++k) {
                const int t = g * GROUP + k;
                f32x2 C[4];
                if (!LOCAL) load_twice(tile.c, t, sg, C);
#pragma unroll
                for (int n = 0; n < 4; ++n) h[n] = fma2(decay[g & 1][k][n], h[n], add[g & 1][k][n]);
                if (!LOCAL) {
                    f32x2 y = mul2(h[0], C[0]);
#pragma unroll
                    for (int n = 1; n < 4; ++n) y = fma2(h[n], C[n], y);
                    *reinterpret_cast<float2*>(&tile.y[t][sg * S::CW + 2 * cg]) = make_float2(lo_of(y), hi_of(y));
                }
            }
        }
        couple_arrive(barrier + 2 * (k & 1) + 1);
    }
    if (LOCAL) {
        const long long at = ((long long)p.b * split.chunks + chunk) * a.channels + d0;
        store_states2(split.states + at * N, channels, sg * 4, N, whole_states(split.states, N), h);
        if (sg == 0 && channels > 0) split.deltas[at] = dsum[0];
        if (sg == 0 && channels > 1) split.deltas[at + 1] = dsum[1];
    } else if (a.final_state && chunk == split.chunks - 1) {
        store_states2(a.final_state + ((long long)p.b * a.channels + d0) * N, channels, sg * 4, N, whole_states(a.final_state, N), h);
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// A warp owns CW channels, its lanes states and channels as in forward, and walks over tiles of KEEP tokens from the last to the first.  Per tile: the
// lanes form delta, delta u and dyg of the (token, channel) pairs and put them beside B and C; then the states of the tile's tokens are
// formed again from the kept one and go to shared memory; then the tokens are taken in reverse.  A token's sums over the states' lanes (for y, sum g B
// and sum A w) replace its state in shared memory; dB and dC are summed over the warp's channels by shuffles that hand half of the values
// on in each step, and over the block's warps in shared memory.
// Two kept states per 16 tokens instead of one: the states of 8 tokens fill 8 KB, so that 16 warps share an SM.

// What a warp keeps of a tile in shared memory.
template <typename S>
struct BackTile {
    float4 steps[2][KEEP * S::CW / 4 + 4];            // as in Tile
    float4 b[KEEP][S::NS / 4], c[KEEP][S::NS / 4];
    float dyg[KEEP][S::CW];
    float4 h[KEEP][2][32];                            // state before the token: a lane's [state 0, 1 or 2, 3][channel]; then the sums [3][SG][CW]
    float bc[2][KEEP][2][S::NS];                      // dB and dC of the warp's channels, of two tiles
    float bias[S::CW], D[S::CW];
};

// Sums V values over LANES lanes, STRIDE apart, so that lane s of them keeps one: in each step a lane hands half of its values to the lane
// that keeps them, bit k of s deciding which half.  For V < LANES lanes s, s + V, .. share the sum of a value.
template <int V, int LANES, int STRIDE>
__device__ __forceinline__ float spread_sum(float (&v)[V], int s) {
    int left = V;
#pragma unroll
    for (int k = 1; k < LANES; k <<= 1) {
        if (left > 1) {
            left >>= 1;
            const bool up = s & k;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if (i < left) {
                    const float give = up ? v[i] : v[i + left], keep = up ? v[i + left] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, k * STRIDE);
                }
            }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], k * STRIDE);
        }
    }
    return v[0];
}

// dB and dC of a token, the lane's two channels in `v` [4 of dB, 4 of dC], summed over the warp's channels into out [2][states].
template <typename S> __device__ __forceinline__ void bc_sums(float (&v)[8], float (*out)[S::NS], int sg, int cg) {
    if constexpr (S::CG >= 8) {
        const float sum = spread_sum<8, S::CG, 1>(v, cg);
        const int at = (cg & 1) << 2 | (cg & 2) | (cg >> 2 & 1);             // the first step's half is the top bit
        if (cg < 8) out[at >> 2][sg * 4 + (at & 3)] = sum;
    } else if constexpr (S::CG == 4) {                        // 8 values on 4 lanes: two each
        float w[2][4] = {{v[0], v[1], v[2], v[3]}, {v[4], v[5], v[6], v[7]}};
        const int at = (cg & 1) << 1 | (cg >> 1 & 1);
#pragma unroll
        for (int m = 0; m < 2; ++m) out[m][sg * 4 + at] = spread_sum<4, 4, 1>(w[m], cg);
    } else {
        static_assert(S::CG == 2, "");
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float w[2] = {v[i], v[i + 1]};
            out[i >> 2][sg * 4 + (i & 2) + (cg & 1)] = spread_sum<2, 2, 1>(w, cg);
        }
    }
}

// LOCAL: the gradient of the state at the chunk's start from zeros at its end, and the sum of delta.
// partial_bc [blocks of a group][2][batch][length][groups][states], or NULL where neither dB nor dC is wanted; partial_a [batch][chunks][channels][states + 2]: dA, dD, dbias.
template <typename T, typename S, bool LOCAL>
__global__ void __launch_bounds__(32 * BACK_WARPS, S::BACK_PER_SM / BACK_WARPS)
selective_scan_backward_kernel(const el_scan_t a, const ScanSplit split, bool aligned, bool aligned_bc, float* __restrict__ partial_bc,
                               float* __restrict__ partial_a) {
    constexpr int BCQ = S::NS / 4 * KEEP, BCS = (BCQ + 31) / 32;              // quads of B (and of C) of a tile, and per lane
    constexpr int ROWS = 32 / S::QUADS, PAIRS = (KEEP + ROWS - 1) / ROWS;
    constexpr bool FULL = ROWS <= KEEP;                       // every lane has pairs
    constexpr int FLUSH = 16;                                 // tiles after which the sums over tokens go to their outer accumulators
    extern __shared__ float4 shared_[];
    BackTile<S>* const tiles = reinterpret_cast<BackTile<S>*>(shared_);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, chunk = blockIdx.y;
    BackTile<S>& tile = tiles[warp];
    // a block's warps are of one sequence and group; a warp behind the group's last channel works on zeros
    const int per_group = a.channels / a.groups, blocks = (per_group + S::CW * BACK_WARPS - 1) / (S::CW * BACK_WARPS);
    WarpPlace p;
    const int block = blockIdx.x % blocks, in_group = (block * BACK_WARPS + warp) * S::CW;
    p.g = blockIdx.x / blocks % a.groups;
    p.b = blockIdx.x / blocks / a.groups;
    p.d0 = p.g * per_group + in_group;
    p.n = max(min(S::CW, per_group - in_group), 0);
    const int N = a.states, n_live = live_tokens(a, p.b);
    const int begin = chunk * split.tokens, end = min(begin + split.tokens, a.length), stop = min(end, n_live);
    const int sg = lane / S::CG, cg = lane % S::CG;
    const int d0 = p.d0 + 2 * cg, channels = p.n - 2 * cg;
    f32x2 A[4], adj[4], h[4], dA[4];                          // adj: gradient of the state before the token in hand
    float dsum[2] = {};
    load_states2(a.A + (long long)d0 * N, channels, sg * 4, N, whole_states(a.A, N), A);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        A[n] = rates_of(A[n]);
        adj[n] = dA[n] = both(0.0f);
    }
    if (!LOCAL) {
        if (a.d_final_state) load_states2(a.d_final_state + ((long long)p.b * a.channels + d0) * N, channels, sg * 4, N, whole_states(a.d_final_state, N), adj);
        for (int j = split.chunks - 1; j > chunk; --j) {
            const long long at = ((long long)p.b * split.chunks + j) * a.channels + d0;
            f32x2 own[4];
            load_states2(split.states + at * N, channels, sg * 4, N, whole_states(split.states, N), own);
            const f32x2 delta = pair(channels > 0 ? split.deltas[at] : 0.0f, channels > 1 ? split.deltas[at + 1] : 0.0f);
#pragma unroll
            for (int n = 0; n < 4; ++n) adj[n] = after_chunk(A[n], delta, adj[n], own[n]);
        }
    }
    const int quad = lane % S::QUADS * 4, row = lane / S::QUADS, valid = p.n - quad;
    f32x2 dD[2] = {both(0.0f), both(0.0f)}, dbias[2] = {both(0.0f), both(0.0f)};
    if (row == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            tile.bias[quad + j] = a.dt_bias && j < valid ? a.dt_bias[p.d0 + quad + j] : 0.0f;
            tile.D[quad + j] = a.D && j < valid ? a.D[p.d0 + quad + j] : 0.0f;
        }
    }
    __syncwarp();
    const T* up = static_cast<const T*>(a.u) + p.b * a.u_stride_b + p.d0 + quad;
    const T* dtp = static_cast<const T*>(a.dt) + p.b * a.dt_stride_b + p.d0 + quad;
    const T* zp = a.z ? static_cast<const T*>(a.z) + p.b * a.z_stride_b + p.d0 + quad : nullptr;
    const T* dyp = a.dy ? static_cast<const T*>(a.dy) + p.b * a.dy_stride_b + p.d0 + quad : nullptr;
    const T* Bp = static_cast<const T*>(a.B) + p.b * a.B_stride_b + p.g * a.B_stride_g;
    const T* Cp = static_cast<const T*>(a.C) + p.b * a.C_stride_b + p.g * a.C_stride_g;
    const long long out_at = (long long)p.b * a.length * a.channels + p.d0 + quad;
    T* du = a.du ? static_cast<T*>(a.du) + out_at : nullptr;
    T* ddt = a.ddt ? static_cast<T*>(a.ddt) + out_at : nullptr;
    T* dz = a.dz && a.z ? static_cast<T*>(a.dz) + out_at : nullptr;
    // dB and dC: this block's row of the partial sums, for thread's value (token, B or C, state)
    const long long bc_all = (long long)a.batch * a.length * a.groups * N;
    float* bc = LOCAL ? nullptr : partial_bc + 2 * block * bc_all + ((long long)p.b * a.length * a.groups + p.g) * N;
    const int bc_stop = partial_bc ? stop : 0;                // formed, but kept nowhere, if not wanted: a question per tile costs 1 % of all calls
    auto store_bc = [&](int t, int m, int n, float v) {
        if (n < N) bc[m * bc_all + (long long)t * a.groups * N + n] = v;
    };

    Quad<T> u[PAIRS], u_next[PAIRS], dt_next[PAIRS], z_next[PAIRS], dy_next[PAIRS], b_next[BCS], c_next[BCS];
    const int kept = (a.length + KEEP - 1) / KEEP;
    const bool whole_kept = whole_states(a.checkpoints, N);
    auto fetch = [&](int t0) {                                // a tile's inputs; zeros behind the sequence's end
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const int r = row + i * ROWS, t = t0 + r, v = (FULL || r < KEEP) && t < stop ? valid : 0;
            if (!LOCAL) u_next[i] = fetch_quad<T>(up + t * a.u_stride_t, v, aligned);
            dt_next[i] = fetch_quad<T>(dtp + t * a.dt_stride_t, v, aligned);
            if (zp) z_next[i] = fetch_quad<T>(zp + t * a.z_stride_t, v, aligned);
            dy_next[i] = dyp ? fetch_quad<T>(dyp + t * a.dy_stride_t, v, aligned) : quad_zero<T>();
        }
#pragma unroll
        for (int i = 0; i < BCS; ++i) {
            const int q = lane + 32 * i, t = t0 + q / (S::NS / 4), n = q % (S::NS / 4) * 4, v = t < stop && q < BCQ ? N - n : 0;
            if (!LOCAL) b_next[i] = fetch_quad<T>(Bp + t * a.B_stride_t + n, v, aligned_bc);
            c_next[i] = fetch_quad<T>(Cp + t * a.C_stride_t + n, v, aligned_bc);
        }
    };
    // The sums over tokens of the last FLUSH tiles are added to those in memory: in registers alone their rounding errors would grow with the
    // sequence, and second accumulators there would spill.
    float* pa = LOCAL ? nullptr : partial_a + ((long long)p.b * split.chunks + chunk) * a.channels * (N + 2);
    auto flush = [&](bool first) {
        auto put = [&](int d, int n, float v) {
            float* to = pa + (long long)d * (N + 2) + n;
            *to = first ? v : *to + v;
        };
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (channels > 0 && sg * 4 + n < N) put(d0, sg * 4 + n, lo_of(dA[n]));
            if (channels > 1 && sg * 4 + n < N) put(d0 + 1, sg * 4 + n, hi_of(dA[n]));
            dA[n] = both(0.0f);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float skip = j & 1 ? hi_of(dD[j / 2]) : lo_of(dD[j / 2]), step = j & 1 ? hi_of(dbias[j / 2]) : lo_of(dbias[j / 2]);
#pragma unroll
            for (int o = S::QUADS; o < 32; o <<= 1) {         // over the rows
                skip += __shfl_xor_sync(0xffffffffu, skip, o);
                step += __shfl_xor_sync(0xffffffffu, step, o);
            }
            if (row == 0 && j < valid) {
                put(p.d0 + quad + j, N, skip);
                put(p.d0 + quad + j, N + 1, step);
            }
        }
        dD[0] = dD[1] = dbias[0] = dbias[1] = both(0.0f);
    };
    const int n_tiles = stop > begin ? (stop - begin + KEEP - 1) / KEEP : 0;
    if (!LOCAL) {                                             // padding
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int t = begin + n_tiles * KEEP + row; t < end; t += ROWS) {
            if (du) store_quad<T>(du + (long long)t * a.channels, valid, aligned, zero);
            if (ddt) store_quad<T>(ddt + (long long)t * a.channels, valid, aligned, zero);
            if (dz) store_quad<T>(dz + (long long)t * a.channels, valid, aligned, zero);
        }
        const int bc_end = partial_bc ? end : 0;
        for (int t = max(begin, stop); t < bc_end; ++t)
            for (int i = threadIdx.x; i < 2 * S::NS; i += 32 * BACK_WARPS) store_bc(t, i / S::NS, i % S::NS, 0.0f);
    }
    if (n_tiles > 0) fetch(begin + (n_tiles - 1) * KEEP);
    for (int k = n_tiles - 1; k >= 0; --k) {
        const int t0 = begin + k * KEEP;
        // on its way while the steps are formed: one tile ahead it would take registers from the walk over the tokens
        if (!LOCAL) load_states2(a.checkpoints + (((long long)p.b * kept + t0 / KEEP) * a.channels + d0) * N, channels, sg * 4, N, whole_kept, h);
        __syncwarp();                                         // the last tile has been read
        f32x2 raw_sig[PAIRS][2], dz_of[PAIRS][2];             // what ddelta and the ungated y are multiplied by for ddt and dz
        const float4 bias = *reinterpret_cast<const float4*>(&tile.bias[quad]);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const int r = row + i * ROWS;
            if (!LOCAL) u[i] = u_next[i];
            const float4 uv = LOCAL ? make_float4(0.f, 0.f, 0.f, 0.f) : widen<T>(u[i]), dv = widen<T>(dt_next[i]), yv = widen<T>(dy_next[i]);
            const f32x2 raw[2] = {add2(pair(dv.x, dv.y), pair(bias.x, bias.y)), add2(pair(dv.z, dv.w), pair(bias.z, bias.w))};
            f32x2 g[2] = {pair(yv.x, yv.y), pair(yv.z, yv.w)}, delta[2] = {raw[0], raw[1]};
            raw_sig[i][0] = raw_sig[i][1] = both(1.0f);
            if (a.softplus) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float e0 = exp_minus_abs(lo_of(raw[j])), e1 = exp_minus_abs(hi_of(raw[j]));
                    raw_sig[i][j] = pair(sigmoid_of(lo_of(raw[j]), e0), sigmoid_of(hi_of(raw[j]), e1));
                    delta[j] = softplus2(lo_of(raw[j]), hi_of(raw[j]), e0, e1);
                }
            }
            if (zp) {
                const float4 zv = widen<T>(z_next[i]);
                const f32x2 zz[2] = {pair(zv.x, zv.y), pair(zv.z, zv.w)};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f32x2 s = sigmoid2(zz[j]);
                    dz_of[i][j] = mul2(g[j], silu_slope2(zz[j], s));
                    g[j] = mul2(g[j], mul2(zz[j], s));
                }
            }
            const uint32_t live = t0 + r < stop ? 0xffffffffu : 0u;
            if (FULL || r < KEEP) {
                const int at = r * S::QUADS + quad / 4;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    delta[j] = pair(__uint_as_float(__float_as_uint(lo_of(delta[j])) & live), __uint_as_float(__float_as_uint(hi_of(delta[j])) & live));
                    const f32x2 d_u = mul2(delta[j], j ? pair(uv.z, uv.w) : pair(uv.x, uv.y));
                    tile.steps[j][at] = make_float4(lo_of(delta[j]), hi_of(delta[j]), lo_of(d_u), hi_of(d_u));
                }
                *reinterpret_cast<float4*>(&tile.dyg[r][quad]) = make_float4(lo_of(g[0]), hi_of(g[0]), lo_of(g[1]), hi_of(g[1]));
            }
        }
#pragma unroll
        for (int i = 0; i < BCS; ++i) {
            const int q = lane + 32 * i, r = q / (S::NS / 4), n = q % (S::NS / 4);
            if (BCQ % 32 != 0 && q >= BCQ) continue;
            if (!LOCAL) {
                const float4 bv = widen<T>(b_next[i]);
                tile.b[r][n] = bv;
            }
            const float4 cv = widen<T>(c_next[i]);
            tile.c[r][n] = cv;
        }
        __syncwarp();
        if (k > 0) fetch(t0 - KEEP);
        if (!LOCAL) {                                         // the tile's states
#pragma unroll 4                                              // 4 x 1024 x 8192: two 924 us, four 893, eight 933 (registers)
            for (int t = 0; t < KEEP; ++t) {
                tile.h[t][0][lane] = make_float4(lo_of(h[0]), hi_of(h[0]), lo_of(h[1]), hi_of(h[1]));
                tile.h[t][1][lane] = make_float4(lo_of(h[2]), hi_of(h[2]), lo_of(h[3]), hi_of(h[3]));
                f32x2 B[4];
                load_twice(tile.b, t, sg, B);
                const float4 s = tile.steps[cg & 1][t * S::QUADS + (cg >> 1)];
#pragma unroll
                for (int n = 0; n < 4; ++n) h[n] = fma2(decay_of(A[n], pair(s.x, s.y)), h[n], mul2(pair(s.z, s.w), B[n]));
            }
        }
#pragma unroll 4
        for (int t = KEEP - 1; t >= 0; --t) {
            f32x2 C[4], g[4];
            load_twice(tile.c, t, sg, C);
            const float4 s = tile.steps[cg & 1][t * S::QUADS + (cg >> 1)];
            const f32x2 dl = pair(s.x, s.y), du2 = pair(s.z, s.w);
            const float2 dv = *reinterpret_cast<const float2*>(&tile.dyg[t][2 * cg]);
            const f32x2 dyg = pair(dv.x, dv.y);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                g[n] = fma2(C[n], dyg, adj[n]);
                adj[n] = mul2(decay_of(A[n], dl), g[n]);
            }
            if (LOCAL) {
                dsum[0] += s.x;
                dsum[1] += s.y;
            } else {
                const float4 p0 = tile.h[t][0][lane], p1 = tile.h[t][1][lane];
                const f32x2 before[4] = {pair(p0.x, p0.y), pair(p0.z, p0.w), pair(p1.x, p1.y), pair(p1.z, p1.w)};
                f32x2 B[4], y = both(0.0f), gb = both(0.0f), wa = both(0.0f);
                load_twice(tile.b, t, sg, B);
                float sums[8];                                // dB, dC of the lane's two channels
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    y = fma2(h[n], C[n], y);
                    gb = fma2(g[n], B[n], gb);
                    const f32x2 w = mul2(adj[n], before[n]), db = mul2(g[n], du2), dc = mul2(h[n], dyg);
                    wa = fma2(w, A[n], wa);
                    dA[n] = fma2(w, dl, dA[n]);
                    sums[n] = lo_of(db) + hi_of(db);
                    sums[4 + n] = lo_of(dc) + hi_of(dc);
                    h[n] = before[n];
                }
                __syncwarp();                                 // the state before token t has been read by all lanes
                float* out = reinterpret_cast<float*>(tile.h[t]) + sg * S::CW + 2 * cg;
                *reinterpret_cast<float2*>(out) = make_float2(lo_of(y), hi_of(y));
                *reinterpret_cast<float2*>(out + S::SG * S::CW) = make_float2(lo_of(gb), hi_of(gb));
                *reinterpret_cast<float2*>(out + 2 * S::SG * S::CW) = make_float2(lo_of(wa), hi_of(wa));
                bc_sums<S>(sums, tile.bc[k & 1][t], sg, cg);
            }
        }
        if (LOCAL) continue;
        __syncthreads();                                      // all warps' dB and dC of this tile; the last one's were of the other buffer
        for (int i = threadIdx.x; i < KEEP * 2 * S::NS; i += 32 * BACK_WARPS) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < BACK_WARPS; ++w) v += reinterpret_cast<const float*>(tiles[w].bc[k & 1])[i];
            const int t = t0 + i / (2 * S::NS);
            if (t < bc_stop) store_bc(t, i / S::NS & 1, i % S::NS, v);        // not padding's: zero times a state that may not be finite
        }
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const int r = row + i * ROWS, t = t0 + r;
            const float* in = reinterpret_cast<const float*>(tile.h[r % KEEP]) + quad;
            f32x2 sum[3][2];
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                sum[q][0] = sum[q][1] = both(0.0f);
#pragma unroll
                for (int s = 0; s < S::SG; ++s) {             // odd rows start with the other half of the banks
                    const float4 v = *reinterpret_cast<const float4*>(in + q * S::SG * S::CW + (s ^ (r & 1)) * S::CW);
                    sum[q][0] = add2(sum[q][0], pair(v.x, v.y));
                    sum[q][1] = add2(sum[q][1], pair(v.z, v.w));
                }
            }
            const float4 uv = widen<T>(u[i]), gv = *reinterpret_cast<const float4*>(&tile.dyg[r % KEEP][quad]);
            const float4 Dv = *reinterpret_cast<const float4*>(&tile.D[quad]);
            float4 o_u, o_t, o_z;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 dl = *reinterpret_cast<const float2*>(&tile.steps[j][r % KEEP * S::QUADS + quad / 4]);
                const f32x2 uu = j ? pair(uv.z, uv.w) : pair(uv.x, uv.y), dyg = j ? pair(gv.z, gv.w) : pair(gv.x, gv.y), D = j ? pair(Dv.z, Dv.w) : pair(Dv.x, Dv.y);
                const f32x2 ou = fma2(D, dyg, mul2(pair(dl.x, dl.y), sum[1][j]));
                const f32x2 ot = mul2(fma2(sum[2][j], both(LN2), mul2(uu, sum[1][j])), raw_sig[i][j]);       // A was times log2(e)
                const f32x2 oz = zp ? mul2(dz_of[i][j], fma2(D, uu, sum[0][j])) : both(0.0f);
                (j ? o_u.z : o_u.x) = lo_of(ou); (j ? o_u.w : o_u.y) = hi_of(ou);
                (j ? o_t.z : o_t.x) = lo_of(ot); (j ? o_t.w : o_t.y) = hi_of(ot);
                (j ? o_z.z : o_z.x) = lo_of(oz); (j ? o_z.w : o_z.y) = hi_of(oz);
                if ((FULL || r < KEEP) && t < stop) {
                    dD[j] = fma2(dyg, uu, dD[j]);
                    dbias[j] = add2(dbias[j], ot);
                }
            }
            if ((FULL || r < KEEP) && t < end) {
                const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
                const bool on = t < stop;
                if (du) store_quad<T>(du + (long long)t * a.channels, valid, aligned, on ? o_u : zero);
                if (ddt) store_quad<T>(ddt + (long long)t * a.channels, valid, aligned, on ? o_t : zero);
                if (dz) store_quad<T>(dz + (long long)t * a.channels, valid, aligned, on ? o_z : zero);
            }
        }
        if (k % FLUSH == 0) flush(k / FLUSH == (n_tiles - 1) / FLUSH);
    }
    if (LOCAL) {
        const long long at = ((long long)p.b * split.chunks + chunk) * a.channels + d0;
        store_states2(split.states + at * N, channels, sg * 4, N, whole_states(split.states, N), adj);
        if (sg == 0 && channels > 0) split.deltas[at] = dsum[0];
        if (sg == 0 && channels > 1) split.deltas[at + 1] = dsum[1];
        return;
    }
    if (a.d_initial_state && chunk == 0) store_states2(a.d_initial_state + ((long long)p.b * a.channels + d0) * N, channels, sg * 4, N, whole_states(a.d_initial_state, N), adj);
    if (n_tiles == 0) flush(true);
}

template <typename T>
__global__ void __launch_bounds__(256)
scan_bc_sums_kernel(const float* __restrict__ partial, int parts, long long all, T* __restrict__ dB, T* __restrict__ dC) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * all) return;
    T* out = i < all ? dB : dC;
    if (!out) return;
    float s = 0.0f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) s += partial[2 * p * all + i];
    out[i < all ? i : i - all] = from_float<T>(s);
}

static __global__ void __launch_bounds__(256)
scan_a_sums_kernel(const float* __restrict__ partial, int parts, int channels, int N, float* __restrict__ dA, float* __restrict__ dD,
                   float* __restrict__ dbias) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)channels * (N + 2);
    if (i >= all) return;
    float s = 0.0f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) s += partial[p * all + i];
    const int d = (int)(i / (N + 2)), n = (int)(i % (N + 2));
    if (n < N) {
        if (dA) dA[(long long)d * N + n] = s;
    } else if (n == N) {
        if (dD) dD[d] = s;
    } else if (dbias) {
        dbias[d] = s;
    }
}

// ---- one token ----------------------------------------------------------------------------------------------------------

// LANES lanes share a channel, four states each, and go through the sequences of their block's share: A is read once for them.
// Bound: memory, the state read and written (128 bytes per channel of 16 states); for few sequences one memory latency.
template <typename T, int LANES>
__global__ void __launch_bounds__(128)
selective_scan_step_kernel(const el_scan_t a, int share) {
    const int lane = threadIdx.x % LANES, d = (blockIdx.x * 128 + threadIdx.x) / LANES, n0 = lane * 4, N = a.states;
    const bool real = d < a.channels;
    const int dc = min(d, a.channels - 1), g = dc / (a.channels / a.groups);
    const int b0 = blockIdx.y * share, b1 = min(b0 + share, a.batch);
    const bool aligned_bc = N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C)) % (4 * sizeof(T)) == 0 &&
                            (a.B_stride_b | a.B_stride_g | a.C_stride_b | a.C_stride_g) % 4 == 0;
    float A[4];
    load_states(a.A + (long long)dc * N, n0, N, whole_states(a.A, N), A);
    const float bias = a.dt_bias ? a.dt_bias[dc] : 0.0f, D = a.D ? a.D[dc] : 0.0f;
#pragma unroll
    for (int n = 0; n < 4; ++n) A[n] *= LOG2E;                // infinite ones too: there is no padding here
    const bool whole = whole_states(a.initial_state, N) && whole_states(a.final_state, N);
    // The next sequence's inputs are fetched ahead: the compiler itself cannot move loads of a state before the stores of another one.  64 sequences of
    // 8192 channels: 25.6 -> 20.5 us; two ahead 20.8.
    struct Inputs { float h[4]; T u, dt, z; Quad<T> B, C; };
    auto fetch = [&](int b, Inputs& in) {
        load_states(a.initial_state + ((long long)b * a.channels + dc) * N, n0, N, whole, in.h);
        in.u = static_cast<const T*>(a.u)[b * a.u_stride_b + dc];
        in.dt = static_cast<const T*>(a.dt)[b * a.dt_stride_b + dc];
        in.z = a.z ? static_cast<const T*>(a.z)[b * a.z_stride_b + dc] : T(0.0f);
        in.B = fetch_quad<T>(static_cast<const T*>(a.B) + b * a.B_stride_b + g * a.B_stride_g + n0, N - n0, aligned_bc);
        in.C = fetch_quad<T>(static_cast<const T*>(a.C) + b * a.C_stride_b + g * a.C_stride_g + n0, N - n0, aligned_bc);
    };
    Inputs next;
    if (b0 < b1) fetch(b0, next);
    for (int b = b0; b < b1; ++b) {
        const Inputs now = next;
        if (b + 1 < b1) fetch(b + 1, next);
        const long long at = ((long long)b * a.channels + dc) * N;
        const float u = to_float<T>(now.u), raw = to_float<T>(now.dt) + bias;
        const float delta = a.softplus ? softplus_of(raw, exp_minus_abs(raw)) : raw, du = delta * u;
        const float4 B = widen<T>(now.B), C = widen<T>(now.C);
        const float Bv[4] = {B.x, B.y, B.z, B.w}, Cv[4] = {C.x, C.y, C.z, C.w};
        float h[4], y = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            h[n] = __fmaf_rn(ex2(__fmaf_rn(A[n], delta, DECAY_SHIFT)), now.h[n], du * Bv[n]);
            y = __fmaf_rn(Cv[n], h[n], y);
        }
        if (real) store_states(a.final_state + at, n0, N, whole, h);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
        if (real && lane == 0) {
            y = __fmaf_rn(D, u, y);
            const float z = to_float<T>(now.z);
            if (a.z) y *= z * sigmoid(z);
            static_cast<T*>(a.y)[(long long)b * a.channels + d] = from_float<T>(y);
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------

template <typename F> static int scan_by_type(int dtype, F f) {
    switch (dtype) {
        case EL_F16: return f(__half());
        case EL_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}
// The number of states is rounded up to a power of two from 8 on; states that a channel does not have stay zero.
template <typename F> static int scan_by_shape(const el_scan_t& a, F f) {
    if (a.states <= 8) return f(Shape<8>());
    if (a.states <= 16) return f(Shape<16>());
    if (a.states <= 32) return f(Shape<32>());
    return f(Shape<64>());
}
static long long parts_of(const el_scan_t& a, int width) {     // pieces of that many channels, none of them in two groups
    return (long long)a.batch * a.groups * ((a.channels / a.groups + width - 1) / width);
}

// A sequence is cut into chunks when its channels leave much of the GPU idle: all chunks run side by side, first for the state that each adds on
// its own (half of a forward pass again, a quarter of a backward pass), then, from the states that those give, for the outputs.  As many chunks as the
// SMs take at once (`slots` warps each): one more would be a second round.  Below `enough` warps an SM, as measured, 16 states, us:
//   forward (slots 8, enough 3)    16384 x 2048 channels 0.9 warps an SM: 9 chunks 417, 10 chunks 568;  4096 x 8192 3.5: whole 343, 2 chunks 464
//   backward (slots 16, enough 12) 4096 x 8192 channels 3.5: whole 3459, 4 chunks 1138;  4 x 1024 x 8192 13.8: whole 915, 2 chunks 1263 (1093 and 874 now)
static ScanSplit scan_split(const el_scan_t& a, long long warps, int slots, int enough, float* states) {
    int sms = 148;
    device_sm_count(&sms);
    ScanSplit s = {1, a.length > 0 ? a.length : 1, states, nullptr};
    if (warps > 0 && warps < (long long)enough * sms) {
        long long chunks = (long long)slots * sms / warps;
        if (chunks > 32) chunks = 32;                         // a chunk's first warps go through those before it one by one
        if (chunks > a.length / 64) chunks = a.length / 64;
        if (chunks >= 2) {
            s.tokens = (int)((a.length + chunks - 1) / chunks + TILE - 1) / TILE * TILE;
            s.chunks = (int)(((long long)a.length + s.tokens - 1) / s.tokens);       // length + tokens may pass 31 bits; a chunk's end does not
        }
    }
    s.deltas = states + (size_t)a.batch * s.chunks * a.channels * a.states;
    return s;
}
template <typename S> static ScanSplit forward_split(const el_scan_t& a, float* states) {
    return scan_split(a, parts_of(a, S::CW), S::PER_SM / 2, S::PER_SM * 3 / 16, states);
}
static size_t split_floats(const el_scan_t& a, const ScanSplit& s) { return s.chunks > 1 ? (size_t)a.batch * s.chunks * a.channels * (a.states + 1) : 0; }

size_t selective_scan_checkpoint_bytes(const el_scan_t& a) {
    return (size_t)a.batch * ((a.length + KEEP - 1) / KEEP) * a.channels * a.states * sizeof(float);
}
size_t selective_scan_workspace_bytes(const el_scan_t& a) {
    if (a.batch == 0 || a.channels == 0) return 0;
    size_t floats = 0;
    scan_by_shape(a, [&](auto shape) {
        floats = split_floats(a, forward_split<decltype(shape)>(a, nullptr));
        return EL_OK;
    });
    return floats * sizeof(float);
}

// Backward's workspace: partial sums of dB and dC, of dA, dD and dbias, and the chunks' states.
// dB and dC, the larger part, have no room where neither is wanted; a struct that names no gradient yet asks for all of them.
struct ScanBackwardPlan { ScanSplit split; long long blocks; float *bc, *a; size_t floats; };
static bool scan_wants_bc(const el_scan_t& a) {
    return a.dB || a.dC || !(a.du || a.ddt || a.dz || a.dA || a.dD || a.ddt_bias || a.d_initial_state);
}
template <typename S> static ScanBackwardPlan scan_backward_plan(const el_scan_t& a, float* ws) {
    ScanBackwardPlan p;
    p.blocks = parts_of(a, S::CW * BACK_WARPS);
    p.split = scan_split(a, parts_of(a, S::CW), S::BACK_PER_SM, S::BACK_PER_SM * 3 / 4, nullptr);
    const size_t per_group = (a.channels / a.groups + S::CW * BACK_WARPS - 1) / (S::CW * BACK_WARPS);
    const size_t n_bc = scan_wants_bc(a) ? 2 * per_group * a.batch * a.length * a.groups * a.states : 0, n_a = (size_t)a.batch * p.split.chunks * a.channels * (a.states + 2);
    p.bc = n_bc ? ws : nullptr;
    p.a = ws + n_bc;
    p.split.states = p.a + n_a;
    p.split.deltas = p.split.states + (size_t)a.batch * p.split.chunks * a.channels * a.states;
    p.floats = n_bc + n_a + split_floats(a, p.split);
    return p;
}
size_t selective_scan_backward_workspace_bytes(const el_scan_t& a) {
    if (a.batch == 0 || a.channels == 0) return 0;
    size_t floats = 0;
    scan_by_shape(a, [&](auto shape) {
        floats = scan_backward_plan<decltype(shape)>(a, nullptr).floats;
        return EL_OK;
    });
    return floats * sizeof(float);
}

// Whether four channels of each activation can be read at once: bases and strides are whole vectors, groups too.
static bool scan_vector(const void* p, long long s0, long long s1, long long s2, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % (dtype == EL_F32 ? 16 : 8) == 0 && s0 % 4 == 0 && s1 % 4 == 0 && s2 % 4 == 0;
}
static bool scan_aligned(const el_scan_t& a) {
    return a.channels / a.groups % 4 == 0 && scan_vector(a.u, a.u_stride_b, a.u_stride_t, 0, a.dtype) &&
           scan_vector(a.dt, a.dt_stride_b, a.dt_stride_t, 0, a.dtype) && scan_vector(a.z, a.z_stride_b, a.z_stride_t, 0, a.dtype) &&
           scan_vector(a.y, 0, 0, 0, a.dtype) && scan_vector(a.dy, a.dy_stride_b, a.dy_stride_t, 0, a.dtype) && scan_vector(a.du, 0, 0, 0, a.dtype) &&
           scan_vector(a.ddt, 0, 0, 0, a.dtype) && scan_vector(a.dz, 0, 0, 0, a.dtype);
}
static bool scan_aligned_bc(const el_scan_t& a) {
    return a.states % 4 == 0 && scan_vector(a.B, a.B_stride_b, a.B_stride_t, a.B_stride_g, a.dtype) &&
           scan_vector(a.C, a.C_stride_b, a.C_stride_t, a.C_stride_g, a.dtype);
}

// Allows a kernel its shared memory, once per device.
template <typename K> static int scan_shared(K kernel, int bytes, DeviceOnce& once) {
    int dev = 0;
    EL_CUDA_TRY(cudaGetDevice(&dev));
    if (!once.is_done(dev)) {
        EL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        once.mark(dev);
    }
    return EL_OK;
}

template <typename T, typename S, bool LOCAL> static int launch_scan_pass(const el_scan_t& a, const ScanSplit& s, long long warps, cudaStream_t st) {
    constexpr int shared = 2 * COUPLES * sizeof(Tile<S>);
    static DeviceOnce once;
    const int rc = scan_shared(selective_scan_kernel<T, S, LOCAL>, shared, once);
    if (rc != EL_OK) return rc;
    const dim3 grid((unsigned)((warps + COUPLES - 1) / COUPLES), s.chunks);
    selective_scan_kernel<T, S, LOCAL><<<grid, 64 * COUPLES, shared, st>>>(a, s, scan_aligned(a), scan_aligned_bc(a));
    return check_launch();
}

int launch_selective_scan(const el_scan_t& a, cudaStream_t st) {
    return scan_by_type(a.dtype, [&](auto t) {
        return scan_by_shape(a, [&](auto shape) {
            using T = decltype(t);
            using S = decltype(shape);
            const long long warps = parts_of(a, S::CW);
            if (warps > (1ll << 31) - COUPLES) return (int)EL_ERR_TOO_LARGE;
            const ScanSplit s = forward_split<S>(a, static_cast<float*>(a.workspace));
            const int rc = s.chunks > 1 ? launch_scan_pass<T, S, true>(a, s, warps, st) : EL_OK;
            return rc != EL_OK ? rc : launch_scan_pass<T, S, false>(a, s, warps, st);
        });
    });
}

template <typename T, typename S, bool LOCAL> static int launch_scan_backward_pass(const el_scan_t& a, const ScanBackwardPlan& p, cudaStream_t st) {
    constexpr int shared = BACK_WARPS * sizeof(BackTile<S>);
    static DeviceOnce once;
    const int rc = scan_shared(selective_scan_backward_kernel<T, S, LOCAL>, shared, once);
    if (rc != EL_OK) return rc;
    const dim3 grid((unsigned)p.blocks, p.split.chunks);
    selective_scan_backward_kernel<T, S, LOCAL><<<grid, 32 * BACK_WARPS, shared, st>>>(a, p.split, scan_aligned(a), scan_aligned_bc(a), p.bc, p.a);
    return check_launch();
}

int launch_selective_scan_backward(const el_scan_t& a, cudaStream_t st) {
    return scan_by_type(a.dtype, [&](auto t) {
        return scan_by_shape(a, [&](auto shape) {
            using T = decltype(t);
            using S = decltype(shape);
            const ScanBackwardPlan p = scan_backward_plan<S>(a, static_cast<float*>(a.workspace));
            if (p.blocks > (1ll << 31) - 1) return (int)EL_ERR_TOO_LARGE;
            int rc = EL_OK;
            if (p.blocks > 0) {                               // else all sums are empty: zeros
                if (p.split.chunks > 1) rc = launch_scan_backward_pass<T, S, true>(a, p, st);
                if (rc == EL_OK) rc = launch_scan_backward_pass<T, S, false>(a, p, st);
            }
            if (rc != EL_OK) return rc;
            const long long all = (long long)a.batch * a.length * a.groups * a.states, cols = (long long)a.channels * (a.states + 2);
            if ((a.dB || a.dC) && all > 0) {
                scan_bc_sums_kernel<T><<<(unsigned)((2 * all + 255) / 256), 256, 0, st>>>(p.bc, (int)(p.blocks / ((long long)a.batch * a.groups)), all,
                                                                                         static_cast<T*>(a.dB), static_cast<T*>(a.dC));
                if ((rc = check_launch()) != EL_OK) return rc;
            }
            if ((a.dA || a.dD || a.ddt_bias) && cols > 0)
                scan_a_sums_kernel<<<(unsigned)((cols + 255) / 256), 256, 0, st>>>(p.a, a.batch * p.split.chunks, a.channels, a.states, a.dA, a.dD,
                                                                                 a.ddt_bias);
            return check_launch();
        });
    });
}

int launch_selective_scan_step(const el_scan_t& a, cudaStream_t st) {
    return scan_by_type(a.dtype, [&](auto t) {
        auto launch = [&](auto lanes) {
            constexpr int LANES = decltype(lanes)::value;
            const long long blocks = ((long long)a.channels * LANES + 127) / 128;
            if (blocks > (1ll << 31) - 1) return (int)EL_ERR_TOO_LARGE;
            int sms = 148;
            device_sm_count(&sms);
            // sequences of a block: as many as leave every SM its 16 blocks
            long long share = blocks * a.batch / (16 * sms);
            share = share < 1 ? 1 : share > a.batch ? a.batch : share;
            while ((a.batch + share - 1) / share > 65535) ++share;
            selective_scan_step_kernel<decltype(t), LANES><<<dim3((unsigned)blocks, (unsigned)((a.batch + share - 1) / share)), 128, 0, st>>>(a, (int)share);
            return check_launch();
        };
        if (a.states <= 4) return launch(std::integral_constant<int, 1>());
        if (a.states <= 8) return launch(std::integral_constant<int, 2>());
        if (a.states <= 16) return launch(std::integral_constant<int, 4>());
        if (a.states <= 32) return launch(std::integral_constant<int, 8>());
        return launch(std::integral_constant<int, 16>());
    });
}

}  // namespace el
