// The absorbed form for 16-bit activations on the tensor cores (latent_step.cu has the formulas and the launches around it).
//
// The cached rows are int8 already, so they go to the tensor cores as they are (kind::i8, exact int32 sums) and nothing is dequantised: what multiplies
// them is split into two 8-bit digits instead, x = step * (256 hi + lo), 16 bits of a row's largest magnitude.  One copy of a tile of tokens in
// shared memory serves both products:
//   scores   S [128 tokens x 2 heads' digits] = rows (K-major: tokens by latent channels) * query digits;  with the rotated part in 16-bit floats beside it
//            s[j,h] = absmax[j] / 127 * step[h] * (256 S_hi + S_lo) + key[j] . w[h]
//   sums     O [latent channels x 2 heads' digits] = rows (MN-major: the same bytes, read as channels by tokens) * digits of p[j,h] absmax[j] / largest absmax
// p = 2^(s - m) with m the running maximum of the head, so p <= 1 and a digit step is 2^-15 of the largest weight that a token of the tile can have: finer
// than bfloat16's 2^-8 of each weight where weights matter.  The tiles' int32 sums are added up in float32 registers, scaled when m grows.
//
// Warps 0-7: thread t of each half is token t of the tile and takes 16 heads' scores; then two of the four blocks of 128 latent channels, a thread a channel.
// The sums of a tile are taken after the next tile's scores, so that the tensor core has work meanwhile.  Warp 8 issues the products.  Warps
// 9 and 10 load, each half of a tile's tokens: by tensor maps where pages are multiples of 8 tokens (a box lies in one page), otherwise by 16-byte
// asynchronous copies of each token's row.
// Bound: a tile of 128 tokens of rank 512 and 64 rotated channels is 82 KB, 3400 cycles of an SM's share of the HBM, and 2800 of its tensor core (36 products of some
// 75 cycles each: with 64 columns the left operand's way through shared memory sets their pace).  It takes 5100: scores 2500 and sums 1400 in the same eight warps, the
// rest waiting for the next scores.  Sequences of up to 8192 tokens, 64 of them, 32 heads: this kernel 59 of the step's 88 us, 3.1 TB/s.
#include "latent_step.cuh"
#include "latent_tc.cuh"

namespace el {

namespace tc {
int make_map(CUtensorMap* m, const void* base, uint64_t cols, uint64_t rows, uint64_t pitch, uint32_t box_cols, uint32_t box_rows, int swizzle_bytes);
}

using namespace tc;
using namespace latent;

namespace {

constexpr int TOKENS = 128, CHUNK = TOKENS * 128;      // a tile; 128 bytes of every token
constexpr int WARP_MMA = 8, WARP_LOAD = 9, THREADS = 11 * 32;
constexpr float STEPS = 32512.0f;                      // 127 * 256: the largest value of two digits whose high one is at most 127
constexpr float MAGIC = 12582912.0f;                   // 1.5 * 2^23: adding it rounds to an integer, whose low bits are the sum's

// bytes i of four words as one word
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t sel) { return prmt(prmt(a, b, sel), prmt(c, d, sel), 0x5410u); }
// the largest value of a warp's lanes, NaN if there is one
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// whether a barrier's phase has ended, without waiting for it (mbar_try may wait for a while)
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y) : "memory");
}
// bytes that a barrier's phase waits for, without an arrival
__device__ __forceinline__ void mbar_expect_tx_only(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// The parts of a worker's range: sequence after sequence, tile after tile.
struct Walk {
    const el_latent_step_t& a;
    long long t, last, before;
    int b;
    int p0, p1;                                        // positions of the current part
    __device__ Walk(const el_latent_step_t& args, long long first, long long end) : a(args), t(first), last(end) { step_find(a, first, b, before); open(); }
    __device__ __forceinline__ void open() {
        while (t < last) {
            const int n = step_tokens(a, b), here = (n + STEP_TILE - 1) / STEP_TILE;
            if (here > 0) {
                const long long stop = before + here < last ? before + here : last;
                p0 = (int)(t - before) * STEP_TILE;
                const long long e = (stop - before) * STEP_TILE;
                p1 = (int)(e < n ? e : n);
                return;
            }
            ++b;
        }
    }
    __device__ __forceinline__ bool more() const { return t < last; }
    __device__ __forceinline__ int tiles() const { return (p1 - p0 + TOKENS - 1) / TOKENS; }
    __device__ __forceinline__ void next() {
        const int here = step_tiles(a, b);
        t = before + here < last ? before + here : last;
        before += here;
        ++b;
        open();
    }
};

// Sums 16 values over a warp: lane l has the sum of value l % 16.
__device__ __forceinline__ float reduce16(const float (&v)[16]) {
    const int lane = threadIdx.x & 31;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v[i];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int i = 0; i < w; ++i) x[i] = (up ? x[i + w] : x[i]) + __shfl_xor_sync(0xffffffffu, up ? x[i] : x[i + w], w);
    }
    return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 16);
}

__device__ __forceinline__ float reduce16max(const float (&v)[16]) {
    const int lane = threadIdx.x & 31;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v[i];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int i = 0; i < w; ++i) x[i] = mamba::max_nan(up ? x[i + w] : x[i], __shfl_xor_sync(0xffffffffu, up ? x[i] : x[i + w], w));
    }
    return mamba::max_nan(x[0], __shfl_xor_sync(0xffffffffu, x[0], 16));
}
template <typename T>
__global__ void __launch_bounds__(THREADS, 1)
step_tc_kernel(const __grid_constant__ CUtensorMap tmRows, const __grid_constant__ CUtensorMap tmKeys, const el_latent_step_t a, const uint8_t* __restrict__ images,
               const float* __restrict__ steps, const StepParts parts, int workers, const int box_bits) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const StepImage image(a);
    const int box = box_bits ? 1 << box_bits : 0;                            // 8 to 32 tokens
    const int R = a.rank, P = a.rot_dim, HP = image.hp, N = 2 * HP, KC = image.chunks, key_steps = (R + 31) / 32, rot_steps = (P + 15) / 16;
    const int stage_bytes = (KC + (P ? 1 : 0)) * CHUNK;
    // two stages [rows][keys]; the query's image; p digits [tokens][128]
    const uint32_t q_at = base + 2 * stage_bytes, w_at = q_at + image.w_at(), p_at = q_at + image.bytes();
    uint8_t* tail = gen + (p_at - base) + CHUNK;
    float* scale_of = reinterpret_cast<float*>(tail);                       // [2][128]
    uint32_t* seen = reinterpret_cast<uint32_t*>(tail + 1024);              // [2][4]
    float* step_of = reinterpret_cast<float*>(tail + 1088);                 // [2][32], by part
    float* factor = reinterpret_cast<float*>(tail + 1344);                  // [2][32], by tile
    float* weight = reinterpret_cast<float*>(tail + 1600);                  // [2], by tile
    float* wmax = reinterpret_cast<float*>(tail + 1632);                    // [2 halves][2][4 warps][16 heads]
    float* smax = reinterpret_cast<float*>(tail + 2656);                    // [2 halves][2][4 warps]
    float* wsum = reinterpret_cast<float*>(tail + 2720);                    // [2 halves][4 warps][16 heads]
    float* heads_of = reinterpret_cast<float*>(tail + 3232);                // [8 warps][2][16 heads]: maxima and factors for the warp's own lanes
    const uint32_t bars = p_at + CHUNK + 4256;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (2 + s); };
    auto s_full = [&](int s) { return bars + 8u * (4 + s); };
    const uint32_t p_full = bars + 48, o_full = bars + 56, o_empty = bars + 64, q_empty = bars + 72;
    auto half_at = [&](int half) { return bars + 80u + 8u * half; };
    volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(tail + 4256 + 96);

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int w = blockIdx.x / image.groups, group = blockIdx.x - w * image.groups, h0 = group * 32;
    int32_t* status = a.dev_status;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(full(s), 2);
            mbar_init(empty(s), 1);
            mbar_init(s_full(s), 1);
            mbar_init(half_at(s), 4);
        }
        mbar_init(p_full, 8);
        mbar_init(o_full, 1);
        mbar_init(o_empty, 8);
        mbar_init(q_empty, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == WARP_MMA) tmem_alloc<512>(smem_u32((const void*)tmem_holder));
    if (box && warp == WARP_LOAD && elect_one()) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmRows) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmKeys) : "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = *tmem_holder;
    const uint32_t O = tmem, S = tmem + 256;                                // O of chunk c at 64 c; S of tile g at 128 (g & 1), its rotated part 64 further

    asm volatile("griddepcontrol.launch_dependents;");
    const long long tiles = step_all_tiles(a);
    workers = step_active(workers, tiles);
    const long long first = w < workers ? w * tiles / workers : 0, last = w < workers ? (w + 1) * tiles / workers : 0;

    if (warp >= WARP_LOAD) {
        // ================= loads =================
        const int mine = warp - WARP_LOAD;                                            // half of every tile's tokens
        int g = 0, part = 0;
        bool ok = true;
        if (first < last) {
            for (Walk k(a, first, last); k.more() && ok; k.next(), ++part) {
                const int count = k.tiles();
                for (int i = 0; i < count && ok; ++i, ++g) {
                    const int s = g & 1;
                    const uint32_t at = base + s * stage_bytes, gone = ((uint32_t)(g >> 1) & 1u) ^ 1u;
                    const int p = k.p0 + i * TOKENS;
                    long long row[2];
                    float sc[2];
                    if (box) {                                                  // lane l looks up box l
                        const int first_box = mine * 64 >> box_bits, pos = p + (first_box + lane) * box;
                        const long long start = lane * box < 64 && pos < k.p1 ? step_row(a, k.b, pos) : -1;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int to = q * 32 + lane;
                            const long long r = __shfl_sync(0xffffffffu, start, to >> box_bits);
                            row[q] = r >= 0 && p + mine * 64 + to < k.p1 ? r + (to & (box - 1)) : -1;
                            sc[q] = row[q] >= 0 ? a.absmax[row[q]] : 0.0f;
                        }
                        // the stage is taken for the time of most of a tile: the bytes come as far as the L2 meanwhile
                        if (g >= 2 && start >= 0) {
#pragma unroll 4
                            for (int c = 0; c < KC; ++c) tma_prefetch_2d(&tmRows, c * 128, (int)start);
                            if (P) tma_prefetch_2d(&tmKeys, 0, (int)start);
                        }
                        __syncwarp();
                        if (!mbar_wait_warp(empty(s), gone, status, 1)) { ok = false; break; }
                        const unsigned there = __ballot_sync(0xffffffffu, start >= 0);
                        if (elect_one()) mbar_expect_tx_only(full(s), __popc(there) * box * 128 * (KC + (P ? 1 : 0)) + (i == 0 && mine == 0 ? image.bytes() : 0));
                        __syncwarp();
                        if (start >= 0) {                                       // a lane loads its box
                            const uint32_t to = at + ((first_box + lane) << (box_bits + 7));
#pragma unroll 4
                            for (int c = 0; c < KC; ++c) tma_load_2d(to + c * CHUNK, &tmRows, full(s), c * 128, (int)start);
                            if (P) tma_load_2d(to + KC * CHUNK, &tmKeys, full(s), 0, (int)start);
                        }
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int pos = p + mine * 64 + q * 32 + lane;
                            row[q] = pos < k.p1 ? step_row(a, k.b, pos) : -1;
                            sc[q] = row[q] >= 0 ? a.absmax[row[q]] : 0.0f;
                        }
                        if (!mbar_wait_warp(empty(s), gone, status, 1)) { ok = false; break; }
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
#pragma unroll 8
                            for (int t = 0; t < 32; ++t) {
                                const long long r = __shfl_sync(0xffffffffu, row[q], t);
                                const int to = mine * 64 + q * 32 + t;
                                if (lane * 16 < R && r >= 0)
                                    copy16(at + (lane >> 3) * CHUNK + to * 128 + (((lane & 7) ^ (to & 7)) << 4), a.latents + r * R + lane * 16, true);
                            }
                            if (P) {
                                const int pieces = (P + 15) / 16 * 2;                 // of 8 channels, zeros behind the last
#pragma unroll 4
                                for (int t = 0; t < 32; t += 4) {
                                    const int tt = t + (lane >> 3), c = lane & 7, to = mine * 64 + q * 32 + tt;
                                    const long long r = __shfl_sync(0xffffffffu, row[q], tt);
                                    if (c < pieces) {
                                        const bool there = r >= 0 && c * 8 < P;
                                        copy16(at + KC * CHUNK + to * 128 + ((c ^ (to & 7)) << 4), there ? static_cast<const T*>(a.cache_keys) + r * P + c * 8 : a.cache_keys, there);
                                    }
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        scale_of[s * 128 + mine * 64 + q * 32 + lane] = __fdiv_rn(sc[q], 127.0f);
                        const uint32_t have = __ballot_sync(0xffffffffu, row[q] >= 0);
                        if (lane == 0) seen[s * 4 + mine * 2 + q] = have;
                    }
                    if (i == 0 && mine == 0) {                                        // the part's query
                        if (part > 0 && !mbar_wait_warp(q_empty, (uint32_t)(part - 1) & 1u, status, 2)) { ok = false; break; }
                        griddep_wait();                                               // the kernel in front made it
                        const long long bg = (long long)k.b * image.groups + group;
                        if (elect_one()) {
                            if (!box) mbar_expect_tx_only(full(s), image.bytes());
                            bulk_load(q_at, images + bg * image.bytes(), image.bytes(), full(s));
                        }
                        __syncwarp();
                        step_of[(part & 1) * 32 + lane] = lane < HP ? steps[bg * 32 + lane] : 0.0f;
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full(s));
                }
            }
        }
    } else if (warp == WARP_MMA) {
        // ================= products =================
        const uint32_t i_s = make_idesc(0, 0, N), i_o = make_idesc(1, 1, N), i_r = idesc_f16<T>(0, 0, HP);
        auto scores = [&](int g) {
            const uint32_t at = base + (g & 1) * stage_bytes, to = S + (g & 1) * 128;
            for (int k = 0; k < key_steps; ++k) {
                const int c = k >> 2, x = (k & 3) * 32;
                umma_i8(to, make_desc(at + c * CHUNK + x, 16), make_desc(q_at + c * N * 128 + x, 16), i_s, k != 0);
            }
            for (int k = 0; k < rot_steps; ++k) umma_f16(to + 64, make_desc(at + KC * CHUNK + k * 32, 16), make_desc(w_at + k * 32, 16), i_r, k != 0);
            umma_commit(s_full(g & 1));
        };
        auto sums = [&](int g) {
            const uint32_t at = base + (g & 1) * stage_bytes;
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int k = 0; k < TOKENS / 32; ++k) umma_i8(O + c * 64, make_desc(at + c * CHUNK + k * 4096, CHUNK), make_desc(p_at + k * 4096, CHUNK), i_o, k != 0);
            umma_commit(o_full);
            umma_commit(empty(g & 1));
        };
        if (first < last) {
            // Scores of a tile as soon as it is there and the threads have read those of two tiles before; sums of a tile as soon as its digits are there and the
            // sums before have been taken.  Whichever is ready goes first.
            Walk k(a, first, last);
            int g = 0, left = k.tiles(), done = 0, total = -1;                        // scores issued, tiles of the part without them, sums issued
            long long since = clock64();
            while (true) {
                bool moved = false;
                if (total < 0 && g < done + 2 && __all_sync(0xffffffffu, mbar_test(full(g & 1), (uint32_t)(g >> 1) & 1u))) {
                    tcgen05_fence_after();
                    --left;
                    if (elect_one()) {
                        scores(g);
                        if (left == 0) umma_commit(q_empty);
                    }
                    __syncwarp();
                    ++g;
                    if (left == 0) {
                        k.next();
                        if (k.more()) left = k.tiles();
                        else total = g;
                    }
                    moved = true;
                }
                if (done < g && __all_sync(0xffffffffu, mbar_test(p_full, (uint32_t)done & 1u)) &&
                    (done == 0 || __all_sync(0xffffffffu, mbar_test(o_empty, (uint32_t)(done - 1) & 1u)))) {
                    tcgen05_fence_after();
                    if (elect_one()) sums(done);
                    __syncwarp();
                    ++done;
                    moved = true;
                }
                if (done == total) break;
                const long long now = clock64();
                if (moved) since = now;
                const bool lost = now - since > WAIT_LIMIT_CYCLES ||
                                  (now - since > (1 << 22) && status != nullptr && *reinterpret_cast<volatile int32_t*>(status) != 0);
                if (__any_sync(0xffffffffu, lost)) {
                    if (status != nullptr) atomicCAS(status, 0, 3);
                    break;
                }
            }
        }
    } else if (first < last) {
        // ================= softmax and sums =================
        const int half = warp >> 2, quarter = warp & 3, token = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const bool scoring = half * 16 < HP;                                          // 16 heads have one half
        float acc[2][32];                                                             // channels of chunks 2 half, 2 half + 1; heads
        float top = -INFINITY, sum[16];                                               // of head lane % 16; of all
        bool ok = true;
        int g = 0, part = 0;
        uint32_t met = 0;
        // The four warps of a half meet.  (A bar.sync would wait for good for a warp whose bounded wait gave up.)
        auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(half_at(half));
            ok = mbar_wait_warp(half_at(half), met & 1u, status, 9);
            ++met;
            return ok;
        };

        auto softmax = [&](int j) {
            if (!(ok = mbar_wait_warp(s_full(j & 1), (uint32_t)(j >> 1) & 1u, status, 6) && mbar_wait_warp(full(j & 1), (uint32_t)(j >> 1) & 1u, status, 6))) return;
            tcgen05_fence_after();
            float s[16];
            const float sc = scale_of[(j & 1) * 128 + token];
            const bool here = (seen[(j & 1) * 4 + quarter] >> lane) & 1u;
            float* wm = wmax + (half * 2 + (j & 1)) * 64;
            float* sm = smax + (half * 2 + (j & 1)) * 4;
            if (scoring) {
                uint32_t hi[16], lo[16];
                const uint32_t at = S + (j & 1) * 128 + lanes + half * 16;
                tmem_ld16(at, hi);
                tmem_ld16(at + HP, lo);
                tmem_ld_wait();
                const float4* st = reinterpret_cast<const float4*>(step_of + (part & 1) * 32 + half * 16);
#pragma unroll
                for (int h = 0; h < 16; h += 4) {
                    const float4 x = st[h / 4];
                    s[h] = (float)(int)(hi[h] * 256u + lo[h]) * (sc * x.x);
                    s[h + 1] = (float)(int)(hi[h + 1] * 256u + lo[h + 1]) * (sc * x.y);
                    s[h + 2] = (float)(int)(hi[h + 2] * 256u + lo[h + 2]) * (sc * x.z);
                    s[h + 3] = (float)(int)(hi[h + 3] * 256u + lo[h + 3]) * (sc * x.w);
                }
                if (P) {
                    tmem_ld16(at + 64, hi);
                    tmem_ld_wait();
#pragma unroll
                    for (int h = 0; h < 16; ++h) s[h] += __uint_as_float(hi[h]);
                }
#pragma unroll
                for (int h = 0; h < 16; ++h) s[h] = here ? s[h] : -INFINITY;
                const float most = reduce16max(s);
                if (lane < 16) wm[quarter * 16 + lane] = most;
            }
            float big = warp_max(here ? sc : 0.0f);
            if (lane == 0) sm[quarter] = big;
            if (!meet()) return;
            const float4 b4 = *reinterpret_cast<const float4*>(sm);
            big = fmaxf(fmaxf(b4.x, b4.y), fmaxf(b4.z, b4.w));
            const float ratio = big > 0.0f ? sc * (STEPS / big) : 0.0f;
            float scale = 1.0f;
            uint32_t dh[4], dl[4];
            if (scoring) {
                // lane l (and l + 16) has head l's running maximum; every thread needs all of them
                const int h0 = lane & 15;
                const float m = mamba::max_nan(mamba::max_nan(mamba::max_nan(wm[h0], wm[16 + h0]), mamba::max_nan(wm[32 + h0], wm[48 + h0])), top);
                const bool moved = __any_sync(0xffffffffu, m != top);                // the same for all warps of the half
                float* own = heads_of + warp * 32;
                const float f = m == top ? 1.0f : top == -INFINITY ? 0.0f : exp2_neg(top - m);
                own[h0] = m;
                if (moved) own[16 + h0] = f;
                top = m;
                __syncwarp();
                if (moved) {
#pragma unroll
                    for (int h = 0; h < 16; h += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(own + 16 + h);
                        sum[h] *= x.x;
                        sum[h + 1] *= x.y;
                        sum[h + 2] *= x.z;
                        sum[h + 3] *= x.w;
                    }
                }
                scale = f;
                uint32_t v[16];
#pragma unroll
                for (int h = 0; h < 16; h += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(own + h);
                    const float t[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = here ? exp2_neg(s[h + e] - t[e]) : 0.0f;
                        sum[h + e] += y;
                        v[h + e] = __float_as_uint(fmaf(y, ratio, MAGIC));            // the integer is its low 16 bits: MAGIC's are zeros
                    }
                }
                __syncwarp();                                                         // `own` is free again
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    dl[h] = bytes_of(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3], 0x0040u);
                    dh[h] = bytes_of(v[4 * h] + 128u, v[4 * h + 1] + 128u, v[4 * h + 2] + 128u, v[4 * h + 3] + 128u, 0x0051u);
                }
            }
            // The products of the tile before have read its digits, and were issued after all warps took the sums of the tile before that one: the digits, and the
            // factors of two tiles before, may be overwritten.  (Both phases are still the barriers' last ones: the next cannot end without this warp.)
            if (j > 0 && !(ok = mbar_wait_warp(o_full, (uint32_t)(j - 1) & 1u, status, 7) && mbar_wait_warp(p_full, (uint32_t)(j - 1) & 1u, status, 7))) return;
            if (scoring) {
                if (quarter == 0 && lane < 16) factor[(j & 1) * 32 + half * 16 + lane] = scale;
                uint8_t* p = gen + (p_at - base) + token * 128;
                *reinterpret_cast<uint4*>(p + ((half ^ (token & 7)) << 4)) = make_uint4(dh[0], dh[1], dh[2], dh[3]);
                *reinterpret_cast<uint4*>(p + ((HP / 16 + half) ^ (token & 7)) * 16) = make_uint4(dl[0], dl[1], dl[2], dl[3]);
            }
            if (token == 0 && half == 0) weight[j & 1] = big / STEPS;
            fence_async_smem();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        };
        // Called behind softmax(j + 1), which has waited for p_full of tile j (by now that barrier may be a phase further), or for the part's last tile.
        auto gather = [&](int j, bool last_of_part) {
            if (!(ok = mbar_wait_warp(o_full, (uint32_t)j & 1u, status, 8))) return;
            // factors and weights come from both halves' threads, which have all arrived at this barrier
            if (last_of_part && !(ok = mbar_wait_warp(p_full, (uint32_t)j & 1u, status, 8))) return;
            tcgen05_fence_after();
            const float by = weight[j & 1];
            const float* f = factor + (j & 1) * 32;
            const rowio::f32x2 magic = rowio::pair(-MAGIC, -MAGIC), hi_by = rowio::pair(256.0f * by, 256.0f * by), lo_by = rowio::pair(by, by);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if ((2 * half + c) * 128 >= R) break;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    if (hh * 16 >= HP) break;
                    uint32_t hi[16], lo[16];
                    const uint32_t at = O + (2 * half + c) * 64 + lanes + hh * 16;
                    tmem_ld16(at, hi);
                    tmem_ld16(at + HP, lo);
                    tmem_ld_wait();
                    // sums of a tile's digits are below 2^22: adding them to the bits of 1.5 * 2^23 makes floats of them
#pragma unroll
                    for (int h = 0; h < 16; h += 2) {
                        const rowio::f32x2 x = rowio::add2(rowio::pair(__int_as_float((int)hi[h] + __float_as_int(MAGIC)), __int_as_float((int)hi[h + 1] + __float_as_int(MAGIC))), magic);
                        const rowio::f32x2 y = rowio::add2(rowio::pair(__int_as_float((int)lo[h] + __float_as_int(MAGIC)), __int_as_float((int)lo[h + 1] + __float_as_int(MAGIC))), magic);
                        const float2 fs = *reinterpret_cast<const float2*>(f + hh * 16 + h);
                        rowio::f32x2 o = rowio::fma2(x, hi_by, rowio::mul2(rowio::pair(acc[c][hh * 16 + h], acc[c][hh * 16 + h + 1]), rowio::pair(fs.x, fs.y)));
                        o = rowio::fma2(y, lo_by, o);
                        acc[c][hh * 16 + h] = rowio::lo_of(o);
                        acc[c][hh * 16 + h + 1] = rowio::hi_of(o);
                    }
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
        };

        for (Walk k(a, first, last); k.more() && ok; k.next(), ++part) {
            top = -INFINITY;
#pragma unroll
            for (int h = 0; h < 16; ++h) sum[h] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int h = 0; h < 32; ++h) acc[c][h] = 0.0f;
            const int count = k.tiles();
            for (int i = 0; i < count && ok; ++i, ++g) {
                softmax(g);
                if (ok && i > 0) gather(g - 1, false);
            }
            if (!ok) break;
            gather(g - 1, true);
            if (!ok) break;
            // ---- the part's result ----
            const long long slot = (long long)w + k.b;
            if (scoring) {
                const float s = reduce16(sum);
                if (lane < 16) wsum[(half * 4 + quarter) * 16 + lane] = s;
            }
            if (!meet()) break;
            if (scoring && token < 16 && h0 + half * 16 + token < a.heads) {
                const float* ws = wsum + half * 64 + token;
                float* st = parts.stats(slot) + 2 * (h0 + half * 16 + token);
                st[0] = top;
                st[1] = (ws[0] + ws[16]) + (ws[32] + ws[48]);
            }
            if (!meet()) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = (2 * half + c) * 128 + token;
                if (r >= R) continue;
                float* out = parts.vectors(slot) + (long long)h0 * R + r;
#pragma unroll
                for (int h = 0; h < 32; ++h)
                    if (h < HP && h0 + h < a.heads) out[(long long)h * R] = acc[c][h];
            }
        }
    }
    if (status != nullptr && *reinterpret_cast<volatile int32_t*>(status) != 0) {
        // a wait gave up somewhere: copies and products still in flight get time to land before their memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) { }
    }
    // No block ends before the kernel in front has, also one that had no use for the query: what is launched behind the join waits for the join, and by that for
    // both, and may then be given their workspace.
    if (warp == WARP_LOAD) griddep_wait();
    tcgen05_fence_before();
    __syncthreads();
    if (warp == WARP_MMA) {
        tcgen05_fence_after();
        tmem_free<512>(tmem);
    }
}

// Parts begin at multiples of STEP_TILE, so boxes of up to that many tokens do not cross pages that they divide.
int box_of(const el_latent_step_t& a) {
    int g = STEP_TILE;
    while (g > 1 && a.page_size % g) g /= 2;
    // (a tensor map's rows are counted in 31 bits)
    return g >= 8 && a.pages > 0 && (long long)a.pages * a.page_size < (1LL << 31) ? g : 0;
}
int shared_bytes(const el_latent_step_t& a, const StepImage& image) { return 1024 + 2 * (image.chunks + (a.rot_dim ? 1 : 0)) * CHUNK + image.bytes() + CHUNK + 4256 + 112; }

}  // namespace

bool latent_step_tc_takes(const el_latent_step_t& a) {
    return a.dtype != EL_F32 && a.rot_dim % 8 == 0 && reinterpret_cast<uintptr_t>(a.cache_keys) % 16 == 0 && (long long)a.batch * a.heads < (1 << 24);
}

int launch_latent_step_tc(const el_latent_step_t& a, const uint8_t* images, const float* steps, const StepParts& parts, int workers, cudaStream_t st) {
    const StepImage image(a);
    const int box = box_of(a);
    int box_bits = 0;
    while (box > 1 << box_bits) ++box_bits;
    CUtensorMap rows = {}, keys = {};
    if (box) {
        const uint64_t tokens = (uint64_t)a.pages * a.page_size;
        int rc = make_map(&rows, a.latents, a.rank, tokens, a.rank, 128, box, 128);
        if (rc == EL_OK && a.rot_dim) rc = make_map(&keys, a.cache_keys, a.rot_dim * 2, tokens, a.rot_dim * 2, 128, box, 128);
        if (rc != EL_OK) return rc;
    }
    auto run = [&](auto t) {
        using T = decltype(t);
        static DeviceOnce once;
        int dev = 0;
        EL_CUDA_TRY(cudaGetDevice(&dev));
        if (!once.is_done(dev)) {
            EL_CUDA_TRY(cudaFuncSetAttribute(step_tc_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
            once.mark(dev);
        }
        cudaLaunchConfig_t cfg = {};
        // may begin while the query's kernel still runs, and load; the query is read behind griddepcontrol.wait
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3(workers * image.groups);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = shared_bytes(a, image);
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        EL_CUDA_TRY(cudaLaunchKernelEx(&cfg, step_tc_kernel<T>, rows, keys, a, images, steps, parts, workers, box_bits));
        return check_launch();
    };
    return a.dtype == EL_F16 ? run(__half()) : run(__nv_bfloat16());
}

}  // namespace el
