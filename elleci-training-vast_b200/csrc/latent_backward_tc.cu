// The backward pass of latent attention's expanded form on the tensor cores (latent_attention.cu has the formulas, latent_attention_tc.cu the sizes).
//
// Two kernels of one shape: a block holds 128 rows of one side of one head and walks over tiles of 64 rows of the other side.
//   KEYS   rows are keys:    S' = K Q',  dP' = V dO',  dV += P' dO,  dK += dS' Q
//   else   rows are queries: S  = Q K',  dP  = dO V',                dQ += dS K
// with A1, A2 the held matrices (K, V or Q, dO) and B1, B2 the others: S = A1 B1', dP = A2 B2', acc2 += P B2, acc1 += dS B1.  Every sum is formed by one
// block in a fixed order, so no gradient depends on the order of blocks; that is worth forming S and dP twice (5 + 3 products instead of 5).
//
// Warps 0-7: a thread owns a row and half of a tile's columns; it forms p = 2^(s - lse) and ds = p (dp - delta) and writes them to tensor memory as 16-bit
// left factors.  The softmax scale is applied to the sums, so that ds, rounded, is not smaller than it has to be.  Warp 8 issues the products, 9 the loads;
// warps 12-15 write dk or dq while the others are at the next item, whose sums wait until the accumulator has been read.  As many blocks as SMs, which
// take every so many-th item (128 rows of one head), the longest first.
//
// Tensor memory.  KEYS: acc1 192 columns, acc2 128, two S of 64, dP; p and ds go over S and dP, and the next S is formed while the threads work on a tile.
// Queries: there is one sum fewer, so Q and dO are copied into tensor memory (96 + 64 columns): a product of 128 x 64 x 16 then reads 2 KB of shared memory
// instead of 6, which is what bounds it.  The next S and dP follow as soon as the threads have read the last ones; ds has a place of its own.
//
// 4 x 1024 tokens, 32 heads of 128 + 64 and 128 channels, causal: 113 us for dk and dv, 91 us for dq (95 with all operands in shared memory and the
// threads' own stores).  A tile takes 2100 and 1570 cycles, of which the tensor core's rate explains 1280 and 1024; an item's end costs 6000 and 4000, at
// dk's and dv's at the rate at which all SMs write at once.  The clock falls to 1.66 GHz under these kernels.
#include "latent_tc.cuh"

namespace el {

using namespace tc;
using namespace latent;

int attention_maps(const el_attention_t& a, CUtensorMap m[5], int query_rows, int key_rows);

namespace {

constexpr int HELD = 128, STEP = 64;
constexpr int HELD_CHUNK = HELD * 128, STEP_CHUNK = STEP * 128;      // bytes of 64 columns
constexpr int WARP_MMA = 8, WARP_TMA = 9, WARP_OUT = 12, THREADS = 512;
constexpr int MAX_STAGES = 4, BARRIERS = 19;
constexpr int REGS_FACTORS = 168, REGS_OTHER = 88;         // 256 threads of each: 512 of 128

// Columns begin, begin + step .. of `width` accumulator columns, 32 at a time, as 16-bit values times `scale`, for the four rows from `to` on of which `rows`
// are there: four lanes share the stores of their four rows.  `there`: the thread's row has sums (else zeros); `formed`: the accumulator has.
template <typename T>
__device__ __forceinline__ void put_values(uint32_t acc, int begin, int step, int width, float scale, bool formed, bool there, T* to, long long pitch, int rows) {
    const int piece = threadIdx.x & 3;
#pragma unroll 1
    for (int c = begin; c < width; c += step) {
        uint32_t o[16], w[16];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (formed) {
                tmem_ld16(acc + c + 16 * x, o);
                tmem_ld_wait();
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) w[8 * x + k] = there ? pack_word<T>(__uint_as_float(o[2 * k]) * scale, __uint_as_float(o[2 * k + 1]) * scale) : 0u;
        }
        transpose_rows(w);
        if (to && c + piece * 8 < width) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < rows) *reinterpret_cast<uint4*>(to + k * pitch + c + piece * 8) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
        __syncwarp();
    }
}
// the same 16 columns at a time as floats
__device__ __forceinline__ void put_floats(uint32_t acc, int begin, int step, int width, float scale, bool formed, bool there, float* to, long long pitch, int rows) {
    const int piece = threadIdx.x & 3;
#pragma unroll 1
    for (int c = begin; c < width; c += step) {
        uint32_t w[16];
        if (formed) {
            tmem_ld16(acc + c, w);
            tmem_ld_wait();
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) w[k] = there ? __float_as_uint(__uint_as_float(w[k]) * scale) : 0u;
        transpose_rows(w);
        if (to) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < rows) *reinterpret_cast<uint4*>(to + k * pitch + c + piece * 4) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        }
        __syncwarp();
    }
}

struct Plan {
    int key_chunks, rot_chunks, value_chunks, stages;
};

template <typename T, bool KEYS>
__global__ void __launch_bounds__(THREADS, 1)
attention_backward_tc_kernel(const __grid_constant__ CUtensorMap tmA1, const __grid_constant__ CUtensorMap tmA1r, const __grid_constant__ CUtensorMap tmA2,
                             const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmB1r, const __grid_constant__ CUtensorMap tmB2,
                             const el_attention_t a, const float* __restrict__ delta, float* __restrict__ rot_parts, const Plan plan) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const int QC = plan.key_chunks + plan.rot_chunks, VC = plan.value_chunks, NS = plan.stages;
    const int held_bytes = (QC + VC) * HELD_CHUNK, stage_bytes = (QC + VC) * STEP_CHUNK;
    const uint32_t ring = base + held_bytes, stats = ring + NS * stage_bytes, bars = stats + NS * 2 * STEP * 4;
    uint8_t* ring_gen = gen + held_bytes;
    const float* stats_gen = reinterpret_cast<const float*>(ring_gen + NS * stage_bytes);
    const uint32_t a_full = bars, a_empty = bars + 8, landed = bars + 16, done = bars + 24;
    auto s_full = [&](int i) { return bars + 8u * (4 + i); };
    auto dp_full = [&](int i) { return bars + 8u * (6 + i); };
    auto p_full = [&](int i) { return bars + 8u * (8 + i); };
    auto ds_full = [&](int i) { return bars + 8u * (10 + i); };
    const uint32_t a2_full = bars + 136, a2_empty = bars + 144, acc_free = bars + 128, a_ready = bars + 96, s_read = bars + 104, dp_read = bars + 112, ds_read = bars + 120;
    auto full = [&](int s) { return bars + 8u * (BARRIERS + s); };
    auto empty = [&](int s) { return bars + 8u * (BARRIERS + MAX_STAGES + s); };
    volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(ring_gen + NS * (stage_bytes + 2 * STEP * 4) + 8 * (BARRIERS + 2 * MAX_STAGES));

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int all = KEYS ? a.keys : a.length, other = KEYS ? a.length : a.keys, tiles = (all + HELD - 1) / HELD;
    const unsigned items = (unsigned)tiles * a.batch * a.heads;
    int32_t* status = a.dev_status;
    // an item: its rows, and the tiles of the other side that they meet
    struct Item {
        int b, h, r0, live, other_live, begin, n;
        Sequence seq;
        __device__ __forceinline__ Item(const el_attention_t& a, unsigned item, int tiles) : Item(a, Place(a, item), tiles) {}
        __device__ __forceinline__ Item(const el_attention_t& a, const Place& at, int tiles) : b(at.batch), h(at.head), r0((KEYS ? at.tile : tiles - 1 - at.tile) * HELD), seq(a, at.batch) {
            live = KEYS ? seq.keys : seq.queries;
            other_live = KEYS ? seq.queries : seq.keys;
            int first = 0, end = 0;
            if (r0 < live) {
                first = KEYS ? seq.query_begin(r0) / STEP * STEP : 0;
                end = KEYS ? seq.queries : seq.key_end(r0 + HELD);
            }
            begin = uniform(first);
            n = uniform(end > first ? (end - first + STEP - 1) / STEP : 0);
        }
        __device__ __forceinline__ long long stat_row(const el_attention_t& a) const { return ((long long)b * a.heads + h) * lse_pitch(a.length); }
    };

    if (warp == WARP_TMA && elect_one()) {
        prefetch_map(&tmA1);
        prefetch_map(&tmA2);
        prefetch_map(&tmB1);
        prefetch_map(&tmB2);
        if (plan.rot_chunks) {
            prefetch_map(&tmA1r);
            prefetch_map(&tmB1r);
        }
        mbar_init(a_full, 1);
        mbar_init(a_empty, KEYS ? 1 : 8);
        mbar_init(a_ready, 8);
        mbar_init(s_read, 8);
        mbar_init(dp_read, 8);
        mbar_init(ds_read, 1);
        mbar_init(a2_full, 1);
        mbar_init(a2_empty, 1);
        mbar_init(acc_free, 4);
        mbar_init(landed, 1);
        mbar_init(done, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(dp_full(i), 1);
            mbar_init(p_full(i), 8);
            mbar_init(ds_full(i), 8);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == WARP_MMA) tmem_alloc<512>(smem_u32((const void*)tmem_holder));
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = uniform(*tmem_holder);
    // KEYS: acc1 192 columns, acc2 128, S_i at 64 i, dP.  Else acc1, A1 96, A2 64, S, dP, dS 32.
    const uint32_t ACC1 = tmem, ACC2 = tmem + 192, A1 = tmem + 192, A2 = A1 + 96, S = KEYS ? tmem + 320 : A2 + 64, DP = KEYS ? S + 128 : S + 64, DS = KEYS ? DP : DP + 64;

    if (warp >= WARP_MMA) fewer_registers<REGS_OTHER>();
    if (warp == WARP_TMA) {
        // ================= loads =================
        int s = 0;
        uint32_t ph = 0, land = 0, a_phase = 1;
        bool ok = true;
        each_item(items, [&](unsigned item) {
            const Item it(a, item, tiles);
            if (it.n == 0) return true;
            const int b = it.b, h = it.h;
            const int qh = (int)(h * a.q_stride_h), qrh = (int)(h * a.q_rot_stride_h), kh = (int)(h * a.k_stride_h), vh = (int)(h * a.v_stride_h), gh = (int)(h * a.dout_stride_h);
            const int x1 = KEYS ? kh : qh, x1r = KEYS ? 0 : qrh, x2 = KEYS ? vh : gh, y1 = KEYS ? qh : kh, y1r = KEYS ? qrh : 0, y2 = KEYS ? gh : vh;
            if (!(ok = mbar_wait_warp(a_empty, a_phase, status, 1))) return false;
            if (elect_one()) {
                mbar_expect_tx(a_full, KEYS ? QC * HELD_CHUNK : held_bytes);
                for (int c = 0; c < plan.key_chunks; ++c) tma_load_3d(base + c * HELD_CHUNK, &tmA1, a_full, x1 + c * CHUNK_COLS, it.r0, b);
                if (plan.rot_chunks) tma_load_3d(base + plan.key_chunks * HELD_CHUNK, &tmA1r, a_full, x1r, it.r0, b);
                if (!KEYS)
                    for (int c = 0; c < VC; ++c) tma_load_3d(base + (QC + c) * HELD_CHUNK, &tmA2, a_full, x2 + c * CHUNK_COLS, it.r0, b);
            }
            __syncwarp();
            if (KEYS) {                                              // the item before has left A2 a tile later than A1
                if (!(ok = mbar_wait_warp(a2_empty, a_phase, status, 1))) return false;
                if (elect_one()) {
                    mbar_expect_tx(a2_full, VC * HELD_CHUNK);
                    for (int c = 0; c < VC; ++c) tma_load_3d(base + (QC + c) * HELD_CHUNK, &tmA2, a2_full, x2 + c * CHUNK_COLS, it.r0, b);
                }
                __syncwarp();
            }
            a_phase ^= 1u;
            for (int j = 0; j < it.n; ++j) {
                if (!(ok = mbar_wait_warp(empty(s), ph ^ 1u, status, 1))) return false;
                const int c0 = it.begin + j * STEP, rows = it.other_live - c0;
                // rows behind the sequence's end may be anything, and zero times anything is not always zero: they are cleared
                const bool late = rows < STEP && c0 + rows < other;
                const uint32_t dst = ring + s * stage_bytes, bar = late ? landed : full(s);
                if (elect_one()) {
                    mbar_expect_tx(bar, stage_bytes + (KEYS ? 2 * STEP * 4 : 0));
                    for (int c = 0; c < plan.key_chunks; ++c) tma_load_3d(dst + c * STEP_CHUNK, &tmB1, bar, y1 + c * CHUNK_COLS, c0, b);
                    if (plan.rot_chunks) tma_load_3d(dst + plan.key_chunks * STEP_CHUNK, &tmB1r, bar, y1r, c0, b);
                    for (int c = 0; c < VC; ++c) tma_load_3d(dst + (QC + c) * STEP_CHUNK, &tmB2, bar, y2 + c * CHUNK_COLS, c0, b);
                    if (KEYS) {
                        bulk_load(stats + s * 2 * STEP * 4, a.lse + it.stat_row(a) + c0, STEP * 4, bar);
                        bulk_load(stats + s * 2 * STEP * 4 + STEP * 4, delta + it.stat_row(a) + c0, STEP * 4, bar);
                    }
                }
                __syncwarp();
                if (late) {
                    if (!(ok = mbar_wait_warp(landed, land, status, 2))) return false;
                    land ^= 1u;
                    for (int c = 0; c < QC + VC; ++c) {
                        uint4* chunk = reinterpret_cast<uint4*>(ring_gen + s * stage_bytes + c * STEP_CHUNK);
                        for (int k = rows * 8 + lane; k < STEP * 8; k += 32) chunk[k] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (elect_one()) mbar_arrive(full(s));
                    __syncwarp();
                }
                if (++s == NS) { s = 0; ph ^= 1u; }
            }
            return true;
        });
    } else if (warp == WARP_MMA) {
        // ================= products =================
        const int key_steps = a.key_dim / 16, rot_steps = a.rot_dim / 16, value_steps = a.value_dim / 16, D = a.key_dim, R = a.rot_dim, V = a.value_dim;
        const uint32_t i_s = idesc_f16<T>(0, 0, STEP), i_v = idesc_f16<T>(0, 1, V);
        const bool joined = R == 0 || D % 64 == 0;               // acc1's columns are the chunks' columns, one after another
        const uint32_t i_1 = idesc_f16<T>(0, 1, joined ? D + R : D), i_r = idesc_f16<T>(0, 1, R);
        uint32_t t = 0;                                          // tiles so far: the parities of S, dP and their barriers go by it
        // a product of held chunks and a tile's at `rows`: in shared memory both, or the held ones in tensor memory; one thread, as the others
        auto product = [&](uint32_t to, uint32_t held, uint32_t rows, int chunks, auto steps) {
            uint32_t x = KEYS ? desc_low(held, 16) : held, y = desc_low(rows, 16);
#pragma unroll 1
            for (int c = 0; c < chunks; ++c) {
                if (KEYS) umma_f16_chunk(to, x, y, i_s, c != 0, steps(c));
                else umma_f16_ts_chunk(to, x, y, i_s, c != 0, steps(c));
                x += KEYS ? HELD_CHUNK >> 4 : 32;
                y += STEP_CHUNK >> 4;
            }
        };
        auto scores = [&](uint32_t t, uint32_t rows) {
            const uint32_t buf = KEYS ? t & 1 : 0;
            product(S + buf * 64, KEYS ? base : A1, rows, QC, [&](int c) { return c < plan.key_chunks ? min(4, key_steps - 4 * c) : rot_steps; });
            umma_commit(s_full(buf));
        };
        auto grads = [&](uint32_t rows) {
            product(DP, KEYS ? base + QC * HELD_CHUNK : A2, rows + QC * STEP_CHUNK, VC, [&](int c) { return min(4, value_steps - 4 * c); });
            umma_commit(dp_full(0));
        };
        // acc += left factors at `f` times 64 rows of chunks at `rows`; over S or dP each half of the threads writes over its own columns
        auto sums = [&](uint32_t acc, uint32_t f, uint32_t rows, uint32_t idesc, bool more) {
            const uint32_t y = desc_low(rows, STEP_CHUNK), second = KEYS ? 32 : 16;
            umma_f16_ts(acc, f, desc_of(y), idesc, more);
            umma_f16_ts(acc, f + 8, desc_of(y + 128), idesc, 1u);
            umma_f16_ts(acc, f + second, desc_of(y + 256), idesc, 1u);
            umma_f16_ts(acc, f + second + 8, desc_of(y + 384), idesc, 1u);
        };
        bool ok = true;
        int next = 0;                                            // the stage of the next tile
        uint32_t next_phase = 0, a_phase = 0, acc_phase = 1;
        auto advance = [&]() {
            if (++next == NS) {
                next = 0;
                next_phase ^= 1u;
            }
        };
        each_item(items, [&](unsigned item) {
            const Item it(a, item, tiles);
            const int n = it.n;
            if (n == 0) return true;
            ok = mbar_wait_warp(KEYS ? a_full : a_ready, a_phase, status, 3) && mbar_wait_warp(full(next), next_phase, status, 3);
            tcgen05_fence_after();
            if (!ok) return false;
            int slot = next;
            if (elect_one()) {
                scores(t, ring + slot * stage_bytes);
                if (KEYS && n == 1) umma_commit(a_empty);
            }
            __syncwarp();
            if (KEYS) {
                ok = mbar_wait_warp(a2_full, a_phase, status, 3);
                tcgen05_fence_after();
                if (!ok) return false;
            }
            a_phase ^= 1u;
            if (elect_one()) {
                grads(ring + slot * stage_bytes);
                if (KEYS && n == 1) umma_commit(a2_empty);
            }
            __syncwarp();
            advance();
            for (int j = 0; j < n; ++j, ++t) {
                const uint32_t rows = ring + slot * stage_bytes, next_rows = ring + next * stage_bytes;
                if (j + 1 < n) {
                    ok = mbar_wait_warp(full(next), next_phase, status, 4) && (KEYS || mbar_wait_warp(s_read, t & 1u, status, 4));
                    tcgen05_fence_after();
                    if (!ok) return false;
                    if (elect_one()) {
                        scores(t + 1, next_rows);
                        if (KEYS && j + 2 == n) umma_commit(a_empty);
                    }
                    __syncwarp();
                    if (!KEYS) {
                        ok = mbar_wait_warp(dp_read, t & 1u, status, 5);
                        tcgen05_fence_after();
                        if (!ok) return false;
                        if (elect_one()) grads(next_rows);
                        __syncwarp();
                    }
                }
                if (KEYS) {
                    ok = mbar_wait_warp(p_full(t & 1), (t >> 1) & 1u, status, 5);
                    tcgen05_fence_after();
                    if (!ok) return false;
                    if (elect_one()) sums(ACC2, S + (t & 1) * 64, rows + QC * STEP_CHUNK, i_v, j != 0);
                    __syncwarp();
                }
                ok = mbar_wait_warp(ds_full(t & 1), (t >> 1) & 1u, status, 6) && (j > 0 || mbar_wait_warp(acc_free, acc_phase, status, 6));
                tcgen05_fence_after();
                if (!ok) return false;
                if (elect_one()) {
                    sums(ACC1, DS, rows, i_1, j != 0);
                    if (!joined) sums(ACC1 + D, DS, rows + plan.key_chunks * STEP_CHUNK, i_r, j != 0);
                    umma_commit(empty(slot));
                    if (KEYS) {
                        if (j + 1 < n) grads(next_rows);
                        if (j + 2 == n) umma_commit(a2_empty);
                    } else {
                        umma_commit(ds_read);
                    }
                    if (j + 1 == n) umma_commit(done);
                }
                __syncwarp();
                slot = next;
                if (j + 1 < n) advance();
            }
            acc_phase ^= 1u;
            return true;
        });
    } else if (warp < WARP_MMA) {
        // ================= probabilities and their gradients =================
        more_registers<REGS_FACTORS>();
        const int half = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, cols = half * 32;
        const float by = a.scale * mamba::LOG2E;
        const rowio::f32x2 by2 = rowio::pair(by, by);
        bool ok = true;
        int slot = 0;
        uint32_t phase = 0, t = 0, a_phase = 0, done_phase = 0;
        each_item(items, [&](unsigned item) {
            const Item it(a, item, tiles);
            const int n = it.n, row = it.r0 + quarter * 32 + lane;
            float lse = INFINITY, del = 0.0f;
            if (!KEYS && row < it.seq.queries) {
                lse = a.lse[it.stat_row(a) + row];
                del = delta[it.stat_row(a) + row];
            }
            // columns (of all) that the row meets: first .. last - 1
            long long first = 0, last = 0;
            if (row < it.live) {
                first = KEYS ? it.seq.query_begin(row) : 0;
                last = KEYS ? it.seq.queries : row + it.seq.shift + 1;
                if (!KEYS && last > it.seq.keys) last = it.seq.keys;
            }
            if (!KEYS && n > 0) {                                    // the held matrices go to tensor memory, half of the threads every other chunk
                if (!(ok = mbar_wait_warp(a_full, a_phase, status, 7))) return false;
                a_phase ^= 1u;
#pragma unroll 1
                for (int c = half; c < QC + VC; c += 2) {
                    const uint8_t* from = gen + c * HELD_CHUNK + (quarter * 32 + lane) * 128;
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint4 v = *reinterpret_cast<const uint4*>(from + ((k ^ (lane & 7)) << 4));
                        w[4 * k] = v.x;
                        w[4 * k + 1] = v.y;
                        w[4 * k + 2] = v.z;
                        w[4 * k + 3] = v.w;
                    }
                    tmem_st32((c < QC ? A1 + c * 32 : A2 + (c - QC) * 32) + lanes, w);
                }
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(a_ready);
                    mbar_arrive(a_empty);
                }
            }
            for (int j = 0; j < n; ++j, ++t) {
                const int c0 = it.begin + j * STEP + cols, buf = KEYS ? t & 1 : 0;
                const uint32_t sph = KEYS ? (t >> 1) & 1u : t & 1u;
                const float* st = stats_gen + slot * 2 * STEP + cols;
                if (!(ok = mbar_wait_warp(s_full(buf), sph, status, 7))) break;
                tcgen05_fence_after();
                uint32_t s[32], w[16];
                tmem_ld32(S + buf * 64 + lanes + cols, s);
                tmem_ld_wait();
                if (!KEYS) {
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_read);
                }
                // what a bulk copy brought is visible to who has waited for it: a phase that the product's issuer has already seen
                if (KEYS && !(ok = mbar_wait_warp(full(slot), phase, status, 8))) break;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 l = make_float4(lse, lse, lse, lse);
                    if (KEYS) l = *reinterpret_cast<const float4*>(st + k);
                    const rowio::f32x2 x = rowio::fma2(rowio::pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), by2, rowio::pair(-l.x, -l.y));
                    const rowio::f32x2 y = rowio::fma2(rowio::pair(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])), by2, rowio::pair(-l.z, -l.w));
                    s[k] = __float_as_uint(mamba::ex2(rowio::lo_of(x)));
                    s[k + 1] = __float_as_uint(mamba::ex2(rowio::hi_of(x)));
                    s[k + 2] = __float_as_uint(mamba::ex2(rowio::lo_of(y)));
                    s[k + 3] = __float_as_uint(mamba::ex2(rowio::hi_of(y)));
                }
                const int lo = (int)(first - c0 < 0 ? 0 : first - c0 > 32 ? 32 : first - c0), hi = (int)(last - c0 < 0 ? 0 : last - c0 > 32 ? 32 : last - c0);
                const bool partial = __any_sync(0xffffffffu, lo > 0 || hi < 32);
                if (partial) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) s[k] = k >= lo && k < hi ? s[k] : 0u;
                }
                if (KEYS) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) w[k] = pack_word<T>(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
                    tmem_st16(S + buf * 64 + lanes + cols, w);
                    tmem_st_wait();
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(buf));
                }
                if (!(ok = mbar_wait_warp(dp_full(0), t & 1u, status, 9))) break;
                tcgen05_fence_after();
                uint32_t g[32];
                tmem_ld32(DP + lanes + cols, g);
                tmem_ld_wait();
                if (!KEYS) {
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(dp_read);
                }
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 d = make_float4(del, del, del, del);
                    if (KEYS) d = *reinterpret_cast<const float4*>(st + STEP + k);
                    const rowio::f32x2 x = rowio::mul2(rowio::pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])),
                                                       rowio::add2(rowio::pair(__uint_as_float(g[k]), __uint_as_float(g[k + 1])), rowio::pair(-d.x, -d.y)));
                    const rowio::f32x2 y = rowio::mul2(rowio::pair(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])),
                                                       rowio::add2(rowio::pair(__uint_as_float(g[k + 2]), __uint_as_float(g[k + 3])), rowio::pair(-d.z, -d.w)));
                    g[k] = __float_as_uint(rowio::lo_of(x));
                    g[k + 1] = __float_as_uint(rowio::hi_of(x));
                    g[k + 2] = __float_as_uint(rowio::lo_of(y));
                    g[k + 3] = __float_as_uint(rowio::hi_of(y));
                }
                if (partial) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) g[k] = k >= lo && k < hi ? g[k] : 0u;
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k] = pack_word<T>(__uint_as_float(g[2 * k]), __uint_as_float(g[2 * k + 1]));
                if (!KEYS && t > 0) {                                // the products of the tile before have read its factors
                    if (!(ok = mbar_wait_warp(ds_read, (t - 1) & 1u, status, 9))) break;
                    tcgen05_fence_after();
                }
                tmem_st16(KEYS ? DP + lanes + cols : DS + lanes + half * 16, w);
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full(t & 1));
                if (++slot == NS) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) return false;
            if (KEYS) {                                              // dv and the rotated part; the other warps write dk
                if (n > 0) {
                    if (!(ok = mbar_wait_warp(done, done_phase, status, 10))) return false;
                    done_phase ^= 1u;
                    tcgen05_fence_after();
                }
                const int first_row = row & ~3, rows = all - first_row;
                const bool there = n > 0 && row < it.live;
                put_values<T>(ACC2 + lanes, half * 32, 64, a.value_dim, 1.0f, n > 0, there,
                              a.dv ? static_cast<T*>(a.dv) + it.b * a.dv_stride_b + first_row * a.dv_stride_t + it.h * a.dv_stride_h : nullptr, a.dv_stride_t, rows);
                put_floats(ACC1 + a.key_dim + lanes, half * 16, 32, a.rot_dim, a.scale, n > 0, there,
                           rot_parts ? rot_parts + (((long long)it.b * a.heads + it.h) * a.keys + first_row) * a.rot_dim : nullptr, a.rot_dim, rows);
                tcgen05_fence_before();                              // the sums have been read: the next item's wait for these warps' factors
            }
            return true;
        });
    } else if (warp >= WARP_OUT) {
        // ================= dk or dq: while the other warps are at the next item, whose sums wait for the accumulator =================
        const int quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        uint32_t done_phase = 0;
        each_item(items, [&](unsigned item) {
            const Item it(a, item, tiles);
            const int n = it.n, row = it.r0 + quarter * 32 + lane, first_row = row & ~3, rows = all - first_row;
            if (n > 0) {
                if (!mbar_wait_warp(done, done_phase, status, 10)) return false;
                done_phase ^= 1u;
                tcgen05_fence_after();
            }
            const bool there = n > 0 && row < it.live;
            if (KEYS) {
                put_values<T>(ACC1 + lanes, 0, 32, a.key_dim, a.scale, n > 0, there,
                              a.dk ? static_cast<T*>(a.dk) + it.b * a.dk_stride_b + first_row * a.dk_stride_t + it.h * a.dk_stride_h : nullptr, a.dk_stride_t, rows);
            } else {
                const long long at = ((long long)it.b * a.length + first_row) * a.heads + it.h;
                put_values<T>(ACC1 + lanes, 0, 32, a.key_dim, a.scale, n > 0, there, a.dq ? static_cast<T*>(a.dq) + at * a.key_dim : nullptr, (long long)a.heads * a.key_dim, rows);
                put_values<T>(ACC1 + a.key_dim + lanes, 0, 32, a.rot_dim, a.scale, n > 0, there, a.dq_rot ? static_cast<T*>(a.dq_rot) + at * a.rot_dim : nullptr,
                              (long long)a.heads * a.rot_dim, rows);
            }
            if (n > 0) {
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_free);
            }
            return true;
        });
    }
    if (status != nullptr && *reinterpret_cast<volatile int32_t*>(status) != 0) {
        // a wait gave up somewhere: copies and products still in flight get time to land before their memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) { }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == WARP_MMA) {
        tcgen05_fence_after();
        tmem_free<512>(tmem);
    }
}

Plan plan_of(const el_attention_t& a) {
    Plan p;
    p.key_chunks = (a.key_dim + 63) / 64;
    p.rot_chunks = (a.rot_dim + 63) / 64;
    p.value_chunks = (a.value_dim + 63) / 64;
    const int chunks = p.key_chunks + p.rot_chunks + p.value_chunks;
    const int room = (227 * 1024 - 2048 - chunks * HELD_CHUNK) / (chunks * STEP_CHUNK + 2 * STEP * 4);
    p.stages = room < MAX_STAGES ? room : MAX_STAGES;
    return p;
}
int shared_bytes(const Plan& p) {
    const int chunks = p.key_chunks + p.rot_chunks + p.value_chunks;
    return 1024 + chunks * HELD_CHUNK + p.stages * (chunks * STEP_CHUNK + 2 * STEP * 4) + 8 * (BARRIERS + 2 * MAX_STAGES) + 16;
}

template <typename T, bool KEYS>
int launch(const el_attention_t& a, const CUtensorMap* held, const CUtensorMap* step, const float* delta, float* rot_parts, cudaStream_t st) {
    static DeviceOnce once;
    int dev = 0;
    EL_CUDA_TRY(cudaGetDevice(&dev));
    if (!once.is_done(dev)) {
        EL_CUDA_TRY(cudaFuncSetAttribute(attention_backward_tc_kernel<T, KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        once.mark(dev);
    }
    const Plan plan = plan_of(a);
    int sms = 148;
    device_sm_count(&sms);
    const unsigned items = blocks_of(a, KEYS ? a.keys : a.length, HELD);
    attention_backward_tc_kernel<T, KEYS><<<items < (unsigned)sms ? items : sms, THREADS, shared_bytes(plan), st>>>(
        held[0], held[1], held[2], step[0], step[1], step[2], a, delta, rot_parts, plan);
    return check_launch();
}

}  // namespace

int launch_attention_backward_tc(const el_attention_t& a, const float* delta, float* rot_parts, cudaStream_t st) {
    CUtensorMap m[5], g;                                         // q, q_rot, k, k_rot, v and dout
    auto run = [&](auto t, auto keys) {
        using T = decltype(t);
        constexpr bool KEYS = decltype(keys)::value;
        const int query_rows = KEYS ? STEP : HELD, key_rows = KEYS ? HELD : STEP;
        int rc = attention_maps(a, m, query_rows, key_rows);
        if (rc == EL_OK) rc = make_map_tokens(&g, a.dout, (a.heads - 1) * a.dout_stride_h + a.value_dim, a.length, a.dout_stride_t, a.batch, a.dout_stride_b, query_rows);
        if (rc != EL_OK) return rc;
        const CUtensorMap by_key[3] = {m[2], m[3], m[4]}, by_query[3] = {m[0], m[1], g};
        return KEYS ? launch<T, true>(a, by_key, by_query, delta, rot_parts, st) : launch<T, false>(a, by_query, by_key, delta, rot_parts, st);
    };
    auto typed = [&](auto keys) { return a.dtype == EL_F16 ? run(__half(), keys) : run(__nv_bfloat16(), keys); };
    int rc = EL_OK;
    if (a.dk || a.dv || rot_parts) rc = typed(std::true_type());
    if (rc == EL_OK && (a.dq || a.dq_rot)) rc = typed(std::false_type());
    return rc;
}

}  // namespace el
