// The forward pass of latent attention's expanded form on the tensor cores (latent_attention.cu has the formulas): 16-bit types, head sizes that are
// multiples of 16 up to 128 (content), 64 (rotated) and 128 (value).
//
// A block takes 256 queries of one head as two tiles of 128 rows, which share the keys' tiles of 128: while the softmax of one tile runs, the
// tensor core works on the other.  Warps: 0-3 and 4-7 softmax of the two tiles (a thread owns a row), 8 issues the products, 9 the loads.
//   S_i = Q_i K'   accumulator of 128 columns in tensor memory; the thread reads its row, forms p = 2^(s - reference) and writes it back as 16-bit
//                  values over S_i, where it is the left factor of
//   O_i += P_i V   whose sums stay in tensor memory.  The reference of a row follows its maximum only when that has grown by more than 2^8:
//                  then the row of O_i is scaled.  P stays below 2^8, sums are float32.
// As many blocks as SMs, which take every so many-th item (a pair of tiles of one head), the longest first: while a block's threads write an item's output, its
// next item's queries and keys are on their way and their first products run.
// Order of products: P_0 V, S_0 of the next keys, P_1 V, S_1 of the next keys.  Keys and values go through one ring of 16 KB chunks in the order in
// which they are first used.
// Bound: one sequence of 8192 tokens, 32 heads of 128 + 64 and 128 channels, causal: 550 us, 1.25 PFLOP/s at the 1.63 GHz that the power leaves (64 % of the tensor
// pipe's cycles, then the exponentials).  4 x 1024 tokens: 73 us, 0.6 PFLOP/s: a first round of items that reads all heads' keys at once, and an item's end for every 5 tiles.
#include "latent_tc.cuh"

namespace el {

using namespace tc;
using namespace latent;

namespace {

constexpr int TILE = 128;                       // rows of a query tile, and keys of a tile
constexpr int CHUNK = TILE * 128;               // bytes of 64 columns of a tile
constexpr int MAX_SLOTS = 12;
constexpr int WARP_MMA = 8, WARP_TMA = 9, THREADS = 384;        // (warps 10 and 11 fill a group of four, for the split of registers)
constexpr int REGS_SOFTMAX = 216, REGS_OTHER = 64;              // 256 x 216 + 128 x 64 of the launch's 384 x 168
constexpr float GROWTH = 8.0f;                  // exponent of 2 by which a row's maximum may outgrow its reference

struct Plan {
    int key_chunks, rot_chunks, value_chunks;   // of 64 columns
    int slots;
    int splits;                                 // items that share a pair of tiles, each a part of its keys
};

// What an item leaves where the keys are split: for every row its reference and sum, and the sums with values, not yet divided.
struct Parts {
    float *sums, *stats;
    long long rows;                             // batch * heads * the padded length
    __device__ __forceinline__ float* sum_of(int split, long long row, int width) const { return sums + (split * rows + row) * width; }
    __device__ __forceinline__ float* stats_of(int split, long long row) const { return stats + (split * rows + row) * 2; }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 1)
attention_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQr, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmKr, const __grid_constant__ CUtensorMap tmV, const el_attention_t a, const Plan plan, const Parts parts) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const int QC = plan.key_chunks + plan.rot_chunks, VC = plan.value_chunks, NS = plan.slots;
    const uint32_t ring = base + 2 * QC * CHUNK;
    uint8_t* ring_gen = gen + 2 * QC * CHUNK;
    const uint32_t bars = ring + NS * CHUNK;
    auto q_full = [&](int i) { return bars + 8u * i; };
    auto s_full = [&](int i) { return bars + 8u * (2 + i); };
    auto p_full = [&](int i) { return bars + 8u * (4 + i); };
    auto o_full = [&](int i) { return bars + 8u * (6 + i); };
    const uint32_t landed = bars + 8u * 8;
    auto slot_full = [&](int s) { return bars + 8u * (9 + s); };          // of the chunks of one tile, at its first chunk's slot
    auto slot_empty = [&](int s) { return bars + 8u * (9 + MAX_SLOTS + s); };
    volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(ring_gen + NS * CHUNK + 8 * (11 + 2 * MAX_SLOTS));

    const uint32_t q_empty = slot_empty(MAX_SLOTS);             // two
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int pairs = (a.length + 2 * TILE - 1) / (2 * TILE);
    const unsigned items = (unsigned)pairs * a.batch * a.heads * plan.splits;
    int32_t* status = a.dev_status;
    // an item: its queries, its first key tile, and how many from there its two query tiles take
    struct Item {
        int b, h, i0, split, j0, n0, n1, n;
        Sequence seq;
        __device__ __forceinline__ Item(const el_attention_t& a, unsigned item, int pairs, int splits) : Item(a, Place(a, splits == 1 ? item : item / splits), pairs, splits, splits == 1 ? 0 : item % splits) {}
        __device__ __forceinline__ Item(const el_attention_t& a, const Place& at, int pairs, int splits, int part)
            : b(at.batch), h(at.head), i0((pairs - 1 - at.tile) * 2 * TILE), split(part), seq(a, at.batch) {
            n0 = i0 < seq.queries ? (seq.key_end(i0 + TILE) + TILE - 1) / TILE : 0;
            n1 = i0 + TILE < seq.queries ? (seq.key_end(i0 + 2 * TILE) + TILE - 1) / TILE : 0;
            j0 = 0;
            if (splits > 1) {
                const int all = n0 > n1 ? n0 : n1, j1 = (int)((long long)all * (part + 1) / splits);
                j0 = (int)((long long)all * part / splits);
                n0 = max(min(n0, j1) - j0, 0);
                n1 = max(min(n1, j1) - j0, 0);
            }
            j0 = uniform(j0);
            n0 = uniform(n0);
            n1 = uniform(n1);
            n = n0 > n1 ? n0 : n1;
        }
    };

    if (warp == WARP_TMA && elect_one()) {
        prefetch_map(&tmQ);
        prefetch_map(&tmK);
        prefetch_map(&tmV);
        if (plan.rot_chunks) {
            prefetch_map(&tmQr);
            prefetch_map(&tmKr);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full(i), 1);
            mbar_init(q_empty + 8u * i, 1);
            mbar_init(s_full(i), 1);
            mbar_init(p_full(i), 4);
            mbar_init(o_full(i), 1);
        }
        mbar_init(landed, 1);
        for (int s = 0; s < NS; ++s) {
            mbar_init(slot_full(s), 1);
            mbar_init(slot_empty(s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == WARP_MMA) tmem_alloc<512>(smem_u32((const void*)tmem_holder));
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = uniform(*tmem_holder);
    const uint32_t S = tmem, O = tmem + 256;                    // S_i at 128 i, O_i at 256 + 128 i

    if (warp >= WARP_MMA) fewer_registers<REGS_OTHER>();
    if (warp == WARP_TMA) {
        // ================= loads =================
        int s = 0;
        uint32_t ph = 0, land = 0, q_phase[2] = {1u, 1u};
        bool ok = true;
        each_item(items, [&](unsigned item) {
            const Item it(a, item, pairs, plan.splits);
            for (int i = 0; i < 2 && ok; ++i) {
                if ((i == 0 ? it.n0 : it.n1) == 0) continue;
                if (!mbar_wait_warp(q_empty + 8u * i, q_phase[i], status, 1)) { ok = false; break; }
                q_phase[i] ^= 1u;
                if (elect_one()) {
                    mbar_expect_tx(q_full(i), QC * CHUNK);
                    for (int c = 0; c < plan.key_chunks; ++c)
                        tma_load_3d(base + (i * QC + c) * CHUNK, &tmQ, q_full(i), (int)(it.h * a.q_stride_h) + c * CHUNK_COLS, it.i0 + i * TILE, it.b);
                    if (plan.rot_chunks) tma_load_3d(base + (i * QC + plan.key_chunks) * CHUNK, &tmQr, q_full(i), (int)(it.h * a.q_rot_stride_h), it.i0 + i * TILE, it.b);
                }
                __syncwarp();
            }
            for (int j = 0; j < it.n && ok; ++j) {
                // values behind the sequence's end may be anything, and zero times anything is not always zero: those rows are cleared
                const int key = (it.j0 + j) * TILE, live = it.seq.keys - key;
                const bool clear = live < TILE && key + live < a.keys;
                int head = 0;
                for (int c = 0; c < QC + VC; ++c) {
                    if (!mbar_wait_warp(slot_empty(s), ph ^ 1u, status, 1)) { ok = false; break; }
                    const bool value = c >= QC, late = value && clear;
                    if (c == 0 || c == QC) head = s;
                    if (elect_one()) {
                        const uint32_t dst = ring + s * CHUNK, bar = late ? landed : slot_full(head);
                        if (late) mbar_expect_tx(bar, CHUNK);
                        else if (s == head) mbar_expect_tx(bar, (value ? VC : QC) * CHUNK);
                        if (value) tma_load_3d(dst, &tmV, bar, (int)(it.h * a.v_stride_h) + (c - QC) * CHUNK_COLS, key, it.b);
                        else if (c < plan.key_chunks) tma_load_3d(dst, &tmK, bar, (int)(it.h * a.k_stride_h) + c * CHUNK_COLS, key, it.b);
                        else tma_load_3d(dst, &tmKr, bar, 0, key, it.b);
                    }
                    __syncwarp();
                    if (late) {
                        if (!mbar_wait_warp(landed, land, status, 2)) { ok = false; break; }
                        land ^= 1u;
                        uint4* rows = reinterpret_cast<uint4*>(ring_gen + s * CHUNK);
                        for (int k = live * 8 + lane; k < TILE * 8; k += 32) rows[k] = make_uint4(0u, 0u, 0u, 0u);
                        fence_async_smem();
                        __syncwarp();
                        if (c + 1 == QC + VC && elect_one()) mbar_arrive(slot_full(head));
                        __syncwarp();
                    }
                    if (++s == NS) { s = 0; ph ^= 1u; }
                }
            }
            return ok;
        });
    } else if (warp == WARP_MMA) {
        // ================= products =================
        const uint32_t i_s = idesc_f16<T>(0, 0, TILE);
        const int key_steps = a.key_dim / 16, rot_steps = a.rot_dim / 16, V = a.value_dim;
        bool ok = true;
        // A place in the ring, which chunks go through in order (counted, not divided: a division costs more than a product).
        auto after = [&](int slot, int count) { return slot + count >= NS ? slot + count - NS : slot + count; };
        uint32_t phases = 0;                                    // bit s: parity of slot s' next tile
        auto wait_tile = [&](int slot) {
            ok = ok && mbar_wait_warp(slot_full(slot), (phases >> slot) & 1u, status, 3);
            phases ^= 1u << slot;
            tcgen05_fence_after();
        };
        auto release = [&](int slot, int count) {
#pragma unroll 1
            for (int c = 0; c < count; ++c, slot = after(slot, 1)) umma_commit(slot_empty(slot));
        };
        auto scores = [&](int i, int first) {                   // S_i = Q_i K'; one thread
            uint32_t q = desc_low(base + i * QC * CHUNK, 16);
            int slot = first;
#pragma unroll 1
            for (int c = 0; c < QC; ++c) {
                umma_f16_chunk(S + i * 128, q, desc_low(ring + slot * CHUNK, 16), i_s, c != 0, c < plan.key_chunks ? min(4, key_steps - 4 * c) : rot_steps);
                q += CHUNK >> 4;
                slot = slot + 1 == NS ? 0 : slot + 1;
            }
            umma_commit(s_full(i));
        };
        auto values = [&](int i, int first, bool more) {        // O_i += P_i V; one thread
            const int s0 = first, parts = VC == 1 || s0 + 1 < NS ? 1 : 2;             // the chunks lie side by side, or the ring's end is between them
#pragma unroll 1
            for (int c = 0; c < parts; ++c) {
                const uint32_t id = idesc_f16<T>(0, 1, parts == 1 ? V : c == 0 ? 64 : V - 64), v = desc_low(ring + (c == 0 ? s0 : 0) * CHUNK, CHUNK);
                const uint32_t o = O + i * 128 + c * 64, p = S + i * 128;
                umma_f16_ts(o, p, desc_of(v), id, more);
#pragma unroll
                for (int x = 1; x < TILE / 16; ++x) umma_f16_ts(o, p + x * 8, desc_of(v + x * 128), id, 1u);
            }
            umma_commit(o_full(i));
        };
        int place = 0;                                          // of the next tile of keys or values
        uint32_t q_phase[2] = {0u, 0u}, p_phase[2] = {0u, 0u};
        each_item(items, [&](unsigned item) {
            const Item it(a, item, pairs, plan.splits);
            if (it.n == 0) return true;
            const int only = it.n0 == 0 ? 1 : 0;                // the tile that waits for what both need: the first that there is
            for (int i = 0; i < 2; ++i) {
                const int mine = i == 0 ? it.n0 : it.n1;
                if (mine == 0) continue;
                ok = ok && mbar_wait_warp(q_full(i), q_phase[i], status, 4);
                q_phase[i] ^= 1u;
                if (i == only) wait_tile(place);
                if (!ok) break;
                if (elect_one()) {
                    scores(i, place);
                    if (mine == 1) umma_commit(q_empty + 8u * i);
                    if (i == 1 || it.n1 == 0) release(place, QC);
                }
                __syncwarp();
            }
            int v = after(place, QC);
            for (int j = 0; j < it.n && ok; ++j) {
                const int k = after(v, VC);
                bool have_v = false, have_k = false;
                for (int i = 0; i < 2; ++i) {
                    const int mine = i == 0 ? it.n0 : it.n1;
                    if (j >= mine) continue;
                    const bool last = i == 1 || j >= it.n1;     // nothing else reads the values; nor the next keys, if the other tile has no more
                    const bool last_k = i == 1 || j + 1 >= it.n1;
                    if (!have_v) wait_tile(v);
                    have_v = true;
                    ok = ok && mbar_wait_warp(p_full(i), p_phase[i], status, 5);
                    p_phase[i] ^= 1u;
                    tcgen05_fence_after();
                    if (!ok) break;
                    if (elect_one()) {
                        values(i, v, j != 0);
                        if (last) release(v, VC);
                    }
                    __syncwarp();
                    if (j + 1 < mine) {
                        if (!have_k) wait_tile(k);
                        have_k = true;
                        if (!ok) break;
                        if (elect_one()) {
                            scores(i, k);
                            if (j + 2 == mine) umma_commit(q_empty + 8u * i);
                            if (last_k) release(k, QC);
                        }
                        __syncwarp();
                    }
                }
                place = k;
                v = after(k, QC);
            }
            return ok;
        });
    } else if (warp < WARP_MMA) {
        // ================= softmax =================
        more_registers<REGS_SOFTMAX>();
        const int i = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_addr = S + i * 128 + lanes, o_addr = O + i * 128 + lanes;
        const float by = a.scale * mamba::LOG2E;
        bool ok = true;
        uint32_t phase = 0;                                     // of this tile's s_full; o_full of the tile before has the other one
        each_item(items, [&](unsigned item) {
            const Item it(a, item, pairs, plan.splits);
            const int mine = i == 0 ? it.n0 : it.n1, row = it.i0 + i * TILE + quarter * 32 + lane;
            // keys that this row sees: 0 .. sees - 1
            long long sees = row < it.seq.queries ? row + it.seq.shift + 1 : 0;
            sees = sees < 0 ? 0 : sees > it.seq.keys ? it.seq.keys : sees;
            float ref = -INFINITY, sum = 0.0f;
            for (int j = 0; j < mine; ++j, phase ^= 1u) {
                if (!(ok = mbar_wait_warp(s_full(i), phase, status, 6))) break;
                tcgen05_fence_after();
                uint32_t v[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, v[c]);
                tmem_ld_wait();
                const int here = (int)sees - (it.j0 + j) * TILE;               // columns that the row sees
                if (__any_sync(0xffffffffu, here < TILE)) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[c][k] = c * 32 + k < here ? v[c][k] : 0xff800000u;
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(v[c][0]);
#pragma unroll
                    for (int k = 1; k < 32; ++k) top[c] = fmaxf(top[c], __uint_as_float(v[c][k]));
                }
                const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * by;
                const bool grown = m > ref + GROWTH;                 // also a row's first finite maximum
                if (__any_sync(0xffffffffu, grown)) {
                    const float to = grown ? m : ref, factor = grown && ref != -INFINITY ? exp2_neg(ref - m) : 1.0f;
                    if (j > 0) {
                        if (!(ok = mbar_wait_warp(o_full(i), phase ^ 1u, status, 7))) break;
                        tcgen05_fence_after();
                        for (int c = 0; c < a.value_dim; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                            tmem_st16(o_addr + c, o);
                        }
                        tmem_st_wait();
                    }
                    sum *= factor;
                    ref = to;
                }
                const float from = ref == -INFINITY ? 0.0f : -ref;
                const rowio::f32x2 by2 = rowio::pair(by, by), from2 = rowio::pair(from, from);
                rowio::f32x2 part[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) part[c] = rowio::pair(0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < 4; c += 2) {
                    uint32_t p[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const int e = 2 * k, cc = c + e / 32;
                        const rowio::f32x2 x = rowio::fma2(rowio::pair(__uint_as_float(v[cc][e % 32]), __uint_as_float(v[cc][e % 32 + 1])), by2, from2);
                        const float y0 = mamba::ex2(rowio::lo_of(x)), y1 = mamba::ex2(rowio::hi_of(x));
                        part[k & 3] = rowio::add2(part[k & 3], rowio::pair(y0, y1));
                        p[k] = pack_word<T>(y0, y1);
                    }
                    tmem_st32(s_addr + c * 16, p);
                }
                const rowio::f32x2 t = rowio::add2(rowio::add2(part[0], part[1]), rowio::add2(part[2], part[3]));
                sum += rowio::lo_of(t) + rowio::hi_of(t);
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(i));
            }
            const bool empty = ref == -INFINITY && !(sum != sum);    // sees nothing; a NaN is no such row
            const float inv = 1.0f / sum;
            const long long stat_row = ((long long)it.b * a.heads + it.h) * lse_pitch(a.length) + row;
            if (row < lse_pitch(a.length)) {
                if (plan.splits > 1) *reinterpret_cast<float2*>(parts.stats_of(it.split, stat_row)) = make_float2(sum != sum ? sum : ref, sum);
                else if (a.lse) a.lse[stat_row] = empty ? INFINITY : ref + log2f(sum);
            }
            if (ok && mine > 0) ok = mbar_wait_warp(o_full(i), phase ^ 1u, status, 8);
            if (!ok) return false;
            tcgen05_fence_after();
            // four lanes share the stores of their four rows
            const int first = row & ~3;
            if (plan.splits > 1) {                               // (without a tile there are no sums: such a part's are not read)
                float* to = parts.sum_of(it.split, stat_row - (lane & 3), a.value_dim) + (lane & 3) * 4;
                for (int c = 0; c < a.value_dim && mine > 0; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(o_addr + c, o);
                    tmem_ld_wait();
                    transpose_rows(o);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (first + k < lse_pitch(a.length)) *reinterpret_cast<uint4*>(to + (long long)k * a.value_dim + c) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                    __syncwarp();
                }
                tcgen05_fence_before();
                return true;
            }
            T* out = static_cast<T*>(a.out) + (((long long)it.b * a.length + first) * a.heads + it.h) * a.value_dim + (lane & 3) * 8;
            for (int c = 0; c < a.value_dim; c += 32) {
                uint32_t o[32], w[16];
                if (mine > 0) {
                    tmem_ld32(o_addr + c, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = mine == 0 || empty ? 0u : __float_as_uint(__uint_as_float(o[k]) * inv);
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k] = pack_word<T>(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1]));
                if (a.out_rest && row < a.length) {
                    uint4* rest = reinterpret_cast<uint4*>(a.out_rest + (((long long)it.b * a.length + row) * a.heads + it.h) * a.value_dim + c);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        auto four = [&](int x) { return rest_word<T>(w[2 * x], w[2 * x + 1], __uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]), __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3])); };
                        const uint4 r = make_uint4(four(4 * k), four(4 * k + 1), four(4 * k + 2), four(4 * k + 3));
                        if (c + 16 * k < a.value_dim) rest[k] = r;
                    }
                }
                transpose_rows(w);
                if (c + (lane & 3) * 8 < a.value_dim) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (first + k < a.length)
                            *reinterpret_cast<uint4*>(out + (long long)k * a.heads * a.value_dim + c) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                }
                __syncwarp();
            }
            tcgen05_fence_before();                             // the sums have been read: the next item's first product with values waits for these warps' factors
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

// out and lse from the parts of every row.  A warp takes a row; value_dim is a multiple of 16 up to 128, four values a lane.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const el_attention_t a, const Parts parts, int splits) {
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), pitch = lse_pitch(a.length);
    if (row >= parts.rows) return;
    const int lane = threadIdx.x & 31;
    const unsigned bh = (unsigned)(row / pitch), b = bh / a.heads, h = bh - b * a.heads;
    const int i = (int)(row - bh * pitch);
    float top = -INFINITY;
    for (int s = 0; s < splits; ++s) top = mamba::max_nan(top, parts.stats_of(s, row)[0]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    for (int s = 0; s < splits; ++s) {
        const float2 st = *reinterpret_cast<const float2*>(parts.stats_of(s, row));
        if (st.x == -INFINITY) continue;
        const float f = exp2_neg(st.x - top);
        sum = fmaf(f, st.y, sum);
        if (lane * 4 < a.value_dim) {
            const float4 v = *reinterpret_cast<const float4*>(parts.sum_of(s, row, a.value_dim) + lane * 4);
            o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
        }
    }
    const bool empty = top == -INFINITY;
    if (a.lse && lane == 0) a.lse[row] = empty ? INFINITY : top + log2f(sum);
    if (i >= a.length || lane * 4 >= a.value_dim) return;
    const float inv = empty ? 0.0f : 1.0f / sum;
    const long long at = (((long long)b * a.length + i) * a.heads + h) * a.value_dim + lane * 4;
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    const uint2 w = make_uint2(pack_word<T>(o.x, o.y), pack_word<T>(o.z, o.w));
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at) = w;
    if (a.out_rest) *reinterpret_cast<uint32_t*>(a.out_rest + at) = rest_word<T>(w.x, w.y, o.x, o.y, o.z, o.w);
}

// Items that share a pair of query tiles, where there are fewer pairs than SMs: what makes the rounds over the SMs times the tiles of an item least, an item's own
// start and end counted as two tiles and a part's way through memory as one more.  2 x 250 queries, 3999 keys, 32 heads (64 pairs): 1 item 81 us, 2 items 58.
int splits_of(const el_attention_t& a) {
    int sms = 148, best = 1;
    device_sm_count(&sms);
    const long long items = blocks_of(a, a.length, 2 * TILE), n = ((long long)a.keys + TILE - 1) / TILE;
    long long least = 0;
    for (int s = 1; s <= 16 && s <= n && (s == 1 || items < sms); ++s) {
        const long long cost = (items * s + sms - 1) / sms * ((n + s - 1) / s + 2 + (s > 1));
        if (s == 1 || cost < least) {
            least = cost;
            best = s;
        }
    }
    return best;
}

Plan plan_of(const el_attention_t& a) {
    Plan p;
    p.key_chunks = (a.key_dim + 63) / 64;
    p.rot_chunks = (a.rot_dim + 63) / 64;
    p.value_chunks = (a.value_dim + 63) / 64;
    const int room = (227 * 1024 - 2048) / CHUNK - 2 * (p.key_chunks + p.rot_chunks);
    p.slots = room < MAX_SLOTS ? room : MAX_SLOTS;
    p.splits = splits_of(a);
    return p;
}
int shared_bytes(const Plan& p) { return 1024 + (2 * (p.key_chunks + p.rot_chunks) + p.slots) * CHUNK + 8 * (11 + 2 * MAX_SLOTS) + 16; }

bool map_takes(const void* base, long long stride_b, long long stride_t, long long stride_h, int heads) {
    return stride_h >= 0 && (heads - 1) * stride_h < (1LL << 30) && reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride_b % 8 == 0 && stride_t % 8 == 0 && stride_h % 8 == 0;
}

template <typename T> int launch(const el_attention_t& a, const Plan& plan, const CUtensorMap* m, cudaStream_t st) {
    static DeviceOnce once;
    int dev = 0;
    EL_CUDA_TRY(cudaGetDevice(&dev));
    if (!once.is_done(dev)) {
        EL_CUDA_TRY(cudaFuncSetAttribute(attention_tc_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        once.mark(dev);
    }
    int sms = 148;
    device_sm_count(&sms);
    const unsigned items = blocks_of(a, a.length, 2 * TILE) * plan.splits;
    const long long rows = (long long)a.batch * a.heads * lse_pitch(a.length);
    float* sums = static_cast<float*>(a.workspace);
    const Parts parts{sums, plan.splits > 1 ? sums + plan.splits * rows * a.value_dim : nullptr, rows};
    attention_tc_kernel<T><<<items < (unsigned)sms ? items : sms, THREADS, shared_bytes(plan), st>>>(m[0], m[1], m[2], m[3], m[4], a, plan, parts);
    const int rc = check_launch();
    if (rc != EL_OK || plan.splits == 1) return rc;
    attention_join_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a, parts, plan.splits);
    return check_launch();
}

}  // namespace

// Whether the tensor-core kernels take the call.  Scales that are not positive would turn maxima into minima.
bool attention_tc_takes(const el_attention_t& a, bool backward) {
    if (a.dtype == EL_F32 || a.key_dim % 16 || a.rot_dim % 16 || a.value_dim % 16 || a.key_dim < 16 || a.key_dim > 128 || a.rot_dim > 64 || a.value_dim < 16 || a.value_dim > 128)
        return false;
    if (a.length == 0 || a.keys == 0 || !(a.scale > 0.0f && a.scale < 1e30f)) return false;
    if (!map_takes(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h, a.heads) || !map_takes(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h, a.heads) ||
        !map_takes(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h, a.heads) || reinterpret_cast<uintptr_t>(a.out) % 16)
        return false;
    if (a.rot_dim && (!map_takes(a.q_rot, a.q_rot_stride_b, a.q_rot_stride_t, a.q_rot_stride_h, a.heads) || !map_takes(a.k_rot, a.k_rot_stride_b, a.k_rot_stride_t, 0, 1))) return false;
    if (!backward) return true;
    if (!map_takes(a.dout, a.dout_stride_b, a.dout_stride_t, a.dout_stride_h, a.heads)) return false;
    if (a.dk && !map_takes(a.dk, a.dk_stride_b, a.dk_stride_t, a.dk_stride_h, 1)) return false;
    if (a.dv && !map_takes(a.dv, a.dv_stride_b, a.dv_stride_t, a.dv_stride_h, 1)) return false;
    for (const void* p : {(const void*)a.dq, (const void*)a.dq_rot, (const void*)a.lse})
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return true;
}

int attention_maps(const el_attention_t& a, CUtensorMap m[5], int query_rows, int key_rows) {
    int rc = make_map_tokens(&m[0], a.q, (a.heads - 1) * a.q_stride_h + a.key_dim, a.length, a.q_stride_t, a.batch, a.q_stride_b, query_rows);
    if (rc == EL_OK) rc = make_map_tokens(&m[2], a.k, (a.heads - 1) * a.k_stride_h + a.key_dim, a.keys, a.k_stride_t, a.batch, a.k_stride_b, key_rows);
    if (rc == EL_OK) rc = make_map_tokens(&m[4], a.v, (a.heads - 1) * a.v_stride_h + a.value_dim, a.keys, a.v_stride_t, a.batch, a.v_stride_b, key_rows);
    m[1] = m[0];
    m[3] = m[2];
    if (rc == EL_OK && a.rot_dim) rc = make_map_tokens(&m[1], a.q_rot, (a.heads - 1) * a.q_rot_stride_h + a.rot_dim, a.length, a.q_rot_stride_t, a.batch, a.q_rot_stride_b, query_rows);
    if (rc == EL_OK && a.rot_dim) rc = make_map_tokens(&m[3], a.k_rot, a.rot_dim, a.keys, a.k_rot_stride_t, a.batch, a.k_rot_stride_b, key_rows);
    return rc;
}

size_t attention_tc_workspace_bytes(const el_attention_t& a) {
    const int splits = splits_of(a);
    return splits > 1 ? (size_t)splits * a.batch * a.heads * lse_pitch(a.length) * (a.value_dim + 2) * 4 : 0;
}

int launch_attention_tc(const el_attention_t& a, cudaStream_t st) {
    CUtensorMap m[5];
    const int rc = attention_maps(a, m, TILE, TILE);
    if (rc != EL_OK) return rc;
    const Plan plan = plan_of(a);
    return a.dtype == EL_F16 ? launch<__half>(a, plan, m, st) : launch<__nv_bfloat16>(a, plan, m, st);
}

}  // namespace el
