// What the kernels of a step against the cache of latent vectors share (latent_step.cu, latent_step_tc.cu): the division of all sequences' tokens
// among blocks, and the layout of what a block leaves.
//
// The sequences' tiles of STEP_TILE tokens lie one after another, N in all; worker w of G <= N takes tiles w N / G .. (w + 1) N / G - 1, which may be
// parts of several sequences.  Every worker has the same share whatever the lengths are.  What worker w found in sequence b (each head's largest
// score, its sum and its weighted latent vectors) goes to slot w + b: from one part of a worker to its next b grows, and where one worker ends inside a
// sequence the next one begins there, so no two parts share a slot.
#pragma once
#include "latent_common.cuh"

namespace el {
namespace latent {

constexpr int STEP_TILE = 32;

__device__ __forceinline__ int step_tokens(const el_latent_step_t& a, int b) {
    return length_of(a.lengths, b, 0, (int)min((long long)a.pages_per_sequence * a.page_size, 0x7fffff00LL));
}
__device__ __forceinline__ int step_tiles(const el_latent_step_t& a, int b) { return (step_tokens(a, b) + STEP_TILE - 1) / STEP_TILE; }

// Tiles of all sequences; called by a whole warp.
__device__ __forceinline__ long long step_all_tiles(const el_latent_step_t& a) {
    long long n = 0;
#pragma unroll 4
    for (int b = threadIdx.x & 31; b < a.batch; b += 32) n += step_tiles(a, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
}
// The sequence that tile `t` (of all) belongs to and the tiles before that sequence; called by a whole warp, t < all tiles.
__device__ __forceinline__ void step_find(const el_latent_step_t& a, long long t, int& seq, long long& before) {
    const int lane = threadIdx.x & 31;
    before = 0;
    int next = lane < a.batch ? step_tiles(a, lane) : 0;
    for (int b0 = 0;; b0 += 32) {
        const int n = next;
        next = b0 + 32 + lane < a.batch ? step_tiles(a, b0 + 32 + lane) : 0;
        long long upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > t);
        if (past || b0 + 32 >= a.batch) {
            const int l = past ? __ffs(past) - 1 : 31;
            seq = b0 + l;
            before += __shfl_sync(0xffffffffu, upto - n, l);
            return;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}
// workers with something to do: of as many as there are tiles, or fewer, none is without one
__device__ __forceinline__ int step_active(int workers, long long tiles) { return tiles < workers ? (int)tiles : workers; }
// the worker that has tile t
__device__ __forceinline__ int step_worker(long long t, int workers, long long tiles) { return (int)(((t + 1) * workers - 1) / tiles); }

// A slot: for each head its largest score and its sum, and its latent vector.
struct StepParts {
    float *vectors_at, *stats_at;
    int heads, rank;
    __device__ __forceinline__ float* vectors(long long slot) const { return vectors_at + slot * heads * rank; }
    __device__ __forceinline__ float* stats(long long slot) const { return stats_at + slot * heads * 2; }
};

// The query of a group of up to 32 heads as the tensor-core kernel keeps it in shared memory: 128-byte chunks of latent channels, in each a row of a head's
// high digits for every head, then of low digits (rows padded to 16 or 32 heads); behind them w, a row of 64 values for every head.  A row's 16-byte pieces
// change places by its number, as the matrix descriptors' 128-byte swizzle has it.
struct StepImage {
    int chunks, hp, groups;
    bool rotated;
    __host__ __device__ explicit StepImage(const el_latent_step_t& a)
        : chunks((a.rank + 127) / 128), hp(a.heads <= 16 ? 16 : 32), groups((a.heads + 31) / 32), rotated(a.rot_dim > 0) {}
    __host__ __device__ int w_at() const { return chunks * 2 * hp * 128; }
    __host__ __device__ int bytes() const { return w_at() + (rotated ? hp * 128 : 0); }
    __host__ __device__ static int in_row(int row, int byte) { return row * 128 + ((((byte >> 4) ^ row) & 7) << 4) + (byte & 15); }
    // byte of channel c of digit 0 or 1 of head h (of the group); of w's byte x
    __host__ __device__ int digit(int c, int d, int h) const { return (c >> 7) * 2 * hp * 128 + in_row(d * hp + h, c & 127); }
    __host__ __device__ int w(int x, int h) const { return w_at() + in_row(h, x); }
};

// the pool's row of position p of sequence b, or -1
__device__ __forceinline__ long long step_row(const el_latent_step_t& a, int b, int p) {
    const int page = a.block_table[(long long)b * a.pages_per_sequence + p / a.page_size];
    return page < 0 || page >= a.pages ? -1 : (long long)page * a.page_size + p % a.page_size;
}

}  // namespace latent
}  // namespace el
