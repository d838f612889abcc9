// Shared device helpers of the operators of latent attention (latent_attention.cu, latent_attention_tc.cu, latent_cache.cu, latent_step.cu).
#pragma once
#include "mamba_common.cuh"

namespace el {
namespace latent {

// a length from device memory (or `all` where there is none), clamped to 0 .. most
__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int all, int most) {
    const int n = lengths ? lengths[b] : all;
    return n < 0 ? 0 : n > most ? most : n;
}

// The rows of one sequence in an attention: query i (of `queries`) sees key j (of `keys`) if j <= i + shift.  Without causality the shift lets
// every query see every key.
struct Sequence {
    int queries, keys;
    long long shift;
    __device__ __forceinline__ Sequence(const el_attention_t& a, int b) {
        queries = length_of(a.lengths, b, a.length, a.length);
        keys = length_of(a.key_lengths, b, a.keys, a.keys);
        shift = a.causal ? (long long)keys - queries : (long long)keys;
    }
    __device__ __forceinline__ bool sees(int i, int j) const { return i < queries && j < keys && j <= i + shift; }
    // keys that some query of i0 .. i1 - 1 sees: 0 .. end - 1
    __device__ __forceinline__ int key_end(int i1) const {
        const int last = (i1 < queries ? i1 : queries) - 1;
        if (last < 0) return 0;
        const long long e = last + shift + 1;
        return e < 0 ? 0 : e > keys ? keys : (int)e;
    }
    // the first query that sees key j
    __device__ __forceinline__ int query_begin(int j) const {
        const long long i = j - shift;
        return i < 0 ? 0 : i > queries ? queries : (int)i;
    }
};

constexpr int LSE_PAD = 128;          // the rows of a log-sum array are padded to a multiple of this
__host__ __device__ inline long long lse_pitch(int length) { return ((long long)length + LSE_PAD - 1) / LSE_PAD * LSE_PAD; }

// A block's (or work item's) tile, sequence and head: all heads of all sequences take their first tiles first.
struct Place {
    int tile, batch, head;
    __device__ __forceinline__ Place(const el_attention_t& a, unsigned item = blockIdx.x) {
        const unsigned pairs = (unsigned)a.batch * a.heads, t = item / pairs, bh = item - t * pairs;
        tile = (int)t;
        batch = (int)(bh / a.heads);
        head = (int)(bh - (unsigned)batch * a.heads);
    }
};
// Work items in rounds of one for every block, forwards and backwards in turn: items come largest first, so a block that has a larger one of a round has a smaller
// one of the next.  Calls f(item) until it returns false.
template <typename F> __device__ __forceinline__ void each_item(unsigned items, F f) {
    for (unsigned first = 0, back = 0; first < items; first += gridDim.x, back ^= 1u) {
        const unsigned item = first + (back ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (item < items && !f(item)) return;
        if (first + gridDim.x < first) return;
    }
}
inline unsigned blocks_of(const el_attention_t& a, int rows, int tile) { return (unsigned)((rows + (long long)tile - 1) / tile * a.batch * a.heads); }

// What rounding to a 16-bit type took from a float, as a signed byte: 256ths of a step of the type, which are 2^8 (bfloat16) or 2^5 (float16) steps of a
// float32.  Floats of one sign are ordered as their bits are, so it is a difference of bits, across powers of two as well.  (A tie that went down has
// 128 of them: 127 are kept.  Below float16's normal range a step holds more: the byte is clamped and next to nothing comes back.)
template <typename T> __device__ __forceinline__ uint32_t rest_of(float v, float hi) {               // in bits 8 .. 15
    const int d = __float_as_int(v) - __float_as_int(hi);
    return std::is_same<T, __half>::value ? (uint32_t)max(min(d, 4095), -4096) << 3 : (uint32_t)min(d, 32767);
}
// the float of `hi` and byte `at` of `rests`, in the middle of what the byte stands for
template <typename T> __device__ __forceinline__ float with_rest(float hi, uint32_t rests, int at) {
    const int d = (int)prmt(rests, 0x80u, at == 0 ? 0x8804u : at == 1 ? 0x9914u : at == 2 ? 0xaa24u : 0xbb34u);
    return __int_as_float(__float_as_int(hi) + (std::is_same<T, __half>::value ? d >> 3 : d));
}

// 2^x where x <= 0 or -inf (0 then)
__device__ __forceinline__ float exp2_neg(float x) { return mamba::ex2(x); }

}  // namespace latent
}  // namespace el
