// tcgen05 building blocks of the attention kernels (latent_attention_tc.cu, latent_backward_tc.cu, latent_step_tc.cu): 16-bit products with
// float32 sums, operands in shared or tensor memory, and tiles of 64 columns x 128 bytes.
//
// Operands lie in shared memory as chunks of 64 columns (128 bytes) by any number of rows, swizzled by 128 bytes.  A chunk is K-major where its
// columns are the reduction (rows are M or N) and MN-major where its rows are the reduction (columns are M or N).
#pragma once
#include "latent_common.cuh"
#include "tc_ptx.cuh"

namespace el {
namespace tc {

constexpr int CHUNK_COLS = 64;

// The value of lane 0, in a form that the compiler knows to be the same for the whole warp.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// Matrix descriptors by halves: the upper one is the same for all operands here (make_desc), the lower one is the address, which a step along the reduction
// moves by a constant (2 for 32 bytes of a K-major row, 128 for 16 rows of an MN-major one).  One warp issues the products, an instruction every few
// cycles: with descriptors built anew for every product it took 130 cycles for each, where a 128 x 128 x 16 product itself takes 64.
constexpr uint32_t DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo_bytes) { return ((saddr & 0x3FFFFu) >> 4) | ((lbo_bytes >> 4) << 16); }
__device__ __forceinline__ uint64_t desc_of(uint32_t low) { return ((uint64_t)DESC_HIGH << 32) | low; }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// `bytes` (a multiple of 16) from 16-byte aligned global memory
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// d += or = a b, a and b in shared memory
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the same, a in tensor memory: lane m holds row m, a column two neighbouring values
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// d += or = a b over `steps` (1 .. 4) steps of 16 along the reduction, both operands K-major chunks; one thread
__device__ __forceinline__ void umma_f16_chunk(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate, int steps) {
    umma_f16(d_tmem, desc_of(a_low), desc_of(b_low), idesc, accumulate);
    if (steps == 4) {
#pragma unroll
        for (int x = 1; x < 4; ++x) umma_f16(d_tmem, desc_of(a_low + 2 * x), desc_of(b_low + 2 * x), idesc, 1u);
        return;
    }
#pragma unroll 1
    for (int x = 1; x < steps; ++x) umma_f16(d_tmem, desc_of(a_low + 2 * x), desc_of(b_low + 2 * x), idesc, 1u);
}
// the same with the left operand in tensor memory, 8 columns a step
__device__ __forceinline__ void umma_f16_ts_chunk(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate, int steps) {
    umma_f16_ts(d_tmem, a_tmem, desc_of(b_low), idesc, accumulate);
    if (steps == 4) {
#pragma unroll
        for (int x = 1; x < 4; ++x) umma_f16_ts(d_tmem, a_tmem + 8 * x, desc_of(b_low + 2 * x), idesc, 1u);
        return;
    }
#pragma unroll 1
    for (int x = 1; x < steps; ++x) umma_f16_ts(d_tmem, a_tmem + 8 * x, desc_of(b_low + 2 * x), idesc, 1u);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
          "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
          "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t holder) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(holder), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS> __device__ __forceinline__ void tmem_free(uint32_t base) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS) : "memory");
}

// Instruction descriptor of kind::f16: float32 sums, A and B of one type.
template <typename T> __device__ __forceinline__ uint32_t idesc_f16(int a_mn_major, int b_mn_major, int n, int m = 128) {
    constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Four lanes that hold four neighbouring rows, 64 bytes of each (w), exchange them so that each lane has one 16-byte piece of all four: w[4 k ..] becomes
// piece lane % 4 of row k.  A store of piece k then writes 64 neighbouring bytes of eight rows instead of 16 bytes of 32.
__device__ __forceinline__ void transpose_rows(uint32_t (&w)[16]) {
    const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
#pragma unroll
    for (int u = 0; u < 4; u += 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t a = w[4 * u + e], b = w[4 * u + 4 + e], got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
            w[4 * u + e] = odd ? got : a;
            w[4 * u + 4 + e] = odd ? b : got;
        }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t a = w[4 * u + e], b = w[4 * u + 8 + e], got = __shfl_xor_sync(0xffffffffu, upper ? a : b, 2);
            w[4 * u + e] = upper ? got : a;
            w[4 * u + 8 + e] = upper ? b : got;
        }
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
// The split of a block's registers among its groups of four warps; every warp of a group calls one of the two.
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// two values as a word of type T, the first in its low half
template <typename T> __device__ __forceinline__ uint32_t pack_word(float lo, float hi) {
    return std::is_same<T, __half>::value ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
// the rests of four values whose rounded ones are two words
template <typename T> __device__ __forceinline__ uint32_t rest_word(uint32_t w0, uint32_t w1, float x0, float x1, float x2, float x3) {
    float2 a, b;
    if constexpr (std::is_same<T, __half>::value) {
        a = __half22float2(*reinterpret_cast<const __half2*>(&w0));
        b = __half22float2(*reinterpret_cast<const __half2*>(&w1));
    } else {
        a = make_float2(__uint_as_float(w0 << 16), __uint_as_float(w0 & 0xffff0000u));
        b = make_float2(__uint_as_float(w1 << 16), __uint_as_float(w1 & 0xffff0000u));
    }
    using latent::rest_of;
    return prmt(prmt(rest_of<T>(x0, a.x), rest_of<T>(x1, a.y), 0x0051u), prmt(rest_of<T>(x2, b.x), rest_of<T>(x3, b.y), 0x0051u), 0x5410u);
}

// host: a map of [batch, tokens, inner] 16-bit values for boxes of 64 columns and `rows` tokens; out-of-range reads give zeros
int make_map_tokens(CUtensorMap* m, const void* base, uint64_t inner, uint64_t tokens, uint64_t stride_t, uint64_t batch, uint64_t stride_b, uint32_t rows);

}  // namespace tc
}  // namespace el
