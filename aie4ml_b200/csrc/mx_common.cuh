// MXFP4 (OCP microscaling, E2M1 elements, E8M0 scales over blocks of 32): conversions and the block-scaled tcgen05
// instructions shared by the quantisation and the Dense kernels.
//
// Storage.  Codes: two 4-bit values to a byte, even column in the low nibble.  Scales: one byte per row and block,
// value 2^(s - 127), 255 = NaN, in tiles of 128 rows x 4 blocks (512 bytes): byte (r % 32) * 16 + (r / 32) * 4 + b.
// That is the order in which tcgen05.cp moves 32 lanes of 16 bytes into tensor memory, so a tile goes from HBM to
// shared memory as one untiled bulk copy and from there to TMEM as one instruction, without a thread touching it.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "tc_common.cuh"

namespace mx {

constexpr int BLOCK = 32;            // values per scale
constexpr int TILE_ROWS = 128;       // rows per scale tile
constexpr int TILE_BLOCKS = 4;       // blocks (of one row) per scale tile
constexpr int TILE_BYTES = TILE_ROWS * TILE_BLOCKS;
constexpr int KIND_BF16 = 0, KIND_F32 = 1, KIND_MX = 3;   // the fdtype codes of the C ABI

__host__ __device__ inline long long tiles_across(long long cols) { return (cols + TILE_BLOCKS * BLOCK - 1) / (TILE_BLOCKS * BLOCK); }

// byte offset of the scale of (row, block); `across` = tiles_across(cols)
__device__ __forceinline__ long long scale_offset(long long row, long long block, long long across) {
    return ((row >> 7) * across + (block >> 2)) * TILE_BYTES + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// Largest magnitude's float bits (sign cleared; NaN and infinity order above every finite value) -> scale code.
// floor(log2) is the exponent field, 2 is the exponent of the largest E2M1 binade; subnormal and zero maxima take the
// smallest scale.
__device__ __forceinline__ uint32_t scale_code(uint32_t absmax_bits) {
    const uint32_t e = absmax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(127 - s), the factor that brings a block into E2M1's range; exact for every s scale_code returns but 255
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127); s = 0 is the subnormal 2^-127, 255 is NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7FC00000u : s << 23));
}

// Eight scaled values -> eight E2M1 codes, element 0 in the lowest nibble.  Round to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t pack_e2m1(const float* v) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}
// Eight E2M1 codes -> float (exact)
__device__ __forceinline__ void unpack_e2m1(uint32_t w, float* v) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "mov.b32 {lo, hi}, %2;\n\t"
            "cvt.f32.f16 %0, lo;\n\t"
            "cvt.f32.f16 %1, hi;\n\t}" : "=f"(v[2 * i]), "=f"(v[2 * i + 1]) : "r"(h[i]));
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}

// ---- block-scaled tensor-core instructions ------------------------------------------------------
// Instruction descriptor of kind::mxf4: [4,6) byte of B's scale word, [7,10) and [10,12) element types (1 = E2M1),
// [17,23) N >> 3, bit 23 scale type (1 = E8M0), [24,29) M >> 4, [29,31) byte of A's scale word.  Both operands K-major.
constexpr uint32_t make_idesc(int m, int n) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
// one MMA covers 64 values of K = two blocks: bytes 0-1 or 2-3 of the scale words
constexpr uint32_t sf_bits(int half) { return ((uint32_t)(half * 2) << 4) | ((uint32_t)(half * 2) << 29); }

__device__ __forceinline__ void umma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                     uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :: "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// A 512-byte scale tile as the source of tcgen05.cp: 32 rows of 16 bytes without swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// 32 lanes x 4 columns, repeated in each quarter of the lanes
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc) : "memory");
}
// untiled bulk copy HBM -> shared memory; both addresses and the size are multiples of 16 bytes
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(tc::smem_u32(dst)), "l"(src), "r"(bytes), "r"(tc::smem_u32(bar)) : "memory");
}

// ---- activations of the gated Dense -------------------------------------------------------------
constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SIGMOID = 5, ACT_COUNT = 6;

// 1 / (1 + exp(-x)) in float32: exp overflows to infinity for x below -88 and the quotient is then 0, as it should be
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

__device__ __forceinline__ float activate(float x, int act) {
    switch (act) {
        case ACT_RELU: return x < 0.0f ? 0.0f : x;      // a NaN stays one
        case ACT_SILU: return x * sigmoid(x);
        case ACT_GELU: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
        // 0.5 (1 + tanh z) = sigmoid(2 z)
        case ACT_GELU_TANH: return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
        case ACT_SIGMOID: return sigmoid(x);
        default: return x;
    }
}

}  // namespace mx
