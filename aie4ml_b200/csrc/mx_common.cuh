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

// Two float32 values in a 64-bit register pair: one instruction for both, half the issue slots of an epilogue.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ f2 both(float x) { return pack2(x, x); }
__device__ __forceinline__ void unpack2(f2 p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float exp2_approx(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float rcp_approx(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
template <float (*F)(float)>
__device__ __forceinline__ f2 each2(f2 p) {
    float a, b;
    unpack2(p, a, b);
    return pack2(F(a), F(b));
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

// Largest magnitude of 32 values as float bits; a NaN wins (scale_code then finds it)
__device__ __forceinline__ uint32_t abs_max32(const float* v) {
    float m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = fabsf(v[8 * k]);
#pragma unroll
        for (int i = 1; i < 7; i += 2)
            asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m[k]) : "f"(fabsf(v[8 * k + i])), "f"(fabsf(v[8 * k + i + 1])));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[k]) : "f"(fabsf(v[8 * k + 7])));
    }
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m[0]) : "f"(m[1]), "f"(m[2]));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[0]) : "f"(m[3]));
    return __float_as_uint(m[0]) & 0x7FFFFFFFu;
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

// 32 float32 values -> their codes and scale
__device__ __forceinline__ uint32_t quantize32(const float* v, uint32_t* w) {
    const uint32_t s = scale_code(abs_max32(v));
    const f2 inv = both(inverse_scale(s == 255u ? 0u : s));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float q[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) unpack2(mul2(pack2(v[8 * i + 2 * k], v[8 * i + 2 * k + 1]), inv), q[2 * k], q[2 * k + 1]);
        w[i] = s == 255u ? 0u : pack_e2m1(q);
    }
    return s;
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

// true in one lane of a converged warp.  The tensor-core roles run their loops with whole warps and elect a lane for the
// instructions themselves: descriptors then stay in uniform registers, where a loop inside `if (lane == 0)` moves each of
// them over for every instruction.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
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


// ---- back-to-back launches ----------------------------------------------------------------------
// The MXFP4 kernels are launched with programmatic stream serialization: a kernel may be set up (barriers, tensor memory)
// while the one before it in the stream drains.  Nothing in global memory is read or written ahead of grid_wait, which
// returns when the kernels before it have completed and their writes are visible.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// cluster = 0: the kernel has its own cluster size, or none
template <typename... P, typename... A>
inline cudaError_t launch_serialized(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, unsigned cluster, cudaStream_t s,
                                     const A&... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- clusters and CTA pairs ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// shared::cluster address of `local` (a shared::cta address) in CTA `rank`
__device__ __forceinline__ uint32_t map_to_cta(uint32_t local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    return a;
}
// Says that tensor memory has been read (tcgen05.wait::ld before it): no memory of this thread's is handed over, so the arrival
// needs no release, which would first wait for the thread's stores.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
// TMA loads whose completion may be signalled on the peer CTA's barrier (cta_group::2 form, no multicast)
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        :: "r"(tc::smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        :: "r"(tc::smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// Both CTAs of the pair: each copies from its own shared memory, at the same offset, to its own tensor memory
__device__ __forceinline__ void copy_scales_pair(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :: "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// arrives, when the MMAs issued so far are done, on the barrier at this offset in both CTAs
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(bar), "h"((uint16_t)3) : "memory");
}

// ---- tensor maps (host) -------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
    }();
    return fn;
}

// codes [rows, ceil(K / 2) bytes], pitch ld elements; box = 256 values x box_rows, 128-byte swizzle; outside reads as zero
inline bool make_code_map(CUtensorMap* map, const void* base, long long rows, int K, long long ld, int box_rows) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)((K + 1) / 2), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld / 2)};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// scale tiles as [row groups, tiles across K, 512 bytes]; box = two tiles of one row group
inline bool make_scale_map(CUtensorMap* map, const void* base, long long rows, int K) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t across = (cuuint64_t)tiles_across(K);
    cuuint64_t dims[3] = {TILE_BYTES / 4, across, (cuuint64_t)((rows + TILE_ROWS - 1) / TILE_ROWS)};
    cuuint64_t strides[2] = {TILE_BYTES, across * TILE_BYTES};
    cuuint32_t box[3] = {TILE_BYTES / 4, 2, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// an output [rows, cols] for TMA stores of 32 rows: 64 bytes of bf16 or f32 (64-byte swizzle), 32 bytes (64 codes) of MXFP4
inline bool make_out_map(CUtensorMap* map, void* base, int kind, long long rows, int cols, long long ld) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const bool codes = kind == KIND_MX;
    const int esz = kind == KIND_F32 ? 4 : 2;
    cuuint64_t dims[2] = {(cuuint64_t)(codes ? (cols + 1) / 2 : cols), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(codes ? ld / 2 : ld * esz)};
    cuuint32_t box[2] = {(cuuint32_t)(codes ? 32 : 64 / esz), 32};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : kind == KIND_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
              2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---- activations of the gated Dense -------------------------------------------------------------
constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4, ACT_SIGMOID = 5;

constexpr float LOG2E = 1.4426950408889634f;

// 1 / (1 + 2^z): 2^z overflows to infinity where the quotient is 0, as it should be
__device__ __forceinline__ f2 inv_one_plus_exp2(f2 z) { return each2<rcp_approx>(add2(each2<exp2_approx>(z), both(1.0f))); }

// x Phi(x) = max(x, 0) - a Phi(-a), a = |x|, and Phi(-a) = 2^Q(a): log2 Phi(-a) is so near a parabola that nine terms do, with
// one exponential and no quotient.  The coefficients are a least maximum fit (linear programming) of the result's absolute
// error, weighted by max(a, 1/2) Phi(-a) over 0 <= a <= 13, with a relative error of at most 2^-9 (half a bf16 step) down to
// x = -6; that is 3.0e-8 beside the roundings.  Beyond -6, where the result is smaller than 6e-9, its relative error grows to 1.
// Q falls on to below -10^8 at a = 64, where the power is 0.  NaN stays NaN.  Against a term less, fitted without the second
// condition (1.6e-7; 0.4 % at -5 and 1.9 % at -6): a gated 65536 x 256 x 2*1024 takes 48.4 us for 47.3, and a quarter as many
// values of a feed-forward block's hidden tensor change their code (14 for 52 in 2*10^8; the elementary form in 32 bits: 8).  Two
// terms more, 1.6e-8 and 2^-9 down to -10, took 52.7 us.
// (By the rational form of erfc, an exponential and a reciprocal, it took 59 us; erff takes twice the instructions, and 1 + erf
// cancels for negative x.)
__device__ __forceinline__ f2 gelu2(f2 x) {
    float a, b, na, nb, pa, pb;
    unpack2(x, a, b);
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tneg.f32 t, t;\n\tmax.NaN.f32 %0, t, 0fC2800000;\n\t}" : "=f"(na) : "f"(a));    // -64
    asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %1;\n\tneg.f32 t, t;\n\tmax.NaN.f32 %0, t, 0fC2800000;\n\t}" : "=f"(nb) : "f"(b));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(pa) : "f"(a));
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(pb) : "f"(b));
    const f2 n = pack2(na, nb);
    f2 q = fma2(n, both(-1.1569092066565645e-06f), both(-1.913546111609321e-05f));
    q = fma2(n, q, both(-8.965825691120699e-05f));
    q = fma2(n, q, both(0.0003700188244692981f));
    q = fma2(n, q, both(0.007366466801613569f));
    q = fma2(n, q, both(0.0527038499712944f));
    q = fma2(n, q, both(-0.4591405689716339f));
    q = fma2(n, q, both(1.1511132717132568f));
    q = fma2(n, q, both(-0.9999998211860657f));
    return fma2(n, each2<exp2_approx>(q), pack2(pa, pb));
}

template <int ACT>
__device__ __forceinline__ f2 activate2(f2 x) {
    if (ACT == ACT_RELU) {
        float a, b;
        unpack2(x, a, b);
        return pack2(a < 0.0f ? 0.0f : a, b < 0.0f ? 0.0f : b);
    }
    if (ACT == ACT_SILU) return mul2(x, inv_one_plus_exp2(mul2(x, both(-LOG2E))));
    if (ACT == ACT_SIGMOID) return inv_one_plus_exp2(mul2(x, both(-LOG2E)));
    if (ACT == ACT_GELU) return gelu2(x);
    if (ACT == ACT_GELU_TANH) {      // (1 + tanh z) / 2 = 1 / (1 + exp(-2 z)), z = sqrt(2 / pi) (x + 0.044715 x^3)
        constexpr float C = -2.0f * 0.79788456080286536f * LOG2E;
        const f2 z = mul2(x, fma2(mul2(x, x), both(0.044715f * C), both(C)));
        return mul2(x, inv_one_plus_exp2(z));
    }
    return x;
}

// N pairs of one activation, the switch outside the loop
template <int N>
__device__ __forceinline__ void activate_pairs(f2* v, int act) {
    switch (act) {
#define A4C_MX_EACH(A) case A: _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = activate2<A>(v[i]); break;
        A4C_MX_EACH(ACT_RELU) A4C_MX_EACH(ACT_SILU) A4C_MX_EACH(ACT_GELU) A4C_MX_EACH(ACT_GELU_TANH) A4C_MX_EACH(ACT_SIGMOID)
#undef A4C_MX_EACH
        default: break;
    }
}
}  // namespace mx
