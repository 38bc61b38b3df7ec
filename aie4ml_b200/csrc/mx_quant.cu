// Quantisation to and from MXFP4.
//
//   s[r,b]    = max(floor(log2(max |x| over the block)) + 127 - 2, 0), or 255 when the block holds a NaN or an infinity
//   code[r,c] = E2M1(x[r,c] * 2^(127 - s)), nearest even, saturating at 6;     y[r,c] = E2M1 value * 2^(s - 127)
//
// Bound by HBM: one pass, 2 (bfloat16) or 4 (float32) bytes an element on one side and 17/32 byte on the other.  A lane
// takes eight neighbouring columns, so a block is four lanes and its maximum two shuffles; a warp takes 256 columns of a
// row.  A CTA takes 128 rows x 256 columns: exactly two scale tiles, which it gathers in shared memory and writes out
// whole (places beyond the tensor as 0), because single scale bytes 16 bytes apart would touch every 32-byte sector of
// the scale array many times.  Where that leaves SMs idle a CTA takes 32 rows, a quarter of each tile: a word in 16 bytes.
#include "a4c_common.cuh"
#include "a4c_kernels.h"
#include "mx_common.cuh"

namespace {

using namespace mx;

constexpr int COLS = 256;            // columns per CTA: 32 lanes x 8
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;

struct QuantArgs {
    const void* x; long long ldx;
    uint8_t* codes; long long ldc_bytes;
    uint8_t* scales;
    long long rows, cols, across;
    unsigned grid_cols;              // CTAs across the columns
    int vec;                         // x can be read in 16-byte pieces
};

// Eight neighbouring values as they lie in memory; those beyond `valid` read as zero
template <int KIND> struct Raw { uint32_t w[KIND == KIND_BF16 ? 4 : 8]; };

template <int KIND>
__device__ __forceinline__ Raw<KIND> load8(const uint8_t* src, int valid, bool vec) {
    Raw<KIND> r;
    if (KIND == KIND_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(src);
        if (vec && valid == 8) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
            r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                r.w[i] = (2 * i < valid ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < valid ? (uint32_t)p[2 * i + 1] << 16 : 0u);
        }
    } else {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(src);
        if (vec && valid == 8) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p)), b = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
            r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
            r.w[4 % (sizeof(r.w) / 4)] = b.x; r.w[5 % (sizeof(r.w) / 4)] = b.y; r.w[6 % (sizeof(r.w) / 4)] = b.z; r.w[7 % (sizeof(r.w) / 4)] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(r.w) / 4); ++i) r.w[i] = i < valid ? p[i] : 0u;
        }
    }
    return r;
}
template <int KIND>
__device__ __forceinline__ void values_of(const Raw<KIND>& r, float* v) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(r.w) / 4); ++i) {
        if (KIND == KIND_BF16) { v[2 * i] = __uint_as_float(r.w[i] << 16); v[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u); }
        else v[i] = __uint_as_float(r.w[i]);
    }
}

// Largest magnitude of the eight: float bits whose order is that of the magnitudes, NaN above infinity above the rest
template <int KIND>
__device__ __forceinline__ uint32_t abs_max(const Raw<KIND>& r) {
    if (KIND == KIND_BF16) {             // two at a time; a NaN stays one
        uint32_t m = r.w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(r.w[i] & 0x7FFF7FFFu));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(m >> 16));
        return m << 16;
    }
    uint32_t m = r.w[0] & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < (int)(sizeof(r.w) / 4); ++i) m = max(m, r.w[i] & 0x7FFFFFFFu);
    return m;
}

constexpr int BATCH = 4;             // rows whose loads a warp issues before it converts any (the stores between would hold them back)

// QUARTERS x 32 rows per CTA: 4 (whole scale tiles) or 1
template <int KIND, int QUARTERS>
__global__ void __launch_bounds__(THREADS) quantize_kernel(QuantArgs g) {
    constexpr int ROWS = QUARTERS * 32;
    __shared__ __align__(16) uint8_t sc[2 * TILE_BYTES / 4 * QUARTERS];   // [tile][row % 32][quarter][block]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const long long col = (long long)bx * COLS + lane * 8;
    const int valid = (int)max(0LL, min(8LL, g.cols - col));
    if (threadIdx.x < 64 * QUARTERS) reinterpret_cast<uint32_t*>(sc)[threadIdx.x] = 0u;
    __syncthreads();
    grid_wait();
    grid_release();
    const int code_bytes = (valid + 1) >> 1;      // an odd last column leaves a zero in the high nibble
    const int count = (int)max(0LL, min((long long)ROWS, g.rows - row0));
    constexpr int ESZ = KIND == KIND_BF16 ? 2 : 4;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(g.x) + ((row0 + warp) * g.ldx + col) * ESZ;
    const long long src_step = (long long)WARPS * g.ldx * ESZ;
    uint8_t* dst = g.codes + (row0 + warp) * g.ldc_bytes + (col >> 1);
    const long long dst_step = (long long)WARPS * g.ldc_bytes;
    const int b = lane >> 2;                      // block within the CTA's eight
    uint8_t* my_sc = sc + (b >> 2) * 128 * QUARTERS + (b & 3);
    for (int first = warp; first < count; first += BATCH * WARPS) {
        Raw<KIND> raw[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j, src += src_step)
            raw[j] = load8<KIND>(src, first + j * WARPS < count ? valid : 0, g.vec != 0);
#pragma unroll
        for (int j = 0; j < BATCH; ++j, dst += dst_step) {
            const int r = first + j * WARPS;
            if (r >= count) break;                // the same for the whole warp
            uint32_t top = abs_max(raw[j]);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t s = scale_code(top);
            const f2 inv = both(inverse_scale(s == 255u ? 0u : s));
            float v[8];
            values_of(raw[j], v);
#pragma unroll
            for (int k = 0; k < 4; ++k) unpack2(mul2(pack2(v[2 * k], v[2 * k + 1]), inv), v[2 * k], v[2 * k + 1]);
            const uint32_t w = s == 255u ? 0u : pack_e2m1(v);
            if (valid == 8) *reinterpret_cast<uint32_t*>(dst) = w;
            else for (int k = 0; k < code_bytes; ++k) dst[k] = (uint8_t)(w >> (8 * k));
            if ((lane & 3) == 0 && valid > 0) my_sc[((r & 31) * QUARTERS + (r >> 5)) * 4] = (uint8_t)s;
        }
    }
    __syncthreads();
    // a thread per tile and row % 32; the second tile exists when the tensor reaches into it
    if (threadIdx.x < 64) {
        const long long tile = (long long)bx * 2 + (threadIdx.x >> 5);
        if (tile < g.across) {
            uint8_t* dst = g.scales + ((row0 / TILE_ROWS) * g.across + tile) * TILE_BYTES + (threadIdx.x & 31) * 16;
            if (QUARTERS == 4) *reinterpret_cast<uint4*>(dst) = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
            else reinterpret_cast<uint32_t*>(dst)[by & 3] = reinterpret_cast<const uint32_t*>(sc)[threadIdx.x];
        }
    }
}

struct DequantArgs {
    const uint8_t* codes; long long ldc_bytes;
    const uint8_t* scales;
    void* y; long long ldy;
    long long rows, cols, across;
    unsigned grid_cols;
    int vec;                         // y can be written in pieces of eight values (16 or 32 bytes)
};

template <int KIND, int QUARTERS>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(DequantArgs g) {
    constexpr int ROWS = QUARTERS * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const long long col = (long long)bx * COLS + lane * 8;
    const int valid = (int)max(0LL, min(8LL, g.cols - col));
    grid_wait();
    grid_release();
    if (valid == 0) return;
    const int count = (int)max(0LL, min((long long)ROWS, g.rows - row0));
    constexpr int ESZ = KIND == KIND_BF16 ? 2 : 4;
    const uint8_t* src = g.codes + (row0 + warp) * g.ldc_bytes + (col >> 1);
    const long long src_step = (long long)WARPS * g.ldc_bytes;
    uint8_t* dst = reinterpret_cast<uint8_t*>(g.y) + ((row0 + warp) * g.ldy + col) * ESZ;
    const long long dst_step = (long long)WARPS * g.ldy * ESZ;
    const uint8_t* scales = g.scales + scale_offset(row0, col >> 5, g.across);     // row0 is a multiple of 32
    for (int first = warp; first < count; first += BATCH * WARPS) {
        uint32_t code[BATCH];
        uint8_t sc[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j, src += src_step) {
            const int r = first + j * WARPS;
            code[j] = 0;
            sc[j] = 0;
            if (r >= count) continue;
            if (valid == 8) code[j] = __ldcs(reinterpret_cast<const uint32_t*>(src));
            else for (int k = 0; k < (valid + 1) >> 1; ++k) code[j] |= (uint32_t)src[k] << (8 * k);
            sc[j] = __ldg(scales + (r & 31) * 16 + (r >> 5) * 4);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j, dst += dst_step) {
            if (first + j * WARPS >= count) break;
            const f2 scale = both(scale_value(sc[j]));
            float v[8];
            unpack_e2m1(code[j], v);
#pragma unroll
            for (int k = 0; k < 4; ++k) unpack2(mul2(pack2(v[2 * k], v[2 * k + 1]), scale), v[2 * k], v[2 * k + 1]);
            if (KIND == KIND_BF16) {
                const uint4 q = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
                if (g.vec && valid == 8) __stcs(reinterpret_cast<uint4*>(dst), q);
                else {
                    const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int k = 0; k < 8; ++k) if (k < valid) reinterpret_cast<uint16_t*>(dst)[k] = (uint16_t)(p[k >> 1] >> (16 * (k & 1)));
                }
            } else if (g.vec && valid == 8) {          // 32 bytes at once: two 16-byte stores would each fill half a sector
                asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                             :: "l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) if (k < valid) reinterpret_cast<float*>(dst)[k] = v[k];
            }
        }
    }
}

// CTAs of `quarters` x 32 rows; rows of the last scale tile beyond the tensor belong to somebody too
bool grid_of(long long rows, long long cols, int& quarters, unsigned& grid, unsigned& grid_cols) {
    const long long gx = (cols - 1) / COLS + 1, gy = (rows - 1) / TILE_ROWS + 1;
    if (gx > 2147483647LL / gy) return false;
    quarters = gx * gy < 8 * 148 ? 1 : 4;
    grid = (unsigned)(gx * gy * (quarters == 1 ? 4 : 1));
    grid_cols = (unsigned)gx;
    return true;
}

template <int KIND>
cudaError_t launch_quantize(const QuantArgs& g, int quarters, unsigned grid, cudaStream_t s) {
    return launch_serialized(quarters == 1 ? quantize_kernel<KIND, 1> : quantize_kernel<KIND, 4>, grid, THREADS, 0, 0, s, g);
}
template <int KIND>
cudaError_t launch_dequantize(const DequantArgs& g, int quarters, unsigned grid, cudaStream_t s) {
    return launch_serialized(quarters == 1 ? dequantize_kernel<KIND, 1> : dequantize_kernel<KIND, 4>, grid, THREADS, 0, 0, s, g);
}

}  // namespace

int a4c_launch_quantize_mx(const void* x, int kind, long long ldx, uint8_t* codes, long long ldc, uint8_t* scales,
                           long long rows, long long cols, cudaStream_t stream) {
    unsigned grid;
    int quarters;
    QuantArgs g;
    if (!grid_of(rows, cols, quarters, grid, g.grid_cols)) return A4C_ERR_TOO_LARGE;
    const int esz = kind == KIND_BF16 ? 2 : 4;
    g.x = x; g.ldx = ldx; g.codes = codes; g.ldc_bytes = ldc / 2; g.scales = scales; g.rows = rows; g.cols = cols;
    g.across = tiles_across(cols);
    g.vec = ((uintptr_t)x & 15u) == 0 && (ldx * esz) % 16 == 0;
    const cudaError_t e = kind == KIND_BF16 ? launch_quantize<KIND_BF16>(g, quarters, grid, stream) : launch_quantize<KIND_F32>(g, quarters, grid, stream);
    return e == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}

int a4c_launch_dequantize_mx(const uint8_t* codes, long long ldc, const uint8_t* scales, void* y, int kind, long long ldy,
                             long long rows, long long cols, cudaStream_t stream) {
    unsigned grid;
    int quarters;
    DequantArgs g;
    if (!grid_of(rows, cols, quarters, grid, g.grid_cols)) return A4C_ERR_TOO_LARGE;
    const int esz = kind == KIND_BF16 ? 2 : 4;
    g.codes = codes; g.ldc_bytes = ldc / 2; g.scales = scales; g.y = y; g.ldy = ldy; g.rows = rows; g.cols = cols;
    g.across = tiles_across(cols);
    g.vec = ((uintptr_t)y & (8u * esz - 1)) == 0 && ldy % 8 == 0;
    const cudaError_t e = kind == KIND_BF16 ? launch_dequantize<KIND_BF16>(g, quarters, grid, stream) : launch_dequantize<KIND_F32>(g, quarters, grid, stream);
    return e == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}
