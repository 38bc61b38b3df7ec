// Quantisation to and from MXFP4.
//
//   s[r,b]    = max(floor(log2(max |x| over the block)) + 127 - 2, 0), or 255 when the block holds a NaN or an infinity
//   code[r,c] = E2M1(x[r,c] * 2^(127 - s)), nearest even, saturating at 6;     y[r,c] = E2M1 value * 2^(s - 127)
//
// Bound by HBM: one pass, 2 (bfloat16) or 4 (float32) bytes an element on one side and 17/32 byte on the other.  A lane
// takes eight neighbouring columns, so a block is four lanes and its maximum two shuffles; a warp takes 256 columns of a
// row.  A CTA takes 128 rows x 256 columns: exactly two scale tiles, which it gathers in shared memory and writes out
// whole (places beyond the tensor as 0), because single scale bytes 16 bytes apart would touch every 32-byte sector of
// the scale array many times.
#include "a4c_common.cuh"
#include "a4c_kernels.h"
#include "mx_common.cuh"

namespace {

using namespace mx;

constexpr int ROWS = TILE_ROWS;      // rows per CTA
constexpr int COLS = 256;            // columns per CTA: 32 lanes x 8
constexpr int THREADS = 256;
constexpr int ROWS_PER_WARP = ROWS / (THREADS / 32);

struct QuantArgs {
    const void* x; long long ldx;
    uint8_t* codes; long long ldc_bytes;
    uint8_t* scales;
    long long rows, cols, across;
    unsigned grid_cols;              // CTAs across the columns
    int vec;                         // x can be read in 16-byte pieces
};

template <int KIND>
__device__ __forceinline__ void load8(const void* base, long long idx, int valid, bool vec, float* v) {
    if (KIND == KIND_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + idx;
        if (vec && valid >= 8) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < valid ? __uint_as_float((uint32_t)p[i] << 16) : 0.0f;
        }
    } else {
        const float* p = reinterpret_cast<const float*>(base) + idx;
        if (vec && valid >= 8) {
            const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < valid ? p[i] : 0.0f;
        }
    }
}

template <int KIND>
__global__ void __launch_bounds__(THREADS) quantize_kernel(QuantArgs g) {
    __shared__ __align__(16) uint8_t sc[2 * TILE_BYTES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const long long col = (long long)bx * COLS + lane * 8;
    const int valid = (int)max(0LL, min(8LL, g.cols - col));
    reinterpret_cast<uint32_t*>(sc)[threadIdx.x] = 0u;
    __syncthreads();
    grid_wait();
    grid_release();
    const int code_bytes = (valid + 1) >> 1;      // an odd last column leaves a zero in the high nibble
    const bool any = row0 + warp * ROWS_PER_WARP < g.rows;
#pragma unroll 4
    for (int i = 0; any && i < ROWS_PER_WARP; ++i) {
        const int r = warp * ROWS_PER_WARP + i;
        const long long row = row0 + r;
        const bool live = row < g.rows;
        float v[8];
        load8<KIND>(g.x, live ? row * g.ldx + col : 0, live ? valid : 0, g.vec != 0, v);
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const uint32_t s = scale_code(top);
        const float inv = inverse_scale(s == 255u ? 0u : s);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= inv;
        const uint32_t w = s == 255u ? 0u : pack_e2m1(v);
        if (live && valid > 0) {
            uint8_t* dst = g.codes + row * g.ldc_bytes + (col >> 1);
            if (valid == 8) *reinterpret_cast<uint32_t*>(dst) = w;
            else for (int k = 0; k < code_bytes; ++k) dst[k] = (uint8_t)(w >> (8 * k));
            if ((lane & 3) == 0) {
                const int b = lane >> 2;          // block within the CTA's eight
                sc[(b >> 2) * TILE_BYTES + (r & 31) * 16 + (r >> 5) * 4 + (b & 3)] = (uint8_t)s;
            }
        }
    }
    __syncthreads();
    // 64 pieces of 16 bytes; the second tile exists when the tensor reaches into it
    if (threadIdx.x < 64) {
        const long long tile = (long long)bx * 2 + (threadIdx.x >> 5);
        if (tile < g.across)
            reinterpret_cast<uint4*>(g.scales + ((long long)by * g.across + tile) * TILE_BYTES)[threadIdx.x & 31] =
                reinterpret_cast<const uint4*>(sc)[threadIdx.x];
    }
}

struct DequantArgs {
    const uint8_t* codes; long long ldc_bytes;
    const uint8_t* scales;
    void* y; long long ldy;
    long long rows, cols, across;
    unsigned grid_cols;
    int vec;                         // y can be written in 16-byte pieces
};

template <int KIND>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(DequantArgs g) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const long long col = (long long)bx * COLS + lane * 8;
    const int valid = (int)max(0LL, min(8LL, g.cols - col));
    grid_wait();
    grid_release();
    if (valid == 0) return;
#pragma unroll 4
    for (int i = 0; i < ROWS_PER_WARP; ++i) {
        const long long row = row0 + warp * ROWS_PER_WARP + i;
        if (row >= g.rows) return;
        const uint8_t* src = g.codes + row * g.ldc_bytes + (col >> 1);
        uint32_t w = 0;
        if (valid == 8) w = __ldcs(reinterpret_cast<const uint32_t*>(src));
        else for (int k = 0; k < (valid + 1) >> 1; ++k) w |= (uint32_t)src[k] << (8 * k);
        const float scale = scale_value(__ldg(g.scales + scale_offset(row, col >> 5, g.across)));
        float v[8];
        unpack_e2m1(w, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= scale;
        if (KIND == KIND_BF16) {
            uint16_t* dst = reinterpret_cast<uint16_t*>(g.y) + row * g.ldy + col;
            const uint4 q = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
            if (g.vec && valid == 8) __stcs(reinterpret_cast<uint4*>(dst), q);
            else {
                const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int k = 0; k < 8; ++k) if (k < valid) dst[k] = (uint16_t)(p[k >> 1] >> (16 * (k & 1)));
            }
        } else {
            float* dst = reinterpret_cast<float*>(g.y) + row * g.ldy + col;
            if (g.vec && valid == 8) {
                __stcs(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
                __stcs(reinterpret_cast<float4*>(dst) + 1, make_float4(v[4], v[5], v[6], v[7]));
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) if (k < valid) dst[k] = v[k];
            }
        }
    }
}

bool grid_of(long long rows, long long cols, unsigned& grid, unsigned& grid_cols) {
    const long long gx = (cols - 1) / COLS + 1, gy = (rows - 1) / ROWS + 1;
    if (gx > 2147483647LL / gy) return false;
    grid = (unsigned)(gx * gy);
    grid_cols = (unsigned)gx;
    return true;
}

}  // namespace

int a4c_launch_quantize_mx(const void* x, int kind, long long ldx, uint8_t* codes, long long ldc, uint8_t* scales,
                           long long rows, long long cols, cudaStream_t stream) {
    unsigned grid;
    QuantArgs g;
    if (!grid_of(rows, cols, grid, g.grid_cols)) return A4C_ERR_TOO_LARGE;
    const int esz = kind == KIND_BF16 ? 2 : 4;
    g.x = x; g.ldx = ldx; g.codes = codes; g.ldc_bytes = ldc / 2; g.scales = scales; g.rows = rows; g.cols = cols;
    g.across = tiles_across(cols);
    g.vec = ((uintptr_t)x & 15u) == 0 && (ldx * esz) % 16 == 0;
    const cudaError_t e = launch_serialized(kind == KIND_BF16 ? quantize_kernel<KIND_BF16> : quantize_kernel<KIND_F32>, grid, THREADS, 0, 0, stream, g);
    return e == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}

int a4c_launch_dequantize_mx(const uint8_t* codes, long long ldc, const uint8_t* scales, void* y, int kind, long long ldy,
                             long long rows, long long cols, cudaStream_t stream) {
    unsigned grid;
    DequantArgs g;
    if (!grid_of(rows, cols, grid, g.grid_cols)) return A4C_ERR_TOO_LARGE;
    const int esz = kind == KIND_BF16 ? 2 : 4;
    g.codes = codes; g.ldc_bytes = ldc / 2; g.scales = scales; g.y = y; g.ldy = ldy; g.rows = rows; g.cols = cols;
    g.across = tiles_across(cols);
    g.vec = ((uintptr_t)y & 15u) == 0 && (ldy * esz) % 16 == 0;
    const cudaError_t e = launch_serialized(kind == KIND_BF16 ? dequantize_kernel<KIND_BF16> : dequantize_kernel<KIND_F32>, grid, THREADS, 0, 0, stream, g);
    return e == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}
