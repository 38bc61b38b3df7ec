// Quantisation to and from MXFP4.
//
//   s[r,b]    = max(floor(log2(max |x| over the block)) + 127 - 2, 0), or 255 when the block holds a NaN or an infinity
//   code[r,c] = E2M1(x[r,c] * 2^(127 - s)), nearest even, saturating at 6;     y[r,c] = E2M1 value * 2^(s - 127)
//
// Bound by HBM: one pass, 2 (bfloat16) or 4 (float32) bytes an element on one side and 17/32 byte on the other; next to it by
// issue slots, so the work per row is shared out as widely as the block allows.  A lane takes sixteen neighbouring columns (a
// block is two lanes, its maximum one shuffle), half a warp 256 columns of a row.  A CTA takes 128 rows x 256 columns: exactly
// two scale tiles, which it gathers in shared memory and writes out whole (places beyond the tensor as 0), because single scale
// bytes 16 bytes apart would touch every 32-byte sector of the scale array many times.  Where that leaves SMs idle a CTA takes
// 32 rows, a quarter of each tile: a word in 16 bytes.
//
// Measured: 65536 x 4096 bfloat16 104 us there and 108 us back (6.5 and 6.3 TB/s), 65536 x 256 there 7.4 us, one row 1.4 us.
#include <type_traits>

#include "a4c_common.cuh"
#include "a4c_kernels.h"
#include "mx_common.cuh"

namespace {

using namespace mx;

constexpr int COLS = 256;            // columns per CTA
constexpr int PER_LANE = 16;
constexpr int THREADS = 256;
constexpr int PASS = THREADS / 16;   // rows the CTA has under way at once

struct QuantArgs {
    const void* x; long long ldx;
    uint8_t* codes; long long ldc_bytes;
    uint8_t* scales;
    long long rows, cols, across;
    unsigned grid_cols;              // CTAs across the columns
    int vec;                         // x can be read in 16-byte pieces
};

// Sixteen neighbouring values as they lie in memory; those beyond `valid` read as zero
template <int KIND> struct Raw { static constexpr int words = KIND == KIND_BF16 ? 8 : 16; uint32_t w[words]; };

template <int KIND>
__device__ __forceinline__ Raw<KIND> load16(const uint8_t* src, int valid, bool vec) {
    Raw<KIND> r;
    if (vec && valid == PER_LANE) {
#pragma unroll
        for (int i = 0; i < r.words / 4; ++i) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(src) + i);
            r.w[4 * i] = q.x; r.w[4 * i + 1] = q.y; r.w[4 * i + 2] = q.z; r.w[4 * i + 3] = q.w;
        }
    } else if (KIND == KIND_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int i = 0; i < r.words; ++i)
            r.w[i] = (2 * i < valid ? (uint32_t)p[2 * i] : 0u) | (2 * i + 1 < valid ? (uint32_t)p[2 * i + 1] << 16 : 0u);
    } else {
#pragma unroll
        for (int i = 0; i < r.words; ++i) r.w[i] = i < valid ? reinterpret_cast<const uint32_t*>(src)[i] : 0u;
    }
    return r;
}

// Largest magnitude: float bits whose order is that of the magnitudes, NaN above infinity above the rest
template <int KIND>
__device__ __forceinline__ uint32_t abs_max(const Raw<KIND>& r) {
    if (KIND == KIND_BF16) {             // two at a time; a NaN stays one
        uint32_t m = r.w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < r.words; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(r.w[i] & 0x7FFF7FFFu));
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(m >> 16));
        return m << 16;
    }
    uint32_t m = r.w[0] & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < r.words; ++i) m = max(m, r.w[i] & 0x7FFFFFFFu);
    return m;
}

// values 8 h .. 8 h + 7, scaled, as codes
template <int KIND>
__device__ __forceinline__ uint32_t codes_of(const Raw<KIND>& r, int h, f2 inv) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f2 p = KIND == KIND_BF16 ? pack2(__uint_as_float(r.w[(4 * h + k) % r.words] << 16), __uint_as_float(r.w[(4 * h + k) % r.words] & 0xFFFF0000u))
                                       : pack2(__uint_as_float(r.w[(8 * h + 2 * k) % r.words]), __uint_as_float(r.w[(8 * h + 2 * k + 1) % r.words]));
        unpack2(mul2(p, inv), v[2 * k], v[2 * k + 1]);
    }
    return pack_e2m1(v);
}

// QUARTERS x 32 rows per CTA: 4 (whole scale tiles) or 1
template <int KIND, int QUARTERS>
__global__ void __launch_bounds__(THREADS) quantize_kernel(QuantArgs g) {
    constexpr int ROWS = QUARTERS * 32, ESZ = KIND == KIND_BF16 ? 2 : 4;
    constexpr int BATCH = KIND == KIND_BF16 && QUARTERS == 4 ? 4 : 2;   // rows loaded before any is converted (the stores between would hold them back)
    __shared__ __align__(16) uint8_t sc[2 * TILE_BYTES / 4 * QUARTERS];   // [tile][row % 32][quarter][block]
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const long long col = (long long)bx * COLS + l16 * PER_LANE;
    const int valid = (int)max(0LL, min((long long)PER_LANE, g.cols - col));
    const int code_bytes = (valid + 1) >> 1;      // an odd last column leaves a zero in the high nibble
    const int count = (int)max(0LL, min((long long)ROWS, g.rows - row0));
    const bool whole = count == ROWS && (long long)bx * COLS + COLS <= g.cols;
    if (!whole && threadIdx.x < 64 * QUARTERS) reinterpret_cast<uint32_t*>(sc)[threadIdx.x] = 0u;
    __syncthreads();
    grid_wait();
    grid_release();
    const uint8_t* src = reinterpret_cast<const uint8_t*>(g.x) + ((row0 + r0) * g.ldx + col) * ESZ;
    const long long src_step = (long long)PASS * g.ldx * ESZ;
    uint8_t* dst = g.codes + (row0 + r0) * g.ldc_bytes + (col >> 1);
    const long long dst_step = (long long)PASS * g.ldc_bytes;
    const int b = l16 >> 1;                       // block within the CTA's eight
    uint8_t* my_sc = sc + (b >> 2) * 128 * QUARTERS + (b & 3);
    // one row's sixteen values -> codes and, from the even lane, the scale; `inside`: nothing of the CTA lies beyond the tensor
    auto convert = [&](const Raw<KIND>& raw, int r, auto inside, bool live) {
        uint32_t top = abs_max(raw);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        const uint32_t s = scale_code(top);
        const f2 inv = both(inverse_scale(s == 255u ? 0u : s));
        uint2 w = make_uint2(codes_of(raw, 0, inv), codes_of(raw, 1, inv));
        if (s == 255u) w = make_uint2(0u, 0u);
        if (!live) return;
        if (inside.value || valid == PER_LANE) *reinterpret_cast<uint2*>(dst) = w;
        else for (int k = 0; k < code_bytes; ++k) dst[k] = (uint8_t)((k < 4 ? w.x : w.y) >> (8 * (k & 3)));
        if ((l16 & 1) == 0 && (inside.value || valid > 0)) my_sc[((r & 31) * QUARTERS + (r >> 5)) * 4] = (uint8_t)s;
    };
    if (whole && g.vec) {
#pragma unroll 1
        for (int r = r0; r < ROWS; r += BATCH * PASS) {
            Raw<KIND> raw[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j, src += src_step) raw[j] = load16<KIND>(src, PER_LANE, true);
#pragma unroll
            for (int j = 0; j < BATCH; ++j, dst += dst_step) convert(raw[j], r + j * PASS, std::true_type{}, true);
        }
    } else {
#pragma unroll 1
        for (int r = r0; r - r0 < count; r += PASS, src += src_step, dst += dst_step)      // the same trips for both halves of a warp
            convert(load16<KIND>(src, r < count ? valid : 0, g.vec != 0), r, std::false_type{}, r < count);
    }
    __syncthreads();
    // a thread per tile and row % 32; the second tile exists when the tensor reaches into it
    if (threadIdx.x < 64) {
        const long long tile = (long long)bx * 2 + (threadIdx.x >> 5);
        if (tile < g.across) {
            uint8_t* out = g.scales + ((row0 / TILE_ROWS) * g.across + tile) * TILE_BYTES + (threadIdx.x & 31) * 16;
            if (QUARTERS == 4) *reinterpret_cast<uint4*>(out) = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
            else reinterpret_cast<uint32_t*>(out)[by & 3] = reinterpret_cast<const uint32_t*>(sc)[threadIdx.x];
        }
    }
}

struct DequantArgs {
    const uint8_t* codes; long long ldc_bytes;
    const uint8_t* scales;
    void* y; long long ldy;
    long long rows, cols, across;
    unsigned grid_cols;
    int vec;                         // y can be written in 32-byte pieces
};

__device__ __forceinline__ void store32_bytes(void* dst, const uint32_t* w) {
    asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

template <int KIND, int QUARTERS>
__global__ void __launch_bounds__(THREADS) dequantize_kernel(DequantArgs g) {
    constexpr int ROWS = QUARTERS * 32, ESZ = KIND == KIND_BF16 ? 2 : 4, BATCH = QUARTERS == 4 ? 4 : 2;
    const unsigned by = blockIdx.x / g.grid_cols, bx = blockIdx.x - by * g.grid_cols;
    const long long row0 = (long long)by * ROWS;
    const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    const long long col = (long long)bx * COLS + l16 * PER_LANE;
    const int valid = (int)max(0LL, min((long long)PER_LANE, g.cols - col));
    grid_wait();
    grid_release();
    if (valid == 0) return;
    const int count = (int)max(0LL, min((long long)ROWS, g.rows - row0));
    const uint8_t* src = g.codes + (row0 + r0) * g.ldc_bytes + (col >> 1);
    const long long src_step = (long long)PASS * g.ldc_bytes;
    uint8_t* dst = reinterpret_cast<uint8_t*>(g.y) + ((row0 + r0) * g.ldy + col) * ESZ;
    const long long dst_step = (long long)PASS * g.ldy * ESZ;
    const uint8_t* scales = g.scales + scale_offset(row0, col >> 5, g.across);     // row0 is a multiple of 32
    for (int r = r0; r < count; r += BATCH * PASS) {
        uint2 code[BATCH];
        uint8_t sc[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j, src += src_step) {
            const int rr = r + j * PASS;
            code[j] = make_uint2(0u, 0u);
            sc[j] = 0;
            if (rr >= count) continue;
            if (valid == PER_LANE) code[j] = __ldcs(reinterpret_cast<const uint2*>(src));
            else
                for (int k = 0; k < (valid + 1) >> 1; ++k) (k < 4 ? code[j].x : code[j].y) |= (uint32_t)src[k] << (8 * (k & 3));
            sc[j] = __ldg(scales + (rr & 31) * 16 + (rr >> 5) * 4);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j, dst += dst_step) {
            if (r + j * PASS >= count) break;
            const f2 scale = both(scale_value(sc[j]));
            uint32_t w[4 * ESZ];                           // sixteen values
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                unpack_e2m1(h == 0 ? code[j].x : code[j].y, v);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float lo, hi;
                    unpack2(mul2(pack2(v[2 * k], v[2 * k + 1]), scale), lo, hi);
                    if (KIND == KIND_BF16) w[4 * h + k] = pack_bf16x2(lo, hi);
                    else { w[(8 * h + 2 * k) % (4 * ESZ)] = __float_as_uint(lo); w[(8 * h + 2 * k + 1) % (4 * ESZ)] = __float_as_uint(hi); }
                }
            }
            if (g.vec && valid == PER_LANE) {              // whole sectors: 16-byte stores would each fill half of one
                store32_bytes(dst, w);
                if (KIND == KIND_F32) store32_bytes(dst + 32, w + (KIND == KIND_F32 ? 8 : 0));
            } else if (KIND == KIND_BF16) {
#pragma unroll
                for (int k = 0; k < PER_LANE; ++k) if (k < valid) reinterpret_cast<uint16_t*>(dst)[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
            } else {
#pragma unroll
                for (int k = 0; k < PER_LANE; ++k) if (k < valid) reinterpret_cast<uint32_t*>(dst)[k] = w[k % (4 * ESZ)];
            }
        }
    }
}

// CTAs of `quarters` x 32 rows; rows of the last scale tile beyond the tensor belong to somebody too
bool grid_of(long long rows, long long cols, int& quarters, unsigned& grid, unsigned& grid_cols) {
    const long long gx = (cols - 1) / COLS + 1, gy = (rows - 1) / TILE_ROWS + 1;
    if (gx > 2147483647LL / gy) return false;
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    quarters = gx * gy < 8LL * sms ? 1 : 4;
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
    g.vec = ((uintptr_t)y & 31u) == 0 && (ldy * esz) % 32 == 0;
    const cudaError_t e = kind == KIND_BF16 ? launch_dequantize<KIND_BF16>(g, quarters, grid, stream) : launch_dequantize<KIND_F32>(g, quarters, grid, stream);
    return e == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}
