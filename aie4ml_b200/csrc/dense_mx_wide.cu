// Dense and gated Dense over MXFP4 operands with many rows: a CTA pair (tcgen05 cta_group::2) per 256-row tile.
// Same arithmetic as dense_mx.cu.
//
//   Dense: a tile is 256 rows x 256 features.  Gated: 256 rows x 128 features of both projections, the gate's 128 in
//   accumulator columns 0-127 and the other's in 128-255, so that one thread holds both factors of an output.
//
// kind::mxf4 finishes a 256 x 256 x 256 step in 512 cycles; a single CTA on 128 x 256 would have to take in 48 KB of codes
// in that time, the pair takes 32 KB per CTA: its own 128 rows of A and half of the weight rows (for the gated Dense one
// CTA fetches the gate's rows, the other one the second projection's).  Scales go along as 2-tile boxes of a tensor map:
// each CTA its own A rows', both CTAs all 256 weight rows'.
//
// Tensor memory: two accumulators of 256 columns and the scales of two stages (48 columns) are more than 512 columns, so the
// accumulators overlap by 48 columns.  The epilogue first moves those to shared memory and says so on a barrier of its own;
// the next tile's MMAs wait for that and not for the tile's arithmetic.
//
// The scale copies (tcgen05.cp) go down the tensor pipe with the MMAs, which takes both in issue order, so they need no barrier
// when one thread issues both (from a warp of their own, with barriers, a stage took 806 cycles; from here 670).  That thread is
// an elected lane of a converged warp: in a loop under `if (lane == 0)` every descriptor is first moved to a uniform register,
// and the MMAs of a stage took 940 cycles to issue, longer than the 512 they run.
//
// Warps: 0 TMA producer, 1 MMA issuer (leader CTA), 2-17 epilogue: two groups of four warps per
// accumulator, each half of the columns, so that two tiles are converted at once.  A lane holds one row, so an MXFP4 output block
// is 32 values of one thread; rows go out through a swizzled patch of shared memory per warp and TMA stores (directly from
// registers every 16 bytes of a row were an L2 request of their own).  Every wait is bounded.
//
// Bound by the tensor pipe under the power cap: Dense 16384 x 8192 x 8192 440 us, gated 16384 x 4096 x 2*8192 450 us (5.0 and
// 4.9 PFLOP/s); at short reductions by the epilogue's issue slots: gated 65536 x 256 x 2*1024 29 us without activation, 48 us with GELU,
// 56 us to MXFP4, 70 us with both biases (a lane's row needs every column's bias: 16 bytes a lane and four columns, which
// shared memory returns at 128 bytes a cycle).
#include <cuda.h>

#include "a4c_common.cuh"
#include "a4c_kernels.h"
#include "mx_common.cuh"

namespace {

using namespace tc;

constexpr int BM = 256, BM_CTA = 128;
constexpr int BN = 256, BN_CTA = 128;         // weight rows per tile / staged per CTA
constexpr int BK = 256;
constexpr int CODE_BYTES = 128 * BK / 2;      // 128 rows of a stage's codes
constexpr int SF_BYTES = 2 * mx::TILE_BYTES;  // and of its scales
constexpr int STAGE_BYTES = 2 * CODE_BYTES + 3 * SF_BYTES;
constexpr int STAGES = 4;
constexpr int SF_COLS = 24;                   // A 8, weights 16
constexpr int SF_SETS = 2;
// What an instantiation is for: Dense, the gated Dense of one activation (ACT_*), or of the others (told by the arguments).  A switch
// for every 16 columns keeps their arithmetic from overlapping the next columns' loads: gated 65536 x 256 x 2*1024 took
// 51.0 us with it and 47.3 without (GELU to bf16), 55.4 and 50.7 (SiLU to MXFP4).
constexpr int DENSE = -1, GATED_OTHER = -2;
constexpr int TMEM_COLS = 512;
constexpr int SF0 = TMEM_COLS - SF_SETS * SF_COLS;
constexpr int ACC1 = SF0 - BN;                // second accumulator: columns ACC1 .. SF0
constexpr int OVERLAP = BN - ACC1;
constexpr int EPI_WARPS = 16;
constexpr int EPI_WARP0 = 2;                   // first epilogue warp
constexpr int NUM_THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
constexpr int PATCH_BYTES = 32 * 64;            // per epilogue warp: 32 rows of a TMA store's box
constexpr int STASH_BYTES = OVERLAP * 128 * 4;  // per accumulator: the shared columns of this CTA's rows

struct Tail {
    float bias[4][2][128];           // per epilogue group, alternating between tiles: its columns' bias (gated: gate, then the other's)
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint64_t overlap_free[2];
    uint32_t tmem_base;
    volatile int abort_flag;
};
constexpr size_t SMEM_BYTES = 1024 + (size_t)STAGES * STAGE_BYTES + EPI_WARPS * PATCH_BYTES + 2 * STASH_BYTES + sizeof(Tail);

struct Args {
    const float* bias[2];
    void* Y; long long ldy;
    uint8_t* ys; long long y_across;
    long long M;
    int K, N;
    int num_kb;
    int num_m_tiles, num_n_tiles;
    int panel;                       // column tiles per panel of the tile order
    int act;
    int tma_store;                   // the output's base and pitch are multiples of 16 bytes
    uint32_t idesc;
    int* status;
};

// The tiles of one pair, in order: column tile fastest inside a panel of weights that stays in the L2 while the row tiles stream
// past.  With one panel the next tile's place follows by additions (two integer divisions a tile are a fifth of what a warp
// of the epilogue issues for it at short reductions).
struct Tiles {
    int tile, mt, nt, step, step_m, step_n;
    __device__ __forceinline__ Tiles(const Args& g, int pair, int num_pairs) : tile(pair), mt(0), nt(0), step(num_pairs) {
        step_m = num_pairs / g.num_n_tiles;
        step_n = num_pairs - step_m * g.num_n_tiles;
        locate(g);
    }
    __device__ __forceinline__ void locate(const Args& g) {
        if (tile >= g.num_m_tiles * g.num_n_tiles) return;      // beyond the last one there is no panel to divide by
        const int per_panel = g.num_m_tiles * g.panel;
        const int pz = tile / per_panel, rem = tile - pz * per_panel;
        const int width = min(g.panel, g.num_n_tiles - pz * g.panel);
        mt = rem / width;
        nt = pz * g.panel + (rem - mt * width);
    }
    __device__ __forceinline__ void next(const Args& g) {
        tile += step;
        if (g.panel < g.num_n_tiles) { locate(g); return; }
        mt += step_m;
        nt += step_n;
        if (nt >= g.num_n_tiles) { nt -= g.num_n_tiles; ++mt; }
    }
};

// 32 finished neighbouring values of one row (as pairs) -> words of the output type (16 bf16, 32 f32, 4 MXFP4) and its scale
template <int OUT>
__device__ __forceinline__ uint32_t to_words(const mx::f2* p, uint32_t* w) {
    float v[32];
#pragma unroll
    for (int i = 0; i < 16; ++i) mx::unpack2(p[i], v[2 * i], v[2 * i + 1]);
    if (OUT == mx::KIND_BF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = mx::pack_bf16x2(v[2 * i], v[2 * i + 1]);
        return 0;
    }
    if (OUT == mx::KIND_F32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
        return 0;
    }
    return mx::quantize32(v, w);
}

template <int OUT> struct Words { static constexpr int value = OUT == mx::KIND_BF16 ? 16 : OUT == mx::KIND_F32 ? 32 : 4; };

// straight from registers: for outputs that a tensor map cannot describe, and for boxes that reach beyond the row's end (a TMA
// store there wrote up to the next 16 bytes of the row)
template <int OUT>
__device__ __forceinline__ void store_direct(const Args& g, long long row, int col, const uint32_t* w) {
    const int left = g.N - col;
    if (OUT == mx::KIND_BF16) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(g.Y) + row * g.ldy + col;
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i < left) dst[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    } else if (OUT == mx::KIND_F32) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(g.Y) + row * g.ldy + col;
#pragma unroll
        for (int i = 0; i < 32; ++i) if (i < left) dst[i] = w[i];
    } else {
        uint8_t* dst = reinterpret_cast<uint8_t*>(g.Y) + (row * g.ldy + col) / 2;
        const int bytes = (left + 1) >> 1;
        if (left >= 32) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else {
#pragma unroll
            for (int b = 0; b < 16; ++b) if (b < bytes) dst[b] = (uint8_t)(w[b >> 2] >> (8 * (b & 3)));
        }
    }
}

__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t* a) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]),
          "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15])
        : "r"(taddr));
}
// waits for the loads issued so far; the registers pass through, so no use of them is scheduled ahead
__device__ __forceinline__ void tmem_ld_wait16(uint32_t* a) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                   "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15])
                 :: "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 :: "l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

__device__ __forceinline__ void cp_async4_or_zero(void* dst, const void* src, bool any) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(smem_u32(dst)), "l"(src), "r"(any ? 4 : 0) : "memory");
}

template <int ACT>
__device__ __forceinline__ void activate8(mx::f2* v) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = mx::activate2<ACT>(v[k]);
}

// adds 16 neighbouring columns' bias, which lies in shared memory
__device__ __forceinline__ void add_bias(mx::f2* v, const float* bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 b = reinterpret_cast<const float4*>(bias)[i];
        v[2 * i] = mx::add2(v[2 * i], mx::pack2(b.x, b.y));
        v[2 * i + 1] = mx::add2(v[2 * i + 1], mx::pack2(b.z, b.w));
    }
}

// 32 finished neighbouring values of each lane's row, `half` 0 and then 1 of 64 -> output and, for MXFP4, the two scales of the
// 64; a block that lies beyond the row's end gets scale 0
template <int OUT>
__device__ __forceinline__ void store32(const Args& g, const CUtensorMap* map_y, uint8_t* patch, long long row0, int lane, int col, int half,
                                        uint32_t& scales, mx::f2* v) {
    const long long row = row0 + lane;
    constexpr int WORDS = Words<OUT>::value;
    constexpr int BOX = OUT == mx::KIND_F32 ? 16 : OUT == mx::KIND_BF16 ? 32 : 64;     // columns per TMA store: 64 bytes, or 32 of MXFP4
    const int col64 = col - 32 * half;
    const bool boxed = g.tma_store && (OUT == mx::KIND_MX ? col64 + 64 : col + 32) <= g.N;
    if (OUT == mx::KIND_MX && col + 32 > g.N) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (col + 2 * i >= g.N) v[i] = 0;
            else if (col + 2 * i + 1 >= g.N) v[i] &= 0xFFFFFFFFull;
        }
    }
    uint32_t w[WORDS];
    scales = half == 0 ? to_words<OUT>(v, w) : scales | to_words<OUT>(v, w) << 8;
    if (OUT == mx::KIND_MX && half && row < g.M && (col64 >> 5) < (int)g.y_across * mx::TILE_BLOCKS)
        *reinterpret_cast<uint16_t*>(g.ys + mx::scale_offset(row, col64 >> 5, g.y_across)) = (uint16_t)scales;
    if (!boxed) {
        if (row < g.M && col < g.N) store_direct<OUT>(g, row, col, w);
        return;
    }
#pragma unroll
    for (int q = 0; q < 32 / (BOX > 32 ? 32 : BOX); ++q) {
        if (OUT != mx::KIND_MX || half == 0) {             // the patch's last store has been read
            if (lane == 0) tma_store_wait_read();
            __syncwarp();
        }
        if (OUT == mx::KIND_MX) {
            *reinterpret_cast<uint4*>(patch + lane * 32 + half * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)                    // 64-byte swizzle: 16-byte piece p of row r at p ^ (r / 2 & 3)
                *reinterpret_cast<uint4*>(patch + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(w[(16 * q + 4 * i) % WORDS], w[(16 * q + 4 * i + 1) % WORDS], w[(16 * q + 4 * i + 2) % WORDS], w[(16 * q + 4 * i + 3) % WORDS]);
        }
        if (OUT != mx::KIND_MX || half == 1) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(map_y, patch, OUT == mx::KIND_MX ? col64 / 2 : col + BOX * q, (int)row0);
        }
    }
}

template <int MODE, int OUT, bool BIAS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
dense_mx_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_sa,
                     const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ CUtensorMap map_su,
                     const __grid_constant__ CUtensorMap map_y, Args g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);      // by an offset: a pointer made from an integer is no longer known to be shared memory
    uint8_t* patches = smem + (size_t)STAGES * STAGE_BYTES;
    Tail* tail = reinterpret_cast<Tail*>(patches + EPI_WARPS * PATCH_BYTES + 2 * STASH_BYTES);
    constexpr bool GATED = MODE != DENSE;
    constexpr int OUT_COLS = GATED ? 128 : 256;       // output features per tile

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = mx::cluster_rank();
    const bool leader = rank == 0;
    const int num_tiles = g.num_m_tiles * g.num_n_tiles;
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&tail->full[s], 1); mbar_init(&tail->empty[s], 1); }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tail->tmem_full[a], 1);
            mbar_init(&tail->tmem_empty[a], EPI_WARPS);         // two groups of each CTA
            mbar_init(&tail->overlap_free[a], EPI_WARPS / 2);   // one
        }
        tail->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&tail->tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    mx::cluster_sync_all();
    tc_fence_after();
    mx::grid_wait();
    mx::grid_release();
    const uint32_t tmem_base = tail->tmem_base;
    volatile int* abort_flag = &tail->abort_flag;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (Tiles t(g, pair, num_pairs); ok && t.tile < num_tiles; t.next(g)) {
                const int m0 = t.mt * BM + (int)rank * BM_CTA;
                const int n0 = t.nt * OUT_COLS;
                const CUtensorMap* mw = GATED && rank ? &map_u : &map_w;
                const int nw = GATED ? n0 : n0 + (int)rank * BN_CTA;
                const int gw = n0 / mx::TILE_ROWS;
                for (int kb = 0; kb < g.num_kb; ++kb) {
                    ok = mbar_wait(&tail->empty[stage], phase ^ 1u, abort_flag, g.status, 161);
                    if (!ok) break;
                    uint8_t* s = smem + (size_t)stage * STAGE_BYTES;
                    uint8_t* f = s + 2 * CODE_BYTES;
                    const uint32_t bar = mx::map_to_cta(smem_u32(&tail->full[stage]), 0);
                    if (leader) mbar_arrive_expect_tx(&tail->full[stage], 2 * STAGE_BYTES);
                    mx::tma_load_2d_pair(s, &map_a, bar, kb * (BK / 2), m0);
                    mx::tma_load_2d_pair(s + CODE_BYTES, mw, bar, kb * (BK / 2), nw);
                    mx::tma_load_3d_pair(f, &map_sa, bar, 0, 2 * kb, m0 / mx::TILE_ROWS);
                    mx::tma_load_3d_pair(f + SF_BYTES, &map_sw, bar, 0, 2 * kb, gw);
                    mx::tma_load_3d_pair(f + 2 * SF_BYTES, GATED ? &map_su : &map_sw, bar, 0, 2 * kb, GATED ? gw : gw + 1);
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (leader) {
            int stage = 0, it = 0, step = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < num_tiles; tile += num_pairs, ++it) {
                const int acc = it & 1;
                const uint32_t d_tmem = tmem_base + (uint32_t)(acc ? ACC1 : 0);
                for (int kb = 0; kb < g.num_kb; ++kb, ++step) {
                    ok = mbar_wait(&tail->full[stage], phase, abort_flag, g.status, 164);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t s = smem_u32(smem) + (uint32_t)(stage * STAGE_BYTES);
                    const int steps = min(4, (g.K - kb * BK + 63) / 64);
                    const uint32_t sf = tmem_base + (uint32_t)(SF0 + (step % SF_SETS) * SF_COLS);
                    const uint64_t adesc = make_smem_desc(s), bdesc = make_smem_desc(s + CODE_BYTES);
                    // columns of a set: A tile 0, A tile 1, weights tile 0 (8 columns: 256 rows), weights tile 1
                    const uint64_t fdesc = mx::make_scale_desc(s + 2 * CODE_BYTES);
                    if (mx::elect_one()) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (steps <= 2 * h) break;
                            const uint64_t t = fdesc + (uint64_t)(h * (mx::TILE_BYTES >> 4));
                            mx::copy_scales_pair(sf + (uint32_t)(h * 4), t);
                            mx::copy_scales_pair(sf + (uint32_t)(8 + h * 8), t + (uint64_t)(SF_BYTES >> 4));
                            mx::copy_scales_pair(sf + (uint32_t)(12 + h * 8), t + (uint64_t)(2 * SF_BYTES >> 4));
                        }
                    }
                    __syncwarp();
                    if (kb == 0) {               // the tile's first scales are on their way while the epilogue frees the accumulator
                        ok = mbar_wait(&tail->tmem_empty[acc], ((it >> 1) & 1) ^ 1u, abort_flag, g.status, 162) &&
                             (it == 0 || mbar_wait(&tail->overlap_free[acc ^ 1], ((it - 1) >> 1) & 1, abort_flag, g.status, 163));
                        if (!ok) break;
                        tc_fence_after();
                    }
                    if (mx::elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (k >= steps) break;
                            mx::umma_pair(d_tmem, adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), g.idesc | mx::sf_bits(k & 1),
                                          sf + (uint32_t)((k >> 1) * 4), sf + (uint32_t)(8 + (k >> 1) * 8), (uint32_t)((kb | k) != 0));
                        }
                        mx::commit_both(smem_u32(&tail->empty[stage]));
                        if (kb + 1 == g.num_kb) mx::commit_both(smem_u32(&tail->tmem_full[acc]));
                    }
                    __syncwarp();
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else {
        const int quad = warp & 3;
        const int acc = (warp - EPI_WARP0) >> 3, half = ((warp - EPI_WARP0) >> 2) & 1;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc ? ACC1 : 0);
        constexpr int COLS = GATED ? 64 : 128;                 // output columns per group
        uint8_t* patch = patches + (warp - EPI_WARP0) * PATCH_BYTES;
        // The columns that the accumulators share: the last of accumulator 0 (second half; gated: of the other factor), the first of
        // accumulator 1 (first half; gated: of the gate).  Their group has them in `stash`, every thread its own row's.
        const bool holder = half == 1 - acc;
        const int shared0 = acc ? 0 : BN - OVERLAP;            // first shared column of the accumulator
        // (16-byte piece p of row r at p ^ (r / 2 & 3): rows are 12 pieces apart, so eight lanes then meet eight different bank groups)
        uint8_t* stash = patches + EPI_WARPS * PATCH_BYTES + acc * STASH_BYTES + (quad * 32 + lane) * (OVERLAP * 4);
        const uint32_t swz = (uint32_t)(lane >> 1) & 3u;
        static_assert(OVERLAP % 16 == 0 && OVERLAP <= COLS, "the shared columns are whole pieces of one group");
        auto release = [&](uint64_t* bar) {                    // this warp has read its part
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mx::mbar_arrive_cluster(mx::map_to_cta(smem_u32(bar), 0));
        };
        // 16 columns of the accumulator, from `c` on, of this thread's row
        auto take = [&](int c, uint32_t* r) {
            if (holder && (acc ? c < OVERLAP : c >= BN - OVERLAP)) {
                const uint8_t* at = stash + (c - shared0) * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 q = *reinterpret_cast<const uint4*>(at + ((i ^ swz) << 4));
                    r[4 * i] = q.x; r[4 * i + 1] = q.y; r[4 * i + 2] = q.z; r[4 * i + 3] = q.w;
                }
            } else {
                tmem_ld16_async(taddr + (uint32_t)c, r);
            }
        };
        uint32_t scales = 0;
        bool ok = true;
        Tiles t(g, pair + acc * num_pairs, 2 * num_pairs);
        // the bias of a tile's columns is on its way while the group converts the tile before (fetched at the tile's start it cost
        // a gated 65536 x 256 x 2*1024 5.6 us)
        auto fetch_bias = [&](int j) {
            const int i = quad * 32 + lane, n = t.nt * OUT_COLS + half * COLS + (GATED ? i & 63 : i);
            const float* src = GATED && i >= 64 ? g.bias[1] : g.bias[0];
            const bool any = src != nullptr && n < g.N;
            cp_async4_or_zero(&tail->bias[2 * acc + half][j & 1][i], any ? src + n : g.bias[0] ? g.bias[0] : g.bias[1], any);
        };
        if (BIAS && t.tile < num_tiles) fetch_bias(0);
        for (int j = 0; t.tile < num_tiles; ++j) {
            const int nt = t.nt;
            const long long row0 = (long long)t.mt * BM + (int)rank * BM_CTA + quad * 32;
            const float* bias = tail->bias[2 * acc + half][j & 1];
            t.next(g);
            if (BIAS) {
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("bar.sync %0, 128;" :: "r"(1 + 2 * acc + half) : "memory");
                if (t.tile < num_tiles) fetch_bias(j + 1);
            }
            if (ok) ok = mbar_wait(&tail->tmem_full[acc], j & 1, abort_flag, g.status, 165);
            if (!ok) continue;
            tc_fence_after();
            if (holder) {
                uint32_t r[OVERLAP];
#pragma unroll
                for (int i = 0; i < OVERLAP / 16; ++i) tmem_ld16_async(taddr + (uint32_t)(shared0 + 16 * i), r + 16 * i);
#pragma unroll
                for (int i = 0; i < OVERLAP / 16; ++i) tmem_ld_wait16(r + 16 * i);
                release(&tail->overlap_free[acc]);
#pragma unroll
                for (int i = 0; i < OVERLAP / 4; ++i)
                    *reinterpret_cast<uint4*>(stash + (i >> 2) * 64 + (((i & 3) ^ swz) << 4)) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
            }
#pragma unroll 1
            for (int p = 0; p < COLS / 32; ++p) {              // 32 outputs at a time
                const int c = half * COLS + 32 * p, col = nt * OUT_COLS + c;
                mx::f2 v[16];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t a[16], u[16];
                    take(c + 16 * q, a);
                    if (GATED) take(128 + c + 16 * q, u);
                    tmem_ld_wait16(a);
                    if (GATED) tmem_ld_wait16(u);
                    if (q == 1 && p == COLS / 32 - 1) release(&tail->tmem_empty[acc]);
                    mx::f2* x = v + 8 * q;
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = mx::pack2(__uint_as_float(a[2 * k]), __uint_as_float(a[2 * k + 1]));
                    if (BIAS) add_bias(x, bias + 32 * p + 16 * q);
                    if (GATED) {
                        mx::f2 y[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = mx::pack2(__uint_as_float(u[2 * k]), __uint_as_float(u[2 * k + 1]));
                        if (BIAS) add_bias(y, bias + 64 + 32 * p + 16 * q);
                        if (MODE != GATED_OTHER) activate8<MODE>(x);
                        else if (g.act == mx::ACT_RELU) activate8<mx::ACT_RELU>(x);
                        else if (g.act == mx::ACT_SIGMOID) activate8<mx::ACT_SIGMOID>(x);
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[k] = mx::mul2(x[k], y[k]);
                    } else if (g.act == mx::ACT_RELU) {
                        activate8<mx::ACT_RELU>(x);
                    }
                }
                if (row0 < g.M) store32<OUT>(g, &map_y, patch, row0, lane, col, p & 1, scales, v);
            }
        }
        if (lane == 0) tma_store_wait_read();      // the patch outlives its last store
    }

    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = a4c_globaltimer();
        while (a4c_globaltimer() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    tc_fence_before();
    mx::cluster_sync_all();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
}

template <int MODE, int OUT, bool BIAS>
cudaError_t launch_one(const CUtensorMap* m, const Args& g, int grid, cudaStream_t s) {
    static tc::SmemOptIn opt_in;
    const cudaError_t e = opt_in.ensure(dense_mx_wide_kernel<MODE, OUT, BIAS>, SMEM_BYTES);
    if (e != cudaSuccess) return e;
    return mx::launch_serialized(dense_mx_wide_kernel<MODE, OUT, BIAS>, (unsigned)grid, NUM_THREADS, SMEM_BYTES, 0, s, m[0], m[1], m[2], m[3], m[4], m[5], m[6], g);
}
template <int MODE, int OUT>
cudaError_t launch_bias(const CUtensorMap* m, const Args& g, int grid, cudaStream_t s) {
    return g.bias[0] || g.bias[1] ? launch_one<MODE, OUT, true>(m, g, grid, s) : launch_one<MODE, OUT, false>(m, g, grid, s);
}
template <int MODE>
cudaError_t launch(int out_kind, const CUtensorMap* m, const Args& g, int grid, cudaStream_t s) {
    return out_kind == mx::KIND_BF16 ? launch_bias<MODE, mx::KIND_BF16>(m, g, grid, s)
           : out_kind == mx::KIND_F32 ? launch_bias<MODE, mx::KIND_F32>(m, g, grid, s) : launch_bias<MODE, mx::KIND_MX>(m, g, grid, s);
}

}  // namespace

// When the pair kernel is the faster one (microseconds on the device, pair kernel / dense_mx.cu; `ctas` are the latter's tiles of
// 128 rows and features):
//   Dense: once those are more than one per SM.  144 of them: 5.5 / 4.0 at K = 256, 6.6 / 5.4 at 1024, 29.9 / 25.7 at 16384;
//   160: 5.8 / 7.3, 6.9 / 9.9, 30.1 / 48.6.
//   Gated: once they are too many to be cut into smaller row tiles (half the SMs).  64: 5.3 / 4.5 at K = 256, 5.6 / 5.2 at 512;
//   80: 5.5 / 5.8, 6.0 / 6.6.  With a reduction long enough to use the pair's faster main loop earlier than that: 64: 6.4 / 6.6 at
//   K = 1024, 16.1 / 19.3 at 8192;  48: 6.3 / 6.5, 16.1 / 19.0;  32: 6.3 / 5.5, 16.0 / 17.4.
// Up to 128 rows half of each 256-row tile would be empty.
bool a4c_dense_mx_wide_wanted(const A4cMxDense& d, int sms) {
    const long long ctas = ((d.M + 127) / 128) * ((d.N + 127) / 128);
    if (d.M <= 128) return false;
    return d.wu == nullptr ? ctas > sms : ctas * 2 > sms || (ctas * 4 > sms && d.K >= 1024);
}

int a4c_launch_dense_mx_wide(const A4cMxDense& d, int sms, int* status_word, cudaStream_t stream) {
    const bool gated = d.wu != nullptr;
    Args g;
    g.bias[0] = d.bias; g.bias[1] = d.bias_u; g.Y = d.y; g.ldy = d.ldy; g.ys = d.ys; g.y_across = mx::tiles_across(d.N);
    g.M = d.M; g.K = d.K; g.N = d.N; g.act = d.act; g.status = status_word;
    g.num_kb = (d.K + BK - 1) / BK;
    const int cols = gated ? 128 : 256;
    const long long mt = (d.M + BM - 1) / BM, nt = (d.N + cols - 1) / cols;
    if (mt * nt > 2147483647LL - 65536) return A4C_ERR_TOO_LARGE;
    g.num_m_tiles = (int)mt; g.num_n_tiles = (int)nt;
    const long long tile_bytes = (long long)BN * g.num_kb * (BK / 2);
    long long panel = (32LL << 20) / tile_bytes;
    g.panel = (int)(panel < 1 ? 1 : (panel > nt ? nt : panel));
    g.idesc = mx::make_idesc(BM, BN);
    CUtensorMap m[7];
    if (!mx::make_code_map(&m[0], d.a, d.M, d.K, d.lda, BM_CTA) || !mx::make_code_map(&m[1], d.w, d.N, d.K, d.ldw, BN_CTA) ||
        !mx::make_scale_map(&m[3], d.sa, d.M, d.K) || !mx::make_scale_map(&m[4], d.sw, d.N, d.K))
        return A4C_ERR_CUDA;
    m[2] = m[1]; m[5] = m[4];
    if (gated && (!mx::make_code_map(&m[2], d.wu, d.N, d.K, d.ldu, BN_CTA) || !mx::make_scale_map(&m[5], d.su, d.N, d.K))) return A4C_ERR_CUDA;
    const int esz = d.out_kind == mx::KIND_BF16 ? 2 : 4;
    g.tma_store = d.out_kind == mx::KIND_MX || (((uintptr_t)d.y & 15u) == 0 && (d.ldy * esz) % 16 == 0);
    m[6] = m[0];
    if (g.tma_store && !mx::make_out_map(&m[6], d.y, d.out_kind, d.M, d.N, d.ldy)) return A4C_ERR_CUDA;
    const long long pairs = mt * nt < sms / 2 ? mt * nt : sms / 2;
    const int grid = (int)pairs * 2;
    const cudaError_t err = !gated ? launch<DENSE>(d.out_kind, m, g, grid, stream)
                            : d.act == mx::ACT_SILU ? launch<mx::ACT_SILU>(d.out_kind, m, g, grid, stream)
                            : d.act == mx::ACT_GELU ? launch<mx::ACT_GELU>(d.out_kind, m, g, grid, stream)
                            : d.act == mx::ACT_GELU_TANH ? launch<mx::ACT_GELU_TANH>(d.out_kind, m, g, grid, stream)
                                                         : launch<GATED_OTHER>(d.out_kind, m, g, grid, stream);
    return err == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}
