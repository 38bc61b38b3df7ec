// Dense and gated Dense over MXFP4 operands for any number of rows: the tile kernel.
//
//   Dense:  Y[m,n] = relu?(sum_k A[m,k] W[n,k] + bias[n])
//   gated:  Y[m,n] = act(sum_k A[m,k] Wg[n,k] + bg[n]) * (sum_k A[m,k] Wu[n,k] + bu[n])
//
// Products of block-scaled E2M1 values on tcgen05.mma kind::mxf4 (the scales are applied inside the instruction),
// float32 accumulators in TMEM, bias, activation and the rounding to the output type (bfloat16, float32, or MXFP4 with
// its scales) in the epilogue.
//
// With few rows the time is the weights' way out of memory, so the weights are the M operand here (128 of them to a
// tile) and the rows of A the N operand (16 to 128): a tile fetches 16 KB of weights for 2 KB of A at 16 rows, where the
// other way round every tile would carry 128 mostly empty rows.  While that leaves SMs idle the row tiles get smaller, down
// to 32 (the weights' second fetch comes from the L2), and then the reduction is split over a cluster of up to 8 CTAs: each
// rank sends its partial sums to the rank that finishes the row (distributed shared memory), which adds them in rank order,
// so the result does not depend on timing and no workspace exists.
//
// One tile per CTA: warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 epilogue.  A stage is 256 values of K: 128-byte swizzled
// rows of codes and the scale tiles, which the issuer copies on to TMEM (tcgen05.cp) ahead of the stage's MMAs; the tensor pipe
// takes both in issue order.
// A CTA runs all of its code once, so unrolled code costs its way out of memory: the epilogue converts 16 rows at a time.
// Every wait is bounded.
//
// Measured: Dense 1 x 4096 x 4096 4.3 us, gated 4 x 4096 x 2*8192 8.1 us (4.4 TB/s of weights), 1 x 8192 x 2*16384 24.7 us (5.8 TB/s),
// Dense 2048 x 4096 x 1024 9.5 us.
#include <cuda.h>

#include "a4c_common.cuh"
#include "a4c_kernels.h"
#include "mx_common.cuh"

namespace {

using namespace tc;

constexpr int BN = 128;                       // output features per tile
constexpr int MAX_T = 128;                    // rows of A per tile, at most
constexpr int BK = 256;                       // K values per stage (128 bytes of codes)
constexpr int W_BYTES = BN * BK / 2;
constexpr int SF_BYTES = 2 * mx::TILE_BYTES;  // scales of 128 rows x 256 values
constexpr int NUM_THREADS = 192;
constexpr int EPI_THREADS = 128;
constexpr int MAX_STAGES = 12;
constexpr int MAX_GATED_STAGES = 10;
constexpr int MAX_SPLIT = 8;                  // portable cluster size
constexpr int SPLIT_T = 32;                   // most rows per tile when the reduction is split
constexpr int SMEM_BUDGET = 200 * 1024;
constexpr size_t ONE_PER_SM = 116 * 1024;

struct Tail {
    uint64_t full[MAX_STAGES];
    uint64_t empty[MAX_STAGES];
    uint64_t moved[MAX_STAGES];      // the stage's A scales lie in the first columns
    uint64_t done;
    uint32_t tmem_base;
    volatile int abort_flag;
};

struct Args {
    const uint8_t* sa;               // scale tiles
    const uint8_t* sw[2];
    const float* bias[2];
    void* Y; long long ldy;          // elements
    uint8_t* ys; long long y_across; // MXFP4 output: scale tiles
    long long M;
    int N, K;
    int k_tiles;                     // scale tiles across K
    int num_kb;                      // stages of the whole reduction
    int t;                           // rows of A per tile: 16, 32, 64 or 128
    int split, log_split;            // CTAs per tile (cluster size), a power of two
    int num_n_tiles;
    int stages, stage_bytes;
    int part_bytes;                  // behind the stages: the partial sums of a split reduction, or rows on their way to MXFP4
    int act;
    uint32_t idesc;
    int* status;
};

__device__ __forceinline__ void st_cluster(uint32_t local, uint32_t rank, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(mx::map_to_cta(local, rank)), "f"(v) : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    uint32_t a[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]),
          "=r"(a[8]), "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(a[i]);
}

// One value of row m and feature n (this lane's), complete over K
template <int OUT>
__device__ __forceinline__ void store_value(const Args& g, long long m, int n, float v) {
    if (n >= g.N) return;
    if (OUT == mx::KIND_BF16) reinterpret_cast<__nv_bfloat16*>(g.Y)[m * g.ldy + n] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(g.Y)[m * g.ldy + n] = v;
}

// MXFP4 output: a lane holds one feature, a block is 32 of them.  The finished values go through shared memory, rows of 4 blocks
// 36 floats apart (so that the 16-byte reads of a warp, 8 rows x 4 blocks, meet no bank twice), and a thread takes a whole block.
constexpr int MX_BLOCK_PITCH = 36, MX_ROW_PITCH = 4 * MX_BLOCK_PITCH;
__device__ __forceinline__ int mx_slot(int row, int nl) { return row * MX_ROW_PITCH + (nl >> 5) * MX_BLOCK_PITCH + (nl & 31); }

// block t & 3 of row t / 4 for every t = thread, thread + 128, ...; buffered row i is row first + i * step of the tile
__device__ __forceinline__ void store_mx(const Args& g, const float* buf, int count, long long m0, int first, int step, int n0, int thread) {
#pragma unroll 1
    for (int t = thread; t < 4 * count; t += EPI_THREADS) {
        const int b = t & 3, n = n0 + 32 * b;
        const float4* src = reinterpret_cast<const float4*>(buf + (t >> 2) * MX_ROW_PITCH + b * MX_BLOCK_PITCH);
        float v[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 q = src[i];
            v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
        }
        uint32_t w[4];
        const uint32_t s = mx::quantize32(v, w);
        const long long m = m0 + first + (long long)(t >> 2) * step;
        uint8_t* dst = reinterpret_cast<uint8_t*>(g.Y) + (m * g.ldy + n) / 2;
        const int bytes = (min(32, g.N - n) + 1) >> 1;        // <= 0 for a block beyond the row's end, whose scale is 0
        if (bytes == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else {
#pragma unroll
            for (int i = 0; i < 16; ++i) if (i < bytes) dst[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
        g.ys[mx::scale_offset(m, n >> 5, g.y_across)] = (uint8_t)s;
    }
}

// N values (of as many rows) of this lane's feature: bias, activation, product
template <bool GATED, int N>
__device__ __forceinline__ void finish_values(const Args& g, float* a, const float* u, float ba, float bu) {
    mx::f2 v[(N + 1) / 2];
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) v[i] = mx::add2(mx::pack2(a[2 * i], N > 1 ? a[2 * i + 1] : 0.0f), mx::both(ba));
    if (GATED || g.act == mx::ACT_RELU) mx::activate_pairs<(N + 1) / 2>(v, GATED ? g.act : mx::ACT_RELU);
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) {
        float lo, hi;
        mx::unpack2(v[i], lo, hi);
        a[2 * i] = GATED ? lo * (u[2 * i] + bu) : lo;
        if (N > 1) a[2 * i + 1] = GATED ? hi * (u[2 * i + 1] + bu) : hi;
    }
}

template <bool GATED, int OUT>
__global__ void __launch_bounds__(NUM_THREADS, 1)
dense_mx_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                const __grid_constant__ CUtensorMap map_u, Args g) {
    constexpr int NW = GATED ? 2 : 1;
    constexpr int SF_COLS = NW * 8 + 8;               // TMEM columns of one stage's scales: W (each), then A
    constexpr int SF0 = NW * MAX_T;                   // after the accumulators
    constexpr int TMEM_COLS = 512;
    static_assert(SF0 + (GATED ? MAX_GATED_STAGES : MAX_STAGES) * SF_COLS <= TMEM_COLS, "a set of scale columns per stage");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);      // by an offset: a pointer made from an integer is no longer known to be shared memory
    float* part = reinterpret_cast<float*>(smem + (size_t)g.stages * g.stage_bytes);
    Tail* tail = reinterpret_cast<Tail*>(smem + (size_t)g.stages * g.stage_bytes + g.part_bytes);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = mx::cluster_rank();
    const int tile = (int)(blockIdx.x / (unsigned)g.split);
    const long long m0 = (long long)(tile / g.num_n_tiles) * g.t;
    const int n0 = (tile % g.num_n_tiles) * BN;
    const int kb0 = (int)((long long)g.num_kb * rank / g.split), kb1 = (int)((long long)g.num_kb * (rank + 1) / g.split);

    // A column of TMEM holds 32 rows' scales, and an MMA reads them from a multiple of 4 columns on.  A row tile that does not
    // begin with a scale tile has its scales moved to the first columns while they are in shared memory.
    const int sf_row = (int)(m0 % mx::TILE_ROWS) / 32;
    volatile int* abort_flag = &tail->abort_flag;
    const int a_bytes = g.t * (BK / 2);

    // stage: W (and Wu) codes, A codes, then the scales of W (and Wu) and of A
    auto load = [&](int kb, int stage) {
        uint8_t* s = smem + (size_t)stage * g.stage_bytes;
        uint64_t* bar = &tail->full[stage];
        const uint32_t sf = (uint32_t)min(2, g.k_tiles - 2 * kb) * mx::TILE_BYTES;
        const long long w_off = ((long long)(n0 / mx::TILE_ROWS) * g.k_tiles + 2 * kb) * mx::TILE_BYTES;
        mbar_arrive_expect_tx(bar, (uint32_t)(NW * W_BYTES + a_bytes) + (NW + 1) * sf);
        tma_load_2d(s, &map_w, bar, kb * (BK / 2), n0);
        if (GATED) tma_load_2d(s + W_BYTES, &map_u, bar, kb * (BK / 2), n0);
        tma_load_2d(s + NW * W_BYTES, &map_a, bar, kb * (BK / 2), (int)m0);
        uint8_t* f = s + g.stage_bytes - (NW + 1) * SF_BYTES;
        mx::bulk_load(f, g.sw[0] + w_off, sf, bar);
        if (GATED) mx::bulk_load(f + SF_BYTES, g.sw[1] + w_off, sf, bar);
        mx::bulk_load(f + NW * SF_BYTES, g.sa + ((m0 / mx::TILE_ROWS) * g.k_tiles + 2 * kb) * mx::TILE_BYTES, sf, bar);
    };
    const int ahead = min(g.stages, kb1 - kb0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < g.stages; ++s) { mbar_init(&tail->full[s], 1); mbar_init(&tail->empty[s], 1); mbar_init(&tail->moved[s], 1); }
        mbar_init(&tail->done, 1);
        tail->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mx::grid_wait();
        for (int i = 0; i < ahead; ++i) load(kb0 + i, i);      // the first round needs no slot to be emptied
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&tail->tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    mx::grid_wait();
    mx::grid_release();
    if (g.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this rank's memory may be written
    const uint32_t tmem_base = tail->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0 + ahead; kb < kb1; ++kb) {
                if (!mbar_wait(&tail->empty[stage], phase, abort_flag, g.status, 151)) break;
                load(kb, stage);
                if (++stage == g.stages) { stage = 0; phase ^= 1u; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            ok = mbar_wait(&tail->full[stage], phase, abort_flag, g.status, 152) &&
                 (sf_row == 0 || mbar_wait(&tail->moved[stage], phase, abort_flag, g.status, 154));
            if (!ok) break;
            tc_fence_after();
            const uint32_t s = smem_u32(smem) + (uint32_t)(stage * g.stage_bytes);
            const int steps = min(4, (g.K - kb * BK + 63) / 64);   // MMAs of 64 values; beyond K nothing is read
            const uint32_t sf = tmem_base + (uint32_t)(SF0 + stage * SF_COLS);
            const uint64_t wdesc = make_smem_desc(s), adesc = make_smem_desc(s + NW * W_BYTES);
            const uint64_t fdesc = mx::make_scale_desc(s + (uint32_t)(g.stage_bytes - (NW + 1) * SF_BYTES));
            if (mx::elect_one()) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {                      // scale tiles of 128 values of K
                    if (steps <= 2 * h) break;
#pragma unroll
                    for (int o = 0; o < NW + 1; ++o)
                        mx::copy_scales(sf + (uint32_t)(o * 8 + h * 4), fdesc + (uint64_t)((o * SF_BYTES + h * mx::TILE_BYTES) >> 4));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k >= steps) break;
#pragma unroll
                    for (int o = 0; o < NW; ++o)
                        mx::umma(tmem_base + (uint32_t)(o * MAX_T), wdesc + (uint64_t)(o * (W_BYTES >> 4) + k * 2), adesc + (uint64_t)(k * 2),
                                 g.idesc | mx::sf_bits(k & 1), sf + (uint32_t)(o * 8 + (k >> 1) * 4), sf + (uint32_t)(NW * 8 + (k >> 1) * 4),
                                 (uint32_t)(kb != kb0 || k != 0));
                }
                umma_commit(&tail->empty[stage]);
                if (kb + 1 == kb1) umma_commit(&tail->done);
            }
            __syncwarp();
            if (++stage == g.stages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 2 && sf_row != 0) {
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&tail->full[stage], phase, abort_flag, g.status, 155)) break;
            uint32_t* f = reinterpret_cast<uint32_t*>(smem + (size_t)(stage + 1) * g.stage_bytes - SF_BYTES) + lane * 4;
            const int halves = min(2, g.k_tiles - 2 * kb);
            for (int h = 0; h < halves; ++h, f += mx::TILE_BYTES / 4) {
                f[0] = f[sf_row];
                if (g.t == 64) f[1] = f[sf_row + 1];       // rows 64-127 of the scale tile: columns 2 and 3
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail->moved[stage]);
            if (++stage == g.stages) { stage = 0; phase ^= 1u; }
        }
        __syncwarp();
    }

    const int quad = warp & 3;
    const int nl = quad * 32 + lane;                                // feature within the tile
    const int n = n0 + nl;
    const int rows = (int)min((long long)g.t, g.M - m0);
    bool ok = false;
    if (warp >= 2) {
        ok = mbar_wait(&tail->done, 0, abort_flag, g.status, 153);
        tc_fence_after();
    }
    const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16);
    float ba = 0.0f, bu = 0.0f;
    if (warp >= 2 && n < g.N) {
        if (g.bias[0]) ba = __ldg(g.bias[0] + n);
        if (GATED && g.bias[1]) bu = __ldg(g.bias[1] + n);
    }
    // rows on their way to MXFP4: over the stages, which are done with, where they are large enough
    float* rowbuf = g.split > 1 || g.part_bytes == 0 ? reinterpret_cast<float*>(smem) : part;
    if (g.split == 1) {
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < rows; c += 16) {
                float a[16], u[16];
                tmem_ld16(taddr + (uint32_t)c, a);
                if (GATED) tmem_ld16(taddr + (uint32_t)(MAX_T + c), u);
                finish_values<GATED, 16>(g, a, u, ba, bu);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (OUT == mx::KIND_MX) rowbuf[mx_slot(c + i, nl)] = n < g.N ? a[i] : 0.0f;      // g.t rows have room
                    else if (c + i < rows) store_value<OUT>(g, m0 + c + i, n, a[i]);
                }
            }
        }
        if (OUT == mx::KIND_MX && warp >= 2) {
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (ok) store_mx(g, rowbuf, rows, m0, 0, 1, n0, threadIdx.x - 64);
        }
    } else {
        // row r is finished by rank r mod split; part[from][r / split][projection][feature] there
        const int per = g.t >> g.log_split;
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // every rank has started
        if (ok) {
            const uint32_t base = smem_u32(part) + (uint32_t)((int)rank * per * NW * BN + nl) * 4u;
#pragma unroll 1
            for (int c = 0; c < rows; c += 16)
#pragma unroll 1
                for (int o = 0; o < NW; ++o) {
                    float a[16];
                    tmem_ld16(taddr + (uint32_t)(o * MAX_T + c), a);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (c + i < rows)
                            st_cluster(base + (uint32_t)(((c + i) >> g.log_split) * NW + o) * (BN * 4u), (uint32_t)((c + i) & (g.split - 1)), a[i]);
                }
        }
        __syncwarp();
        mx::cluster_sync_all();          // all partial sums have arrived
        if (warp >= 2) {
            const float* p = part + nl;
#pragma unroll 1
            for (int r = (int)rank; r < rows; r += g.split, p += NW * BN) {
                float a = 0.0f, u = 0.0f;
#pragma unroll
                for (int q = 0; q < MAX_SPLIT; ++q)
                    if (q < g.split) {
                        a += p[q * per * NW * BN];
                        if (GATED) u += p[q * per * NW * BN + BN];
                    }
                finish_values<GATED, 1>(g, &a, &u, ba, bu);
                if (OUT == mx::KIND_MX) rowbuf[mx_slot(r >> g.log_split, nl)] = n < g.N ? a : 0.0f;
                else if (ok) store_value<OUT>(g, m0 + r, n, a);
            }
            if (OUT == mx::KIND_MX) {
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (ok) store_mx(g, rowbuf, (rows - (int)rank + g.split - 1) >> g.log_split, m0, (int)rank, g.split, n0, threadIdx.x - 64);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {           // copies in flight must land before the memory is given back
        const uint64_t t0 = a4c_globaltimer();
        while (a4c_globaltimer() - t0 < 2000000ull) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
    }
}

template <bool GATED, int OUT>
cudaError_t launch(const CUtensorMap* m, const Args& g, unsigned grid, size_t smem, cudaStream_t s) {
    static tc::SmemOptIn opt_in;
    const cudaError_t e = opt_in.ensure(dense_mx_kernel<GATED, OUT>, SMEM_BUDGET + 16 * 1024);
    if (e != cudaSuccess) return e;
    return mx::launch_serialized(dense_mx_kernel<GATED, OUT>, grid, NUM_THREADS, smem, (unsigned)g.split, s, m[0], m[1], m[2], g);
}

}  // namespace

int a4c_launch_dense_mx(const A4cMxDense& d, int* status_word, cudaStream_t stream) {
    const bool gated = d.wu != nullptr;
    const int nw = gated ? 2 : 1;
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (a4c_dense_mx_wide_wanted(d, sms)) return a4c_launch_dense_mx_wide(d, sms, status_word, stream);
    Args g;
    g.sa = d.sa; g.sw[0] = d.sw; g.sw[1] = d.su; g.bias[0] = d.bias; g.bias[1] = d.bias_u;
    g.Y = d.y; g.ldy = d.ldy; g.ys = d.ys; g.y_across = mx::tiles_across(d.N);
    g.M = d.M; g.N = d.N; g.K = d.K; g.k_tiles = (int)mx::tiles_across(d.K);
    g.num_kb = (d.K + BK - 1) / BK;
    g.act = d.act; g.status = status_word;
    g.num_n_tiles = (d.N + BN - 1) / BN;
    g.t = d.M > 64 ? 128 : d.M > 32 ? 64 : d.M > 16 ? 32 : 16;
    auto tiles_of = [&](int t) { return (d.M + t - 1) / t * g.num_n_tiles; };
    if (tiles_of(g.t) > 2147483647LL / MAX_SPLIT) return A4C_ERR_TOO_LARGE;
    // Smaller row tiles, then a split reduction, while at most half of the SMs have work and every rank keeps a stage.
    while (g.t > SPLIT_T && tiles_of(g.t) * 2 <= sms) g.t /= 2;
    const long long tiles = tiles_of(g.t);
    g.split = 1;
    while (g.split < MAX_SPLIT && g.t <= SPLIT_T && tiles * g.split * 2 <= sms && g.split * 2 <= g.num_kb) g.split *= 2;
    g.log_split = g.split == 1 ? 0 : g.split == 2 ? 1 : g.split == 4 ? 2 : 3;
    g.idesc = mx::make_idesc(BN, g.t);
    g.stage_bytes = nw * W_BYTES + g.t * (BK / 2) + (nw + 1) * SF_BYTES;
    const int need = (g.num_kb + g.split - 1) / g.split;
    const int limit = gated ? MAX_GATED_STAGES : MAX_STAGES;
    g.part_bytes = g.split > 1 ? nw * g.t * BN * 4 : 0;
    g.stages = (SMEM_BUDGET - g.part_bytes) / g.stage_bytes;
    if (g.stages > limit) g.stages = limit;
    if (need < g.stages) g.stages = need;
    const int row_bytes = d.out_kind == mx::KIND_MX && g.split == 1 ? g.t * MX_ROW_PITCH * 4 : 0;
    if (row_bytes > g.stages * g.stage_bytes) g.part_bytes = row_bytes;      // few stages: it fits beside them
    size_t smem = 1024 + (size_t)g.stages * g.stage_bytes + g.part_bytes + sizeof(Tail);
    // More than half of an SM's shared memory, so that one CTA lives on an SM at a time: the ranks of a cluster wait for
    // one another while they hold tensor memory, and two clusters that shared SMs could each wait for the other's.
    if (smem < ONE_PER_SM) smem = ONE_PER_SM;
    CUtensorMap m[3];
    if (!mx::make_code_map(&m[0], d.a, d.M, d.K, d.lda, g.t) || !mx::make_code_map(&m[1], d.w, d.N, d.K, d.ldw, BN)) return A4C_ERR_CUDA;
    m[2] = m[1];
    if (gated && !mx::make_code_map(&m[2], d.wu, d.N, d.K, d.ldu, BN)) return A4C_ERR_CUDA;
    const unsigned grid = (unsigned)(tiles * g.split);
    cudaError_t err;
    if (gated)
        err = d.out_kind == mx::KIND_BF16 ? launch<true, mx::KIND_BF16>(m, g, grid, smem, stream)
              : d.out_kind == mx::KIND_F32 ? launch<true, mx::KIND_F32>(m, g, grid, smem, stream) : launch<true, mx::KIND_MX>(m, g, grid, smem, stream);
    else
        err = d.out_kind == mx::KIND_BF16 ? launch<false, mx::KIND_BF16>(m, g, grid, smem, stream)
              : d.out_kind == mx::KIND_F32 ? launch<false, mx::KIND_F32>(m, g, grid, smem, stream) : launch<false, mx::KIND_MX>(m, g, grid, smem, stream);
    return err == cudaSuccess ? A4C_OK : A4C_ERR_CUDA;
}
