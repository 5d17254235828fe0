// gm_tile_gemm.cuh -- the matrix products of the vocabulary loss on the fifth-generation
// tensor cores: a persistent kernel of CTA pairs, C[256 x N] per pair and tile.
//
//   warp 0    one lane copies operand tiles into a ring of shared-memory stages (TMA)
//   warp 1    one lane of the pair's first CTA issues tcgen05.mma (M = 256 over both SMs,
//             N = 256 or less, K = 16, fp16 or bf16 in, binary32 accumulators in TMEM)
//   warps 2-5 read the accumulators (each thread one row) and run the epilogue
//
// The accumulators take N TMEM columns and there are two sets of them, so the epilogue of
// one tile runs while the next one is multiplied.  Of the pair, each CTA holds 128 rows of A
// and half of the N rows of B: with N = 256 a stage is 32 KB per CTA and six of them fit.
//
// Where a product has too few tiles for the GPU, a tile's K range is split over several pairs,
// and a kernel of its own adds up what they leave (TilePlan::splits).
//
// Operands are read as they lie in memory, K-major or MN-major, always with the 128-byte
// swizzle: a K-major tile is rows of 64 elements (128 bytes), eight rows to a 1,024-byte
// pattern; an MN-major tile is blocks of 64 columns by 64 K-rows (8 KB each).
//
// Every wait is bounded: one that runs out raises the CTA's abort flag and *status, all
// roles leave their loops, copies in flight are waited for (bounded again) and TMEM is freed.
#pragma once

#include <cuda.h>

#include "gm_lm.cuh"

namespace gm {

constexpr int kTileM = 256, kTileN = 256, kTileK = 64;
constexpr int kHalf = 128;                       // rows of A that one CTA of the pair holds
constexpr int kOperandBytes = kHalf * kTileK * 2;
constexpr int kGemmThreads = 192;
template <int TN> struct Ring {                  // the ring of stages for tiles of TN columns
    static constexpr int kRowsB = TN / 2;
    static constexpr int kStageBytes = kOperandBytes + kRowsB * kTileK * 2;
    static constexpr int kFit = 200 * 1024 / kStageBytes;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr int kSmem = kStages * kStageBytes + 1024;
};

// ---- mbarriers ----
__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ unsigned pair_leader_addr(unsigned addr) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// False when the wait ran out or another role gave up.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, volatile int* abort, long long budget) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (*abort) return false;
        if (clock64() - t0 > budget) { *abort = 1; return false; }
    }
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- TMA: a 2-D box into this CTA's shared memory, bytes counted by a barrier of the pair ----
__device__ __forceinline__ void tma_load(unsigned dst, const CUtensorMap* map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// ---- tcgen05 ----
// Shared-memory matrix descriptor: address, leading and stride byte offsets in units of 16
// bytes, version 1 (bits 46-48), 128-byte swizzle (2 in bits 61-63).  K-major: 1,024 bytes
// from one group of eight rows to the next.  MN-major: 8,192 bytes from one block of 64
// columns to the next, 1,024 from one group of eight K-rows to the next.
__device__ __forceinline__ unsigned long long mat_desc(unsigned addr, bool mn_major) {
    const unsigned long long lead = mn_major ? (8192 >> 4) : 1, stride = 1024 >> 4;
    return (unsigned long long)((addr & 0x3ffffu) >> 4) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)accumulate) : "memory");
}
// Arrives on the barrier at this offset in both CTAs when all MMAs issued so far are done.
__device__ __forceinline__ void mma_commit_pair(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((unsigned short)3) : "memory");
}
__device__ __forceinline__ void tmem_load32(unsigned addr, float (&v)[32]) {
    unsigned r[32];
    __syncwarp();                                    // the load is for whole, converged warps
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Where the work of one turn lies: tile, its share of K, and the turn's number.
struct TileAt { int m, n, split, item, k0, k1; };

// One product: m_tiles x n_tiles tiles, walked m first inside groups of `group` m-tiles, so that
// the operands of the tiles in flight are shared in L2; each in `splits` shares of K.
struct TilePlan {
    int m_tiles, n_tiles, k_blocks, group, splits;
    __device__ __forceinline__ int items() const { return m_tiles * n_tiles * splits; }
    __device__ __forceinline__ TileAt at(int item) const {
        TileAt x;
        const int t = item / splits, per = group * n_tiles;
        const int g = t / per, m0 = g * group;
        const int rows = m_tiles - m0 < group ? m_tiles - m0 : group;
        const int r = t - g * per;
        x.item = item;
        x.n = r / rows;
        x.m = m0 + (r - x.n * rows);
        x.split = item - t * splits;
        x.k0 = (int)((long long)k_blocks * x.split / splits);
        x.k1 = (int)((long long)k_blocks * (x.split + 1) / splits);
        return x;
    }
    // the inverse: number of the tile at (m, n)
    __device__ __forceinline__ int tile_of(int m, int n) const {
        const int m0 = m / group * group;
        const int rows = m_tiles - m0 < group ? m_tiles - m0 : group;
        return m0 * n_tiles + n * rows + (m - m0);
    }
};

// Shares of K per tile, at most 16 and `most_items` in all, for the shortest run on `pairs` CTA
// pairs: rounds of items, each as long as its k-blocks plus a start and an epilogue (about eight).
__device__ __forceinline__ int choose_splits(int tiles, int k_blocks, int pairs, int most_items) {
    int best = 1, best_cost = 0x7fffffff;
    for (int s = 1; s <= 16 && s <= k_blocks && (s == 1 || tiles * s <= most_items); ++s) {
        const int cost = (tiles * s + pairs - 1) / pairs * ((k_blocks + s - 1) / s + 8) + (s > 1 ? 8 : 0);
        if (cost < best_cost) { best_cost = cost; best = s; }
    }
    return best;
}

// MN_A / MN_B: that operand is MN-major.  Ops provides
//   kBf16             whether the inputs are bf16 (else fp16)
//   plan(pairs)       the tiles, read on the device
//   a0, b0            first row of A and of B (first K-row of an MN-major operand) in their maps
//   epilogue(at, row, addr)   the turn, the row inside the tile, the TMEM address of its first
//                     column; called by whole warps, also for rows behind the last one; with an
//                     empty share of K (at.k0 == at.k1) the accumulators hold nothing and C is zero
template <int TN, bool MN_A, bool MN_B, typename Ops>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
tile_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Ops ops,
                 int* status, const long long budget) {
    constexpr int kStages = Ring<TN>::kStages, kStageBytes = Ring<TN>::kStageBytes, kRowsB = Ring<TN>::kRowsB;
    static_assert(!MN_B || TN == 256, "an MN-major B comes in two blocks of 64 columns per CTA");
    extern __shared__ unsigned char dyn[];
    __shared__ __align__(8) unsigned long long full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
    __shared__ unsigned tmem_base;
    __shared__ volatile int abort_flag;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = cluster_rank();
    const unsigned ring = (smem_u32(dyn) + 1023u) & ~1023u;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < kStages; ++s) { mbar_init(smem_u32(&full[s]), 1); mbar_init(smem_u32(&empty[s]), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(smem_u32(&acc_full[b]), 1); mbar_init(smem_u32(&acc_empty[b]), 8); }
        mbar_init(smem_u32(&drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_base;
    // all of the above may run while the kernel before this one ends
    cudaGridDependencySynchronize();
    const TilePlan plan = ops.plan(pairs);
    const int items = plan.items();

    unsigned issued = 0;                                         // k-blocks this thread copied; stage and parity follow from it
    if (warp == 0 && lane == 0) {
        // ---- copies ----
        bool ok = true;
        for (int t = pair; t < items && ok; t += pairs) {
            const TileAt at = plan.at(t);
            const int row_a = at.m * kTileM + (int)rank * kHalf, row_b = at.n * TN + (int)rank * kRowsB;
            for (int k = at.k0; k < at.k1; ++k, ++issued) {
                const int s = issued % kStages;
                const unsigned turn = issued / kStages;
                if (!mbar_wait(smem_u32(&empty[s]), (turn & 1u) ^ 1u, &abort_flag, budget)) { ok = false; break; }
                const unsigned bar = pair_leader_addr(smem_u32(&full[s]));
                if (rank == 0) mbar_expect(smem_u32(&full[s]), 2 * kStageBytes);
                const unsigned a = ring + s * kStageBytes, b = a + kOperandBytes;
                if (MN_A) {
                    tma_load(a, &map_a, row_a, ops.a0 + k * kTileK, bar);
                    tma_load(a + 8192, &map_a, row_a + 64, ops.a0 + k * kTileK, bar);
                } else {
                    tma_load(a, &map_a, k * kTileK, ops.a0 + row_a, bar);
                }
                if (MN_B) {
                    tma_load(b, &map_b, row_b, ops.b0 + k * kTileK, bar);
                    tma_load(b + 8192, &map_b, row_b + 64, ops.b0 + k * kTileK, bar);
                } else {
                    tma_load(b, &map_b, k * kTileK, ops.b0 + row_b, bar);
                }
            }
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- products ----
        // accumulators binary32, inputs fp16 or bf16, N / 8 in bits 17-22, M / 16 in bits 24-28
        const unsigned in = Ops::kBf16 ? 1u : 0u;
        const unsigned idesc = (1u << 4) | (in << 7) | (in << 10) | ((MN_A ? 1u : 0u) << 15) | ((MN_B ? 1u : 0u) << 16) |
                               ((unsigned)(TN / 8) << 17) | ((unsigned)(kTileM / 16) << 24);
        unsigned used = 0;
        int count = 0;
        bool ok = true;
        for (int t = pair; t < items && ok; t += pairs, ++count) {
            const TileAt at = plan.at(t);
            const int b = count & 1;
            if (!mbar_wait(smem_u32(&acc_empty[b]), ((count >> 1) & 1) ^ 1, &abort_flag, budget)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned d = tmem + (unsigned)b * TN;
            for (int k = at.k0; k < at.k1; ++k, ++used) {
                const int s = used % kStages;
                if (!mbar_wait(smem_u32(&full[s]), (used / kStages) & 1u, &abort_flag, budget)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned a = ring + s * kStageBytes;
                const unsigned long long da = mat_desc(a, MN_A), db = mat_desc(a + kOperandBytes, MN_B);
#pragma unroll
                for (int i = 0; i < kTileK / 16; ++i)
                    mma_pair(d, da + (MN_A ? 128 * i : 2 * i), db + (MN_B ? 128 * i : 2 * i), idesc, k > at.k0 || i > 0);
                mma_commit_pair(smem_u32(&empty[s]));
            }
            if (ok) mma_commit_pair(smem_u32(&acc_full[b]));
        }
        if (!ok) {
            mma_commit_pair(smem_u32(&drain));
            const long long t0 = clock64();
            while (!mbar_try(smem_u32(&drain), 0) && clock64() - t0 < budget) {}
        }
    } else if (warp >= 2) {
        // ---- epilogue ----
        const int quarter = warp & 3;                            // the TMEM lanes this warp may read
        const int row = quarter * 32 + lane;
        int count = 0;
        for (int t = pair; t < items; t += pairs, ++count) {
            const TileAt at = plan.at(t);
            const int b = count & 1;
            const bool ok = mbar_wait(smem_u32(&acc_full[b]), (count >> 1) & 1, &abort_flag, budget);
            if (!__all_sync(0xffffffffu, ok)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            ops.epilogue(at, (int)rank * kHalf + row, tmem + (unsigned)b * TN + ((unsigned)(quarter * 32) << 16));
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(pair_leader_addr(smem_u32(&acc_empty[b])));
        }
    }
    __syncwarp();
    __syncthreads();
    if (tid == 0 && abort_flag) {
        // gave up: the copies of the last stages may be in flight; wait for them before leaving
        *status = 1;
        if (rank == 0) {
            for (unsigned i = issued > (unsigned)kStages ? issued - kStages : 0u; i < issued; ++i) {
                const long long t0 = clock64();
                while (!mbar_try(smem_u32(&full[i % kStages]), (i / kStages) & 1u) && clock64() - t0 < budget) {}
            }
        }
    }
    __syncwarp();
    cluster_sync_all();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace gm
