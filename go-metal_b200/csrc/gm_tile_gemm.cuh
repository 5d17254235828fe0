// gm_tile_gemm.cuh -- the matrix products of the vocabulary loss on the fifth-generation
// tensor cores: a persistent kernel of CTA pairs.
//
//   warp 0    one lane copies operand tiles into a ring of shared-memory stages (TMA)
//   warp 1    one lane of the pair's first CTA issues tcgen05.mma (M = 256 over both SMs,
//             N = 256 or less, K = 16, fp16 or bf16 in, binary32 accumulators in TMEM)
//   warps 2-9 read the accumulators (each thread half of a row) and run the epilogue
//
// C is made of tiles of 256 rows by TN columns; TMEM holds two of them, in two slots that take
// turns.  Of a tile's operands each CTA holds 128 rows of A and half of the TN rows of B: with
// N = 256 a stage is 32 KB per CTA and six of them fit.  The epilogue takes a slot's numbers into
// registers, 128 per thread, and frees the slot before it works on them.
//
// Measured on B200 at 8,192 x 4,096 x 32,768: the tensor core is busy in 95 % of the cycles.  In
// a loop of seconds the card's power limit holds it near 1,350 TFLOP/s (the library's products of the
// same shapes reach 1,340 to 1,410).  Tiles of 512 x 256 per pair, whose operands cross L2 a
// quarter less often, were built too and were 5 % slower (81 % of the cycles, TMEM leaves no second
// slot); waiting with the default poll interval cost 6 %, rows stored lane by lane 3 %.
//
// Where a product has too few tiles for the GPU, a tile's K range is split over several pairs,
// and a kernel of its own adds up what they leave (TilePlan::splits).
//
// Operands are read as they lie in memory, K-major or MN-major, always with the 128-byte
// swizzle: a K-major tile is rows of 64 elements (128 bytes), eight rows to a 1,024-byte
// pattern; an MN-major tile is blocks of 64 columns by 64 K-rows (8 KB each).
//
// Every wait is bounded: one that runs out raises the CTA's abort flag and *status, all
// roles leave their loops, copies in flight are waited for (bounded again) and TMEM is freed.  An epilogue
// whose accumulators did not come marks its tile with NaN, so that the outputs show it.
#pragma once

#include <cuda.h>

#include <climits>
#include <type_traits>

#include "gm_lm.cuh"

namespace gm {

constexpr int kTileM = 256, kTileN = 256, kTileK = 64;
constexpr int kHalf = 128;                       // rows of A that one CTA of the pair holds
constexpr int kOperandBytes = kHalf * kTileK * 2;
constexpr int kGemmThreads = 320;
template <int TN> struct Ring {                  // a stage: a block of A, then one of B
    static constexpr int kRowsB = TN / 2;
    static constexpr int kStageBytes = kOperandBytes + kRowsB * kTileK * 2;
    static constexpr int kFit = 193 * 1024 / kStageBytes;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr int kSmem = kStages * kStageBytes + 1024;        // and 8 x kStagingBytes with kStaging
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
// Relaxed: it says that TMEM has been read (tcgen05.wait::ld and the fence in front of it), nothing
// else.  A release would first wait for the lane's stores to memory, which cost a tile's epilogue 1,100
// to 1,700 cycles (16,000 x 256 x 16,000 backward 530 -> 504 us, 64 x 2,048 x 50,257 174 -> 159 us).
__device__ __forceinline__ void mbar_arrive_cluster(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A try sleeps up to this long in hardware.  Short sleeps are polls, and a poll is an access to the
// shared memory that feeds the tensor core: with the default the waiting epilogue warps cost 6 %.
constexpr unsigned kPollNs = 10000000;
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity), "r"(kPollNs) : "memory");
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
// COUNT columns (a multiple of 32) of this thread's TMEM lane, for whole, converged warps.
template <int COUNT>
__device__ __forceinline__ void tmem_read(unsigned addr, float (&v)[COUNT]) {
    unsigned r[COUNT];
    __syncwarp();
#pragma unroll
    for (int c = 0; c < COUNT; c += 32)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                     "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                     "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                     : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]), "=r"(r[c + 6]), "=r"(r[c + 7]),
                       "=r"(r[c + 8]), "=r"(r[c + 9]), "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]), "=r"(r[c + 13]), "=r"(r[c + 14]),
                       "=r"(r[c + 15]), "=r"(r[c + 16]), "=r"(r[c + 17]), "=r"(r[c + 18]), "=r"(r[c + 19]), "=r"(r[c + 20]), "=r"(r[c + 21]),
                       "=r"(r[c + 22]), "=r"(r[c + 23]), "=r"(r[c + 24]), "=r"(r[c + 25]), "=r"(r[c + 26]), "=r"(r[c + 27]), "=r"(r[c + 28]),
                       "=r"(r[c + 29]), "=r"(r[c + 30]), "=r"(r[c + 31])
                     : "r"(addr + c));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // the registers are valid from here on: nothing that uses them may move in front of the wait
#pragma unroll
    for (int c = 0; c < COUNT; c += 8)
        asm volatile("" : "+r"(r[c]), "+r"(r[c + 1]), "+r"(r[c + 2]), "+r"(r[c + 3]), "+r"(r[c + 4]), "+r"(r[c + 5]), "+r"(r[c + 6]), "+r"(r[c + 7]));
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = __uint_as_float(r[i]);
}

// The same, added to what v holds; eight columns at a time, which leaves v its registers.
template <int COUNT>
__device__ __forceinline__ void tmem_add(unsigned addr, float (&v)[COUNT]) {
#pragma unroll
    for (int c = 0; c < COUNT; c += 8) {
        unsigned r[8];
        __syncwarp();
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
                     "tcgen05.wait::ld.sync.aligned;"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(addr + c) : "memory");
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c + k] = __fadd_rn(v[c + k], __uint_as_float(r[k]));
    }
}

// ---- rows to memory ----
// A warp holds 32 rows, one per lane.  Stored as they are, each lane's 16 bytes would be a line of
// their own, and a line is a cycle of the memory that feeds the tensor core; so they go through 4 KB of
// shared memory per warp and leave as whole lines.  The 16-byte units of a row are exchanged by the
// row's number so that neither side has bank conflicts.
constexpr int kStagingBytes = 4096;
__device__ __forceinline__ void stage_put(unsigned stage, int row, int unit, uint4 x) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                 ::"r"(stage + row * 128 + ((unit ^ (row & 7)) << 4)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
__device__ __forceinline__ uint4 stage_get(unsigned stage, int row, int unit) {
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(stage + row * 128 + ((unit ^ (row & 7)) << 4)) : "memory");
    return x;
}

// The staging is this warp's again: the stores that read it have done so.
__device__ __forceinline__ void stage_free() {
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

// 128 columns of 32 rows in a 16-bit type to a map's rows from y on and columns from x on (a multiple of
// 64), by TMA stores that run on while the warp takes its next tile; rows and 16-byte words outside the map
// are not written, `cols` columns exist.  The staging is what the map's 128-byte swizzle says.  Read
// back and stored by the warp itself, a tile's epilogue took 6,000 cycles, more than the product of
// a short K: logits and dW at 64 x 2,048 x 50,257 168 -> 120 us, a backward pass of 1,002 x 1,184 x 10,878 157 -> 103 us.
template <typename T>
__device__ __forceinline__ void rows_to_memory(unsigned stage, const float (&v)[128], int cols, const CUtensorMap* map, int x, int y) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 128; c += 64) {
        if (c >= cols) break;
        stage_free();
#pragma unroll
        for (int u = 0; u < 8; ++u)
            stage_put(stage, lane, u, make_uint4(pack2<T>(v[c + 8 * u], v[c + 8 * u + 1]), pack2<T>(v[c + 8 * u + 2], v[c + 8 * u + 3]),
                                                 pack2<T>(v[c + 8 * u + 4], v[c + 8 * u + 5]), pack2<T>(v[c + 8 * u + 6], v[c + 8 * u + 7])));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n\t"
                         "cp.async.bulk.commit_group;" ::"l"(map), "r"(x + c), "r"(y), "r"(stage) : "memory");
    }
}

// 128 columns of 32 rows as they are (binary32), four at a time, neighbouring lanes with neighbouring
// columns: first old = get(row in the warp, that row's lane's tag, column) for four of them, so that
// what is read is in flight together, then put(row, tag, column, four values, old).
template <typename Get, typename Put>
__device__ __forceinline__ void rows_by_fours(unsigned stage, const float (&v)[128], int cols, int tag, Get get, Put put) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < 128; c += 32) {
        if (c >= cols) break;
        stage_free();
#pragma unroll
        for (int u = 0; u < 8; ++u)
            stage_put(stage, lane, u, make_uint4(__float_as_uint(v[c + 4 * u]), __float_as_uint(v[c + 4 * u + 1]), __float_as_uint(v[c + 4 * u + 2]),
                                                 __float_as_uint(v[c + 4 * u + 3])));
        __syncwarp();
        const int unit = lane & 7, at = c + unit * 4;
#pragma unroll 1
        for (int r = lane >> 3; r < 32; r += 16) {
            decltype(get(0, 0, 0)) old[4];
            int tags[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                tags[i] = __shfl_sync(0xffffffffu, tag, r + i * 4);
                if (at < cols) old[i] = get(r + i * 4, tags[i], at);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 x = stage_get(stage, r + i * 4, unit);
                if (at < cols) put(r + i * 4, tags[i], at, make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)), old[i]);
            }
        }
    }
}

// The work of one turn: a tile, its share of K, and the part it leaves (-1: the whole tile).
struct TileAt { int m, n, part, k0, k1; };

// How many sums a turn's K is cut into where it is to be cut.  The tensor cores cut where
// they add, which shifts a sum of n blocks of 64 towards zero by up to n 2^-23 of it, and a mean loss
// with it: with one sum, by 4.7e-6 of itself at 8,192 columns, 1.3e-6 at 4,096 and 3.4e-7 at 2,048.
// Every sum more costs a read of the accumulators, 570 cycles: 2,048 columns in two sums 3.5 % (1.7e-7),
// 4,096 in two 2 % (6.9e-7).  So: one up to kOneSum columns, two up to 4,096, 1,536 each beyond (the
// logits grow with the columns, and the shift is in proportion to both).
constexpr int kOneSum = 2048;
template <bool LONG>
__device__ __forceinline__ int chunks_of(const TileAt& at) {
    const int n = at.k1 - at.k0;
    return !LONG ? 1 : n <= 64 ? 2 : (n + 23) / 24;
}

// One product: m_tiles x n_tiles tiles, walked m first inside groups of `group` m-tiles, so that
// the operands of the tiles in flight are shared in L2.  The first `whole` tiles are a turn each, the
// others `splits` turns, each with a share of K.
struct TilePlan {
    int count;                                                // rows with a target
    int m_tiles, n_tiles, k_blocks, group, whole, splits;
    __device__ __forceinline__ int tiles() const { return m_tiles * n_tiles; }
    __device__ __forceinline__ int items() const { return whole + (tiles() - whole) * splits; }
    __device__ __forceinline__ void place(int tile, int* m, int* n) const {
        const int per = group * n_tiles, g = tile / per, m0 = g * group;
        const int high = m_tiles - m0 < group ? m_tiles - m0 : group;
        const int r = tile - g * per;
        *n = r / high;
        *m = m0 + (r - *n * high);
    }
    __device__ __forceinline__ TileAt at(int item) const {
        TileAt x{0, 0, -1, 0, k_blocks};
        int tile = item;
        if (item >= whole) {
            x.part = item - whole;
            tile = whole + x.part / splits;
            const int share = x.part % splits;
            x.k0 = (int)((long long)k_blocks * share / splits);
            x.k1 = (int)((long long)k_blocks * (share + 1) / splits);
        }
        place(tile, &x.m, &x.n);
        return x;
    }
};

// A plan without shares of K.
__device__ __forceinline__ TilePlan whole_tiles(int count, int m_tiles, int n_tiles, int k_blocks, int group) {
    return {count, m_tiles, n_tiles, k_blocks, group, m_tiles * n_tiles, 1};
}

// Splits the tiles behind the last full round of `pairs` (or of the round before, too), into at
// most 16 shares each and `most_parts` in all, for the shortest run: rounds of turns, each as long as
// its k-blocks plus a start and an epilogue (about eight).  Called by whole warps: each lane weighs one
// of the 30 choices (weighed one after the other they took 3 us at the start of two kernels).
__device__ __forceinline__ void split_tail(TilePlan* p, int pairs, int most_parts) {
    const int tiles = p->tiles(), k = p->k_blocks, lane = threadIdx.x & 31;
    const int tail = tiles % pairs + (lane >= 15 ? pairs : 0), s = 2 + (lane >= 15 ? lane - 15 : lane);
    const bool possible = lane < 30 && tail > 0 && tail <= tiles && s <= k && tail * s <= most_parts;
    const int cost = (tiles - tail) / pairs * (k + 8) + (tail * s + pairs - 1) / pairs * ((k + s - 1) / s + 8) + 8;
    const int best = __reduce_min_sync(0xffffffffu, possible ? cost : INT_MAX);
    const unsigned at = __ballot_sync(0xffffffffu, possible && cost == best);
    const bool split = at != 0u && best < (tiles + pairs - 1) / pairs * (k + 8);
    const int from = at != 0u ? __ffs((int)at) - 1 : 0;
    const int best_tail = __shfl_sync(0xffffffffu, tail, from), best_s = __shfl_sync(0xffffffffu, s, from);
    p->whole = split ? tiles - best_tail : tiles;
    p->splits = split ? best_s : 1;
}

// A product: the operands' maps, which of them are MN-major, and Ops, which provides
//   kBf16             whether the inputs are bf16 (else fp16)
//   kStaging          whether the epilogue wants shared memory
//   kLong             whether K is cut into several sums, which the epilogue's warps add up
//   begin()           run by one thread before anything else
//   rows_a()          rows of A per CTA, 128 or a smaller multiple of 8 (K-major A only); the box of
//                     its map has as many, the accumulators' other rows hold anything
//   plan(pairs)       the tiles, read on the device by whole warps
//   a0, b0            first row of A and of B (first K-row of an MN-major operand) in their maps
//   once(plan)        what the epilogues of all turns need
//   prepare(plan, at, row)   what the epilogue of this turn needs for the row inside the tile, read
//                     while the product runs
//   epilogue(plan, at, row, v, half, stage, once, prepared)   the row inside the tile, half of its
//                     columns (zeros with an empty share of K), which half, 4 KB of shared memory for
//                     the warp (with kStaging); called by whole warps, also for rows behind the last one
//   gave_up(plan, at, row, half)   a NaN into what this thread would have written
template <typename Ops_, bool MN_A, bool MN_B>
struct Product {
    using Ops = Ops_;
    static constexpr bool kMnA = MN_A, kMnB = MN_B, kAny = true;
    CUtensorMap a, b;
    Ops ops;
    __device__ __forceinline__ TilePlan plan(int pairs) const { return ops.plan(pairs); }
};
struct Nothing {};
struct NoProduct {
    static constexpr bool kAny = false;
    __device__ __forceinline__ TilePlan plan(int) const { return {0, 0, 0, 0, 1, 0, 1}; }
};

// One product, or two whose inputs are ready at the same time: the second one's tiles then fill the
// pairs that the first one's last round leaves idle.
template <int TN, typename First, typename Second>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
tile_gemm_kernel(const __grid_constant__ First first, const __grid_constant__ Second second, int* status, const long long budget) {
    constexpr int kStages = Ring<TN>::kStages, kStageBytes = Ring<TN>::kStageBytes, kRowsB = Ring<TN>::kRowsB;
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
        for (int b = 0; b < 2; ++b) { mbar_init(smem_u32(&acc_full[b]), 1); mbar_init(smem_u32(&acc_empty[b]), 16); }
        mbar_init(smem_u32(&drain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 64) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&first.a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&first.b) : "memory");
        if constexpr (Second::kAny) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&second.a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&second.b) : "memory");
        }
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
    chain_begin();
    if (blockIdx.x == 0 && tid == 0) first.ops.begin();
    const TilePlan plan = first.plan(pairs), plan2 = second.plan(pairs);
    const int items = plan.items(), all = items + plan2.items();

    unsigned issued = 0;                                         // k-blocks this thread copied; stage and parity follow from it
    if (warp == 0 && lane == 0) {
        // ---- copies ----
        auto copy = [&](const auto& product, const TileAt at) {
            using P = std::decay_t<decltype(product)>;
            static_assert(!P::kMnB || TN == 256, "an MN-major B comes in two blocks of 64 columns per CTA");
            const int rows_a = product.ops.rows_a();
            const unsigned bytes = 2u * (unsigned)(rows_a + kRowsB) * (kTileK * 2);          // both CTAs' copies
            const int row_a = (at.m * 2 + (int)rank) * rows_a, row_b = at.n * TN + (int)rank * kRowsB;
            for (int k = at.k0; k < at.k1; ++k, ++issued) {
                const int s = issued % kStages;
                const unsigned turn = issued / kStages;
                if (!mbar_wait(smem_u32(&empty[s]), (turn & 1u) ^ 1u, &abort_flag, budget)) return false;
                const unsigned bar = pair_leader_addr(smem_u32(&full[s]));
                if (rank == 0) mbar_expect(smem_u32(&full[s]), bytes);
                const unsigned a = ring + s * kStageBytes, b = a + kOperandBytes;
                if (P::kMnA) {
                    tma_load(a, &product.a, row_a, product.ops.a0 + k * kTileK, bar);
                    tma_load(a + 8192, &product.a, row_a + 64, product.ops.a0 + k * kTileK, bar);
                } else {
                    tma_load(a, &product.a, k * kTileK, product.ops.a0 + row_a, bar);
                }
                if (P::kMnB) {
                    tma_load(b, &product.b, row_b, product.ops.b0 + k * kTileK, bar);
                    tma_load(b + 8192, &product.b, row_b + 64, product.ops.b0 + k * kTileK, bar);
                } else {
                    tma_load(b, &product.b, k * kTileK, product.ops.b0 + row_b, bar);
                }
            }
            return true;
        };
        bool ok = true;
        for (int t = pair; t < all && ok; t += pairs) {
            if constexpr (Second::kAny)
                if (t >= items) { ok = copy(second, plan2.at(t - items)); continue; }
            ok = copy(first, plan.at(t));
        }
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- products ----
        unsigned used = 0;                                       // k-blocks consumed
        int count = 0;
        auto multiply = [&](const auto& product, const TileAt at) {
            using P = std::decay_t<decltype(product)>;
            // accumulators binary32, inputs fp16 or bf16, N / 8 in bits 17-22, M / 16 in bits 24-28
            const unsigned in = P::Ops::kBf16 ? 1u : 0u;
            const unsigned idesc = (1u << 4) | (in << 7) | (in << 10) | ((P::kMnA ? 1u : 0u) << 15) | ((P::kMnB ? 1u : 0u) << 16) |
                                   ((unsigned)(TN / 8) << 17) | ((unsigned)(kTileM / 16) << 24);
            const int chunks = chunks_of<P::Ops::kLong>(at);
            for (int c = 0; c < chunks; ++c, ++count) {
                const int slot = count & 1;
                if (!mbar_wait(smem_u32(&acc_empty[slot]), ((count >> 1) & 1) ^ 1, &abort_flag, budget)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned d = tmem + (unsigned)slot * 256u;
                const long long n = at.k1 - at.k0;
                const int k0 = at.k0 + (int)(n * c / chunks), k1 = at.k0 + (int)(n * (c + 1) / chunks);
                for (int k = k0; k < k1; ++k, ++used) {
                    const int s = used % kStages;
                    if (!mbar_wait(smem_u32(&full[s]), (used / kStages) & 1u, &abort_flag, budget)) return false;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned a = ring + s * kStageBytes;
                    const unsigned long long da = mat_desc(a, P::kMnA), db = mat_desc(a + kOperandBytes, P::kMnB);
#pragma unroll
                    for (int i = 0; i < kTileK / 16; ++i)
                        mma_pair(d, da + (P::kMnA ? 128 * i : 2 * i), db + (P::kMnB ? 128 * i : 2 * i), idesc, k > k0 || i > 0);
                    mma_commit_pair(smem_u32(&empty[s]));
                }
                mma_commit_pair(smem_u32(&acc_full[slot]));
            }
            return true;
        };
        bool ok = true;
        for (int t = pair; t < all && ok; t += pairs) {
            if constexpr (Second::kAny)
                if (t >= items) { ok = multiply(second, plan2.at(t - items)); continue; }
            ok = multiply(first, plan.at(t));
        }
        if (!ok) {
            mma_commit_pair(smem_u32(&drain));
            const long long t0 = clock64();
            while (!mbar_try(smem_u32(&drain), 0) && clock64() - t0 < budget) {}
        }
    } else if (warp >= 2) {
        // ---- epilogue ----
        const int quarter = warp & 3;                            // the TMEM lanes this warp may read
        const int half = (warp - 2) >> 2;
        const int row = (int)rank * kHalf + quarter * 32 + lane;
        const unsigned staging = ring + kStages * kStageBytes + (warp - 2) * kStagingBytes;
        constexpr int kColumns = TN / 2 < 32 ? 32 : TN / 2;       // a narrow tile is all the first half's
        int count = 0;
        auto finish = [&](const auto& product, const TilePlan& tiles, const auto& once, const TileAt at) {
            const auto prepared = product.ops.prepare(tiles, at, row);
            float v[kColumns];
            auto take = [&](const bool first_sum) {
                const int slot = count & 1;
                const bool ok = mbar_wait(smem_u32(&acc_full[slot]), (count >> 1) & 1, &abort_flag, budget);
                if (!__all_sync(0xffffffffu, ok)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned from = tmem + (unsigned)(slot * 256 + half * kColumns) + ((unsigned)(quarter * 32) << 16);
                if (first_sum) tmem_read<kColumns>(from, v);
                else tmem_add<kColumns>(from, v);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(pair_leader_addr(smem_u32(&acc_empty[slot])));
                ++count;
                return true;
            };
            if (!take(true)) return false;
            using Ops = typename std::decay_t<decltype(product)>::Ops;
            if constexpr (Ops::kLong)
                for (int c = chunks_of<true>(at); c > 1; --c)
                    if (!take(false)) return false;
            if (at.k0 == at.k1) {
#pragma unroll
                for (int j = 0; j < kColumns; ++j) v[j] = 0.0f;
            }
            product.ops.epilogue(tiles, at, row, v, half, staging, once, prepared);
            return true;
        };
        const auto once = first.ops.once(plan);
        const auto once2 = [&] {
            if constexpr (Second::kAny) return second.ops.once(plan2);
            else return Nothing{};
        }();
        bool ok = true;
        int t = pair;
        for (; t < all && ok; t += pairs) {
            if constexpr (Second::kAny)
                if (t >= items) { ok = finish(second, plan2, once2, plan2.at(t - items)); continue; }
            ok = finish(first, plan, once, plan.at(t));
        }
        if (!ok) {
            t -= pairs;                                          // the turn that did not end; its tile is this warp's alone
            bool of_second = false;
            if constexpr (Second::kAny) of_second = t >= items;
            if (!of_second) first.ops.gave_up(plan, plan.at(t), row, half);
            if constexpr (Second::kAny)
                if (of_second) second.ops.gave_up(plan2, plan2.at(t - items), row, half);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
