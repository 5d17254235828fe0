// gm_linear_xent.cu -- softmax cross entropy over a large vocabulary, straight from hidden
// states X [N, D] and table W [V, D], without the logits in memory, and both gradients.
//
//   l = X W^T,  lse_n = log sum_v exp l_nv,  loss_n = lse_n - l_{n, t_n}
//   S = softmax(l) - onehot(t),  dX = c S W,  dW = c S^T X,  c = grad_scale * scale / count
//
// Forward: one matrix product whose epilogue leaves, per row and 128 vocabulary entries, the
// maximum and the sum of exponentials (8 bytes for 128 logits) of all entries but
// the target's, then a small kernel joins them with the target's logit, which comes from a dot
// product of its own.  loss = log(1 + sum of the others / the target's) then keeps its relative
// accuracy when the model is sure of the target, and the target's logit is as good as binary32 makes it (the
// tensor cores cut where they add; the other logits' long sums are taken in parts for that).  Backward: for one
// piece of the vocabulary after the other the logits are formed again, the target's entry of S comes from its
// binary32 logit as in the forward pass, S goes to the workspace in 16 bits, and two products take it from
// there; dX is carried from piece to piece in binary32.  8 N D V operations for a training step: 2
// forward, 2 again for the logits, 4 for the gradients.  Bound by the tensor cores, for a few
// rows by the read of W.
//
// Rows whose target lies outside the vocabulary are left out before all this: an index of the
// others is built on the device, their hidden states are gathered into the workspace, and the
// products see only those.  They cost nothing, and what they hold (padding, NaN) goes nowhere.
//
// Roundings: S is rounded once to the inputs' type, as the operand of a tensor-core product
// has to be.  In fp16 it is first multiplied by 2^15 (|S| <= 1), which keeps probabilities
// down to 2^-29 normal, in bf16 by 2^32, so that the exponential's flush to zero at 2^-126 lies
// below what bf16 holds; the factor is taken out in binary32 in the epilogue.
#include <mutex>

#include "gm_tile_gemm.cuh"

namespace gm {

constexpr int kXentStatusWord = 48;      // of the device's scalars: 1 when a wait of a product ran out
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Half16;
template <> struct Half16<__half> { static constexpr bool kBf16 = false; static constexpr float kUp = 32768.0f, kUpLog2 = 15.0f; };
template <> struct Half16<__nv_bfloat16> { static constexpr bool kBf16 = true; static constexpr float kUp = 4294967296.0f, kUpLog2 = 32.0f; };

// Scalars at the workspace's begin.
struct XentScalars {
    int count;                // rows with a target
    unsigned ticket;
};

__device__ __forceinline__ int up_to(int x, int m) { return (x + m - 1) / m * m; }

// 2^x, results below 2^-126 as zero (PTX ex2.approx.ftz: two units in the last place).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---------------------------------------------------------------- index and gather
// rows[i] = the i-th row with a target, target[i] = that target.  One CTA: eight rows per
// thread and turn, a prefix sum over the CTA.
constexpr int kIndexThreads = 1024;
__global__ void __launch_bounds__(kIndexThreads)
xent_index_kernel(const int* __restrict__ targets, const int n, const int vocab, int* __restrict__ rows, int* __restrict__ target,
                  XentScalars* __restrict__ sc) {
    __shared__ int warp_sum[32];
    __shared__ int carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool wide = (reinterpret_cast<uintptr_t>(targets) & 15) == 0;
    chain_begin();
    if (tid == 0) carry = 0;
    __syncthreads();
    for (long long base = 0; base < n; base += kIndexThreads * 8) {
        int t[8];
        int mine = 0;
        const long long i0 = base + tid * 8;
        if (wide && i0 + 8 <= n) {
            const int4 a = __ldg(reinterpret_cast<const int4*>(targets + i0)), b = __ldg(reinterpret_cast<const int4*>(targets + i0) + 1);
            t[0] = a.x; t[1] = a.y; t[2] = a.z; t[3] = a.w; t[4] = b.x; t[5] = b.y; t[6] = b.z; t[7] = b.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = i0 + k < n ? __ldg(targets + i0 + k) : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (t[k] >= vocab) t[k] = -1;
            mine += t[k] >= 0;
        }
        int scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += x;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        if (warp == 0) {
            int s = warp_sum[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += x;
            }
            warp_sum[lane] = s;
        }
        __syncthreads();
        int at = carry + scan - mine + (warp > 0 ? warp_sum[warp - 1] : 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (t[k] >= 0) {
                rows[at] = (int)(base + tid * 8 + k);
                target[at] = t[k];
                ++at;
            }
        __syncthreads();
        if (tid == 0) carry += warp_sum[31];
        __syncthreads();
    }
    if (tid == 0) { sc->count = carry; sc->ticket = 0u; }
}

// The same for at most kFewIndex rows inside the gathering kernel: every CTA counts the targets
// for itself and finds the row that is its own.  Saves a launch where a call is mostly launches.
constexpr int kGatherThreads = 128;
constexpr int kFewIndex = kGatherThreads * 16;
__device__ __forceinline__ void find_row(const int* __restrict__ targets, const int n, const int vocab, const int r, int* count, int* row, int* target) {
    __shared__ int warp_count[kGatherThreads / 32], found[2];
    const int tid = threadIdx.x, lane = tid & 31;
    const int per = (n + kGatherThreads - 1) / kGatherThreads;         // at most 16, consecutive
    unsigned live = 0;
    for (int k = 0; k < per; ++k) {
        const int i = tid * per + k;
        const int t = i < n ? __ldg(targets + i) : -1;
        if (t >= 0 && t < vocab) live |= 1u << k;
    }
    int scan = __popc(live);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += x;
    }
    if (lane == 31) warp_count[tid >> 5] = scan;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kGatherThreads / 32; ++w) {
        if (w < (tid >> 5)) scan += warp_count[w];
        total += warp_count[w];
    }
    int at = scan - __popc(live);                                      // rows in front of this thread's
    if (r >= at && r < scan) {
        for (int k = 0; k < per; ++k)
            if ((live >> k) & 1u) {
                if (at == r) { found[0] = tid * per + k; found[1] = __ldg(targets + tid * per + k); }
                ++at;
            }
    }
    __syncthreads();
    *count = total;
    *row = r < total ? found[0] : 0;
    *target = r < total ? found[1] : 0;
}

// A target's logit, the dot product of its hidden state and its row of W in binary32.  Both passes take it
// in the same order, 128 threads with eight columns each at a time (VEC: the hidden state begins on a
// 16-byte boundary, as the table's rows do), so that the backward pass has the forward pass's bits.
constexpr int kDotThreads = kGatherThreads;
template <typename T>
__device__ __forceinline__ void dot_eight(const Raw8<T>& x, const T* w, float* dot) {
    float a[8], b[8];
    widen8<T>(x, a);
    widen8<T>(load8<T, true>(w), b);
#pragma unroll
    for (int k = 0; k < 8; ++k) *dot = fmaf(a[k], b[k], *dot);
}
template <typename T>
__device__ __forceinline__ float dot_share(const T* x, const T* w, const int dim, const bool vec, const int tid) {
    float dot = 0.0f;
    const int groups = vec ? dim >> 3 : 0;
    for (int g = tid; g < groups; g += kDotThreads) dot_eight<T>(load8<T, false>(x + g * 8), w + g * 8, &dot);
    for (int c = groups * 8 + tid; c < dim; c += kDotThreads) dot = fmaf(to_f32<T>(x[c]), to_f32<T>(w[c]), dot);
    return dot;
}

// Gathers the hidden states of the rows with a target, zeroes the rows behind them up to a
// whole tile, and clears the outputs of rows without a target.  One CTA per row.  It also takes the logit z of
// the row's target, and leaves that (forward), or, given the rows' log-sum-exp (backward), the target's entry
// of softmax - onehot, exp(z - lse) - 1.
template <typename T>
__global__ void __launch_bounds__(kGatherThreads)
xent_gather_kernel(const T* __restrict__ hidden, const long long ld, const int n, const int dim, const int vocab, const int* __restrict__ targets,
                   int* rows, int* target, XentScalars* sc, const bool few, T* __restrict__ packed,
                   const long long ld_packed, const T* __restrict__ weight, const long long ld_weight, float* __restrict__ of_target,
                   const float* __restrict__ lse_given, float* __restrict__ losses, float* __restrict__ lse, T* __restrict__ dhidden, const bool vec,
                   const bool vec_out) {
    __shared__ float warp_sum[kGatherThreads / 32];
    const int r = blockIdx.x, tid = threadIdx.x;
    chain_begin();
    int count, row, goal;
    if (few) {
        find_row(targets, n, vocab, r, &count, &row, &goal);
        if (tid == 0) {
            if (r < count) { rows[r] = row; target[r] = goal; }
            if (r == 0) { sc->count = count; sc->ticket = 0u; }
        }
    } else {
        count = sc->count;
        row = r < count ? rows[r] : 0;
        goal = r < count ? target[r] : 0;
    }
    const int groups = dim >> 3;
    const T zero = from_f32<T>(0.0f);
    if (r < n) {
        const int t = __ldg(targets + r);
        if (t < 0 || t >= vocab) {
            if (losses && tid == 0) { losses[r] = 0.0f; lse[r] = 0.0f; }
            if (dhidden) {
                T* to = dhidden + (long long)r * ld;
                const int from = vec_out ? groups * 8 : 0;
                if (vec_out)
                    for (int g = tid; g < groups; g += kGatherThreads) *reinterpret_cast<uint4*>(to + g * 8) = make_uint4(0u, 0u, 0u, 0u);
                for (int c = from + tid; c < dim; c += kGatherThreads) to[c] = zero;
            }
        }
    }
    if (r >= up_to(count, kTileM)) return;
    T* to = packed + (long long)r * ld_packed;
    if (r >= count) {
        for (int c = tid; c < dim; c += kGatherThreads) to[c] = zero;
        return;
    }
    const T* from = hidden + (long long)row * ld;
    const T* w = weight + (long long)goal * ld_weight;
    const float norm = lse_given ? __ldg(lse_given + row) : 0.0f;
    float dot = 0.0f;                                                  // as dot_share takes it
    int c0 = 0;
    if (vec) {
        c0 = groups * 8;
        for (int g = tid; g < groups; g += kGatherThreads) {
            const Raw8<T> x = load8<T, false>(from + g * 8);
            *reinterpret_cast<uint4*>(to + g * 8) = x.a;
            dot_eight<T>(x, w + g * 8, &dot);
        }
    }
    for (int c = c0 + tid; c < dim; c += kGatherThreads) {
        to[c] = from[c];
        dot = fmaf(to_f32<T>(from[c]), to_f32<T>(w[c]), dot);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if ((tid & 31) == 0) warp_sum[tid >> 5] = dot;
    __syncthreads();
    if (tid == 0) {
        for (int k = 1; k < kGatherThreads / 32; ++k) dot += warp_sum[k];
        of_target[r] = lse_given ? expm1f(dot - norm) : dot;
    }
}

// ---------------------------------------------------------------- epilogues
// The exponentials of a piece are 2^(scale l - ref) with scale = log2e and ref = m log2e rounded, one operation
// each; their sum is then relative to 2^ref, not to e^m, and those are apart by the rounding of ref (up to 11 units
// in the last place at m = 20, a hundred at 200).  off() takes it out, once per piece.
// Where m log2e would pass binary32 (a piece of nothing but bf16's lowest number, as masks have it) scale is 1 and ref is m:
// logits of that size are equal to m or 1e31 and more below it, so any base gives 1 and 0.  A piece of nothing
// but -inf has zeros.
struct Reference {
    float m, scale, ref;
    __device__ __forceinline__ explicit Reference(const float top)
        : m(top), scale(fabsf(top) > 2e38f ? 1.0f : kLog2e), ref(top == -INFINITY ? 0.0f : top * scale) {}
    __device__ __forceinline__ float off() const { return m == -INFINITY ? 1.0f : exp2f(-fmaf(m, scale, -ref)); }
};

constexpr int kGroupM = 8;      // m-tiles walked together in the gradient products

// Row maximum and sum of exponentials of half a tile's logits (128), the target's left out.
struct Goal { int at; };        // a row's target
// LONG: for more than kOneSum columns.
template <typename T, bool LONG>
struct StatsOps {
    static constexpr bool kBf16 = Half16<T>::kBf16;
    static constexpr bool kStaging = false;
    static constexpr bool kLong = LONG;
    __device__ __forceinline__ void begin() const {}
    __device__ __forceinline__ int rows_a() const { return kHalf; }
    const XentScalars* sc;
    const int* target;
    float2* stats;               // [128 vocabulary entries][row]
    int rows_cap, dim, vocab, group, a0, b0;
    __device__ __forceinline__ TilePlan plan(int) const {
        const int count = sc->count;
        return whole_tiles(count, (count + kTileM - 1) / kTileM, (vocab + kTileN - 1) / kTileN, (dim + kTileK - 1) / kTileK, group);
    }
    __device__ __forceinline__ Nothing once(const TilePlan&) const { return {}; }
    __device__ __forceinline__ void gave_up(const TilePlan&, const TileAt&, int, int) const {}     // the status is read behind it
    __device__ __forceinline__ Goal prepare(const TilePlan& plan, const TileAt& tile, int in_tile) const {
        const int row = tile.m * kTileM + in_tile;
        return {row < plan.count ? __ldg(target + row) - tile.n * kTileN : -1};
    }
    __device__ __forceinline__ void epilogue(const TilePlan& plan, const TileAt& tile, int in_tile, float (&v)[128], int half, unsigned, Nothing,
                                             const Goal goal) const {
        const int row = tile.m * kTileM + in_tile;
        const int width = vocab - tile.n * kTileN - half * 128;           // columns that exist
        if (width <= 0) return;
        if (width < 128) {
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (j >= width) v[j] = -INFINITY;
        }
        const int at = goal.at - half * 128;
        if ((unsigned)at < 128u) {
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (at == j) v[j] = -INFINITY;
        }
        float top[8], sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { top[j] = v[j]; sum[j] = 0.0f; }
#pragma unroll
        for (int j = 8; j < 128; ++j) top[j & 7] = fmaxf(top[j & 7], v[j]);
        const float m = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), fmaxf(fmaxf(top[4], top[5]), fmaxf(top[6], top[7])));
        const Reference r(m);
#pragma unroll
        for (int j = 0; j < 128; ++j) sum[j & 7] += exp2_fast(fmaf(v[j], r.scale, -r.ref));
        const float s = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
        if (row < plan.count) stats[(long long)(2 * tile.n + half) * rows_cap + row] = make_float2(m, s * r.off());
    }
};

// The same for a few rows (at most TN): the vocabulary takes the tile's long side, up to 256 entries by
// TN rows, so that nothing but the read of W is left.  `height` entries per CTA are chosen so that
// all pairs have the same share of the vocabulary.  Rows without a target are multiplied like the
// others, and nothing reads what comes of them.  A warp holds 32 entries of 32 rows at a time, one
// entry per lane, and reduces over its lanes by halving exchanges, after which lane j has row j: one
// {maximum, sum} per warp and row.
template <bool MAX> __device__ __forceinline__ float lanes_to_columns(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float keep = upper ? v[i + o] : v[i], send = upper ? v[i] : v[i + o];
            const float got = __shfl_xor_sync(0xffffffffu, send, o);
            v[i] = MAX ? fmaxf(keep, got) : keep + got;
        }
    }
    return v[0];
}

template <typename T, int TN, bool LONG>
struct FewStatsOps {
    static constexpr bool kBf16 = Half16<T>::kBf16;
    static constexpr bool kStaging = false;
    static constexpr bool kLong = LONG;
    static constexpr int kColumns = TN / 2 < 32 ? 32 : TN / 2;
    XentScalars* sc;
    const int* target;           // by row of the caller
    float2* stats;               // [warp's share of a tile][row]
    int n, rows_cap, dim, vocab, height, a0, b0;
    __device__ __forceinline__ void begin() const { sc->ticket = 0u; }
    __device__ __forceinline__ int rows_a() const { return height; }
    __device__ __forceinline__ TilePlan plan(int) const {
        return whole_tiles(n, (vocab + 2 * height - 1) / (2 * height), 1, (dim + kTileK - 1) / kTileK, 1);
    }
    __device__ __forceinline__ Nothing once(const TilePlan&) const { return {}; }
    __device__ __forceinline__ void gave_up(const TilePlan&, const TileAt&, int, int) const {}     // the status is read behind it
    __device__ __forceinline__ Goal prepare(const TilePlan&, const TileAt&, int) const { return {0}; }
    __device__ __forceinline__ void epilogue(const TilePlan&, const TileAt& tile, int in_tile, float (&all)[kColumns], int half, unsigned, Nothing, const Goal) const {
        const int cta = in_tile / kHalf, local = in_tile % kHalf, lane = threadIdx.x & 31;
        const int base = (tile.m * 2 + cta) * height + (local & ~31);      // entry of the warp's first lane
        const bool real = local < height && base + lane < vocab;
        if (half * kColumns >= TN) return;
        float2* to = stats + (long long)(tile.m * 8 + in_tile / 32) * rows_cap;
#pragma unroll
        for (int q = 0; q < kColumns; q += 32) {
            const int c = half * kColumns + q;
            if (c >= n) break;
            float v[32], w[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = real ? all[q + j] : -INFINITY;
            const int goal = c + lane < n ? __ldg(target + c + lane) : -1;
            for (unsigned hits = __ballot_sync(0xffffffffu, goal >= base && goal < base + 32); hits; hits &= hits - 1) {
                const int j = __ffs((int)hits) - 1;
                const bool mine = __shfl_sync(0xffffffffu, goal, j) == base + lane;
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    if (k == j && mine) v[k] = -INFINITY;              // the target's logit is added by itself
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j] = v[j];
            const float top = lanes_to_columns<true>(w, lane);
            const Reference r(top);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                v[j] = exp2_fast(fmaf(v[j], __shfl_sync(0xffffffffu, r.scale, j), -__shfl_sync(0xffffffffu, r.ref, j)));
            const float sum = lanes_to_columns<false>(v, lane);
            if (c + lane < n) to[c + lane] = make_float2(top, sum * r.off());
        }
    }
};

// S of one tile, rounded to 16 bits, into the workspace; zeros behind the last row and column.  The target's
// entry comes from its binary32 logit (xent_gather_kernel).  From the product's it would be a difference of nearly
// equal numbers for a model that is sure: the tensor cores cut where they add, the log-sum-exp does not go along,
// and where p is 0.999 with a logit of 13 it was off by 35 % at 4,096 columns and by 70 % at 8,192, always to the same
// side.  What is left is the rounding of the log-sum-exp: at most half a unit in its last place, and no wrong sign.
template <typename T>
struct SoftmaxGradOps {
    static constexpr bool kBf16 = Half16<T>::kBf16;
    static constexpr bool kStaging = true;
    static constexpr bool kLong = false;
    __device__ __forceinline__ void begin() const {}
    __device__ __forceinline__ int rows_a() const { return kHalf; }
    const XentScalars* sc;
    const int* target;
    const int* rows;
    const float* lse;            // by row of the caller
    const float* own;            // the targets' entries, by row
    CUtensorMap ds;
    int dim, v0, v1, group, a0, b0;
    static constexpr int kNoRow = INT_MIN;   // `at` of a row behind the last one
    struct Row { int at; float ref; };       // target in the tile; log2 of what the row's exponentials are divided by
    __device__ __forceinline__ TilePlan plan(int) const {
        const int count = sc->count;
        return whole_tiles(count, (count + kTileM - 1) / kTileM, (v1 - v0 + kTileN - 1) / kTileN, (dim + kTileK - 1) / kTileK, group);
    }
    __device__ __forceinline__ Nothing once(const TilePlan&) const { return {}; }
    __device__ __forceinline__ void gave_up(const TilePlan&, const TileAt&, int, int) const {}     // the status is read behind it
    __device__ __forceinline__ Row prepare(const TilePlan& plan, const TileAt& tile, int in_tile) const {
        const int row = tile.m * kTileM + in_tile;
        if (row >= plan.count) return {kNoRow, 0.0f};
        return {__ldg(target + row) - v0 - tile.n * kTileN, fmaf(__ldg(lse + __ldg(rows + row)), kLog2e, -Half16<T>::kUpLog2)};
    }
    __device__ __forceinline__ void epilogue(const TilePlan& plan, const TileAt& tile, int in_tile, float (&v)[128], int half, unsigned stage, Nothing,
                                             const Row row) const {
        const int first_row = tile.m * kTileM + (in_tile & ~31);
        if (first_row >= up_to(plan.count, kTileK)) return;               // dW's sum ends there, and nothing takes what dX makes of such rows
#pragma unroll
        for (int j = 0; j < 128; ++j) v[j] = exp2_fast(fmaf(v[j], kLog2e, -row.ref));
        const int at = row.at == kNoRow ? -1 : row.at - half * 128;
        if ((unsigned)at < 128u) {
            const float x = __ldg(own + tile.m * kTileM + in_tile) * Half16<T>::kUp;
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (at == j) v[j] = x;
        }
        if (row.at == kNoRow) {                                           // whatever its logits: 0 times an infinity of the table is NaN
#pragma unroll
            for (int j = 0; j < 128; ++j) v[j] = 0.0f;
        }
        const int width = v1 - v0 - tile.n * kTileN - half * 128;        // columns that exist, the others are zeros
        if (width < 128) {
#pragma unroll
            for (int j = 0; j < 128; ++j)
                if (j >= width) v[j] = 0.0f;
        }
        rows_to_memory<T>(stage, v, 128, &ds, tile.n * kTileN + half * 128, first_row);
    }
};

// What both gradient products multiply by.  NaN once a wait has run out, in this call or before: an optimizer
// step that follows without a look at the status then finds a gradient that it must not take.
struct GradScale {
    const int* status;
    const float* scale;          // device scalar (the loss scale), or null
    float grad_scale;
    int mean;
    float down;                  // takes out the factor S carries
    __device__ __forceinline__ float value(int count) const {
        float c = scale ? __fmul_rn(grad_scale, *scale) : grad_scale;
        if (mean) c = __fdiv_rn(c, (float)(count > 0 ? count : 1));
        if (*(const volatile int*)status) c = NAN;
        return c * down;
    }
};

// Four columns of a row in a 16-bit type, `cols` of which exist.
template <typename T>
__device__ __forceinline__ float4 get4(const T* from, int cols, bool vec) {
    if (vec && cols >= 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(from);
        const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < cols) v[j] = to_f32<T>(from[j]);
    return make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void put4(T* to, const float4 x, int cols, bool vec) {
    if (vec && cols >= 4) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    } else {
        const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < cols) to[j] = from_f32<T>(v[j]);
    }
}

// dX: S [rows, piece] times W [piece, D]; carried in binary32 over the pieces, scattered to the
// caller's rows by the last one.  A share of K goes to `parts` instead, 256 x 256 numbers per
// turn, and xent_hidden_join_kernel does the rest.
struct HiddenPlan {
    int dim, v0, v1, most_parts;
    __device__ __forceinline__ TilePlan plan(int count, int pairs) const {
        TilePlan p = whole_tiles(count, (count + kTileM - 1) / kTileM, (dim + kTileN - 1) / kTileN, (v1 - v0 + kTileK - 1) / kTileK, kGroupM);
        split_tail(&p, pairs, most_parts);
        return p;
    }
};

template <typename T>
struct HiddenOut {
    float* carried;
    long long ld_carried;
    T* out;
    long long ld_out;
    GradScale scale;
    bool first, last, vec;
    // four columns from c of one row: what was carried, and that with more on top carried on or written
    __device__ __forceinline__ float4 get(int row, int c) const {
        return first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *reinterpret_cast<const float4*>(carried + (long long)row * ld_carried + c);
    }
    __device__ __forceinline__ void put(int row, int to_row, int c, float4 x, const float4 old, int cols, float c_all) const {
        float* acc = carried + (long long)row * ld_carried + c;
        x = make_float4(__fadd_rn(old.x, x.x), __fadd_rn(old.y, x.y), __fadd_rn(old.z, x.z), __fadd_rn(old.w, x.w));
        if (last)
            put4<T>(out + (long long)to_row * ld_out + c, make_float4(__fmul_rn(x.x, c_all), __fmul_rn(x.y, c_all), __fmul_rn(x.z, c_all), __fmul_rn(x.w, c_all)),
                    cols, vec);
        else *reinterpret_cast<float4*>(acc) = x;
    }
};

template <typename T>
struct HiddenGradOps {
    static constexpr bool kBf16 = Half16<T>::kBf16;
    static constexpr bool kStaging = true;
    static constexpr bool kLong = false;
    __device__ __forceinline__ void begin() const {}
    __device__ __forceinline__ int rows_a() const { return kHalf; }
    const XentScalars* sc;
    const int* rows;
    float* parts;
    HiddenPlan shape;
    HiddenOut<T> out;
    int a0, b0;
    __device__ __forceinline__ TilePlan plan(int pairs) const { return shape.plan(sc->count, pairs); }
    __device__ __forceinline__ float once(const TilePlan& plan) const { return out.scale.value(plan.count); }
    __device__ __forceinline__ void gave_up(const TilePlan& plan, const TileAt& tile, int in_tile, int half) const {
        const int row = tile.m * kTileM + in_tile, col = tile.n * kTileN + half * 128;
        if (row >= plan.count || col >= shape.dim) return;
        if (tile.part >= 0) parts[(long long)tile.part * (kTileM * kTileN) + in_tile * kTileN + half * 128] = NAN;
        else if (out.last) out.out[(long long)rows[row] * out.ld_out + col] = from_f32<T>(NAN);
        else out.carried[(long long)row * out.ld_carried + col] = NAN;
    }
    // the caller's row, -1 behind the last one
    __device__ __forceinline__ int prepare(const TilePlan& plan, const TileAt& tile, int in_tile) const {
        const int row = tile.m * kTileM + in_tile;
        return row < plan.count ? __ldg(rows + row) : -1;
    }
    __device__ __forceinline__ void epilogue(const TilePlan& plan, const TileAt& tile, int in_tile, float (&v)[128], int half, unsigned stage,
                                             const float c_all, const int to) const {
        const int col = tile.n * kTileN + half * 128, cols = shape.dim - col;
        const int first_row = tile.m * kTileM + (in_tile & ~31);
        if (tile.part >= 0) {
            float* part = parts + (long long)tile.part * (kTileM * kTileN) + (in_tile & ~31) * kTileN + half * 128;
            if (first_row < plan.count)
                rows_by_fours(stage, v, cols, 0, [](int, int, int) { return 0; },
                              [&](int r, int, int c, float4 x, int) { *reinterpret_cast<float4*>(part + r * kTileN + c) = x; });
        } else {
            rows_by_fours(stage, v, cols, to,
                          [&](int r, int to_row, int c) { return to_row >= 0 ? out.get(first_row + r, col + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f); },
                          [&](int r, int to_row, int c, float4 x, const float4 old) {
                              if (to_row >= 0) out.put(first_row + r, to_row, col + c, x, old, cols - c, c_all);
                          });
        }
    }
};

// Adds up the shares of K of the tiles that were split, in order; one thread per row and four columns.
template <typename T>
__global__ void __launch_bounds__(256)
xent_hidden_join_kernel(const XentScalars* __restrict__ sc, const int* __restrict__ rows, const float* __restrict__ parts, const HiddenPlan shape,
                        const HiddenOut<T> out, const int pairs) {
    chain_begin();
    const int count = sc->count;
    const TilePlan plan = shape.plan(count, pairs);
    const float c_all = out.scale.value(count);
    constexpr int kPerTile = kTileM * kTileN / 4;
    const int work = (plan.tiles() - plan.whole) * kPerTile;             // at most kMostParts tiles
    for (int i = blockIdx.x * 256 + threadIdx.x; i < work; i += gridDim.x * 256) {
        const int tile = i / kPerTile, r = i % kPerTile / (kTileN / 4), c = i % (kTileN / 4) * 4;
        int m, n;
        plan.place(plan.whole + tile, &m, &n);
        const int row = m * kTileM + r, col = n * kTileN + c;
        if (row >= count || col >= shape.dim) continue;
        const int to_row = __ldg(rows + row);
        const float4* p = reinterpret_cast<const float4*>(parts + (long long)tile * plan.splits * (kTileM * kTileN) + r * kTileN + c);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int s = 0; s < plan.splits; ++s) {
            const float4 x = __ldcs(p + s * kPerTile);
            sum = make_float4(__fadd_rn(sum.x, x.x), __fadd_rn(sum.y, x.y), __fadd_rn(sum.z, x.z), __fadd_rn(sum.w, x.w));
        }
        out.put(row, to_row, col, sum, out.get(row, col), shape.dim - col, c_all);
    }
}

// dW of a piece: S^T [piece, rows] times X [rows, D].  MAP: not added to what is there, and stored by
// TMA, which writes the last 16 bytes of a row whole: the columns have to be a multiple of eight.
template <typename T, bool MAP>
struct WeightGradOps {
    static constexpr bool kBf16 = Half16<T>::kBf16;
    static constexpr bool kStaging = true;
    static constexpr bool kLong = false;
    __device__ __forceinline__ void begin() const {}
    __device__ __forceinline__ int rows_a() const { return kHalf; }
    const XentScalars* sc;
    CUtensorMap to;              // of the caller's gradient, with MAP
    T* out;
    long long ld_out;
    GradScale scale;
    int dim, v0, v1, a0, b0;
    bool add, vec;               // vec: rows begin on 16-byte boundaries
    __device__ __forceinline__ TilePlan plan(int) const {
        const int count = sc->count;
        return whole_tiles(count, (v1 - v0 + kTileM - 1) / kTileM, (dim + kTileN - 1) / kTileN, (count + kTileK - 1) / kTileK, kGroupM);
    }
    __device__ __forceinline__ float once(const TilePlan& plan) const { return scale.value(plan.count); }
    __device__ __forceinline__ void gave_up(const TilePlan&, const TileAt& tile, int in_tile, int half) const {
        const int row = tile.m * kTileM + in_tile, col = tile.n * kTileN + half * 128;
        if (row < v1 - v0 && col < dim) out[(long long)(v0 + row) * ld_out + col] = from_f32<T>(NAN);
    }
    __device__ __forceinline__ Nothing prepare(const TilePlan&, const TileAt&, int) const { return {}; }
    __device__ __forceinline__ void epilogue(const TilePlan&, const TileAt& tile, int in_tile, float (&v)[128], int half, unsigned stage,
                                             const float c_all, Nothing) const {
        const int col = tile.n * kTileN + half * 128, cols = dim - col;
        const int first_row = tile.m * kTileM + (in_tile & ~31), rows = v1 - v0 - first_row;
        if (rows <= 0) return;
        T* first = out + (long long)(v0 + first_row) * ld_out + col;
#pragma unroll
        for (int j = 0; j < 128; ++j) v[j] = __fmul_rn(v[j], c_all);
        if constexpr (MAP) rows_to_memory<T>(stage, v, cols, &to, col, v0 + first_row);      // a last piece's rows end with the map
        else
            rows_by_fours(stage, v, cols, 0,
                          [&](int r, int, int c) {
                              return add && r < rows ? get4<T>(first + r * ld_out + c, cols - c, vec) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                          },
                          [&](int r, int, int c, const float4 x, const float4 old) {
                              const float4 y = make_float4(__fadd_rn(old.x, x.x), __fadd_rn(old.y, x.y), __fadd_rn(old.z, x.z), __fadd_rn(old.w, x.w));
                              if (r < rows) put4<T>(first + r * ld_out + c, y, cols - c, vec);
                          });
    }
};

// ---------------------------------------------------------------- joining the row statistics
// By differences of the maxima, so that the side that holds the larger one keeps its sum as it is: a row is
// joined some tens of times, and any factor but 1 there would be an error that many times over.
struct MaxSum { float m, s; };                       // sum of exponentials relative to the maximum
__device__ __forceinline__ MaxSum joined(const MaxSum a, const MaxSum b) {
    const float m = fmaxf(a.m, b.m);
    const float fa = a.m == m ? 1.0f : exp2f((a.m - m) * kLog2e), fb = b.m == m ? 1.0f : exp2f((b.m - m) * kLog2e);
    return {m, fmaf(a.s, fa, b.s * fb)};
}

// Loss and log-sum-exp of a row whose target's logit is z and whose other entries are `a`.  The loss is
// taken as the logarithm of a sum, not as a difference, so a small loss is as good, relatively, as that sum
// (3.5e-7 with 131,072 entries around 200).  A target with
// logit -inf has an infinite loss, and a log-sum-exp that is its other entries'; with logit +inf both
// the loss and its gradient are NaN, as inf - inf is.
struct RowLoss { float loss, lse; };
__device__ __forceinline__ RowLoss row_loss(const float z, const MaxSum a) {
    if (z >= a.m) {
        const float loss = log1pf(a.s * expf(a.m - z)) + (z - z);
        return {loss, z + loss};
    }
    const float rest = logf(a.s + expf(z - a.m));
    return {(a.m - z) + rest, z == -INFINITY ? a.m + rest : z + ((a.m - z) + rest)};
}

// A CTA takes ROWS rows with 256 / ROWS lanes over the vocabulary's pieces; the CTA that finishes
// last adds up the loss.  ROWS is 8 (64 bytes of neighbouring rows; with 32 the walk over the pieces
// is 4 times as long and took 17 us instead of 9 at 1,640 rows), or 1 in a small call.
template <int ROWS>
__global__ void __launch_bounds__(256)
xent_join_kernel(XentScalars* sc, const float2* __restrict__ stats, const int rows_cap, const int tiles, const float* __restrict__ of_target,
                 const int* __restrict__ rows, float* __restrict__ losses, float* __restrict__ lse, float* partial, float* __restrict__ total,
                 const int mean, const int* status) {
    constexpr int WAYS = 256 / ROWS;
    __shared__ MaxSum part[WAYS][ROWS];
    __shared__ int is_last;
    const int x = threadIdx.x % ROWS, y = threadIdx.x / ROWS;
    const int row = blockIdx.x * ROWS + x;
    cudaGridDependencySynchronize();
    const int count = sc->count;
    MaxSum a = {-INFINITY, 0.0f};
    if (row < count) {
        for (int t = y; t < tiles; t += WAYS) {
            const float2 p = __ldcs(stats + (long long)t * rows_cap + row);
            a = joined(a, {p.x, p.y});
        }
    }
    part[y][x] = a;
    for (int o = WAYS / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (y < o) part[y][x] = joined(part[y][x], part[y + o][x]);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        float loss = 0.0f;
        if (y == 0 && row < count) {
            a = part[0][x];
            const RowLoss of = row_loss(of_target[row], a);
            loss = of.loss;
            losses[rows[row]] = loss;
            lse[rows[row]] = of.lse;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        if (threadIdx.x == 0) {
            partial[blockIdx.x] = loss;
            __threadfence();
            is_last = atomicAdd(&sc->ticket, 1u) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!is_last || threadIdx.x >= 32) return;
    __threadfence();
    double sum = 0.0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += 32) sum += (double)((volatile float*)partial)[b];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) {
        if (*status) sum = NAN;                                   // a wait of the product ran out: say so in the result
        total[0] = (float)(mean && count > 0 ? sum / count : sum);
        total[1] = (float)count;
        sc->ticket = 0u;
    }
}

// A few rows: a CTA per row takes the target's logit while the product still runs (it reads only what
// the caller gave), then joins the row's statistics; the last one adds up the loss.
template <typename T>
__global__ void __launch_bounds__(256)
xent_few_join_kernel(XentScalars* sc, const T* __restrict__ hidden, const long long ld, const T* __restrict__ weight, const long long ld_weight,
                     const int* __restrict__ targets, const int dim, const int vocab, const bool vec, const float2* __restrict__ stats, const int rows_cap, const int pieces,
                     float* __restrict__ losses, float* __restrict__ lse, float* partial, float* __restrict__ total, const int mean, const int* status) {
    __shared__ MaxSum part[256];
    __shared__ float dots[kDotThreads / 32];
    __shared__ int is_last;
    const int row = blockIdx.x, n = gridDim.x, tid = threadIdx.x;
    const int goal = __ldg(targets + row);
    const bool live = goal >= 0 && goal < vocab;
    float z = 0.0f;
    if (live && tid < kDotThreads) z = dot_share<T>(hidden + row * ld, weight + goal * ld_weight, dim, vec, tid);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if ((tid & 31) == 0 && tid < kDotThreads) dots[tid >> 5] = z;
    chain_begin();
    MaxSum a = {-INFINITY, 0.0f};
    if (live)
        for (int t = tid; t < pieces; t += 256) {
            const float2 p = __ldcs(stats + (long long)t * rows_cap + row);
            a = joined(a, {p.x, p.y});
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = joined(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
    if ((tid & 31) == 0) part[tid >> 5] = a;
    __syncthreads();
    if (tid == 0) {
        float loss = 0.0f, l = 0.0f;
        if (live) {
            z = dots[0];
            for (int k = 1; k < kDotThreads / 32; ++k) z += dots[k];
            for (int k = 1; k < 8; ++k) a = joined(a, part[k]);
            const RowLoss of = row_loss(z, a);
            loss = of.loss;
            l = of.lse;
        }
        losses[row] = loss;
        lse[row] = l;
        partial[row] = loss;
        __threadfence();
        is_last = atomicAdd(&sc->ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!is_last || tid >= 32) return;
    __threadfence();
    double sum = 0.0;
    int count = 0;
    for (int r = tid; r < n; r += 32) {
        const int t = __ldg(targets + r);
        sum += (double)((volatile float*)partial)[r];
        count += t >= 0 && t < vocab;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(0xffffffffu, sum, o); count += __shfl_xor_sync(0xffffffffu, count, o); }
    if (tid == 0) {
        if (*status) sum = NAN;
        total[0] = (float)(mean && count > 0 ? sum / count : sum);
        total[1] = (float)count;
    }
}

// Rows that TMA cannot read in place (their address or stride is not a multiple of 16 bytes).
template <typename T>
__global__ void __launch_bounds__(256)
xent_copy_kernel(const T* __restrict__ hidden, const long long ld, const int dim, T* __restrict__ packed, const long long ld_packed) {
    chain_begin();
    for (int c = threadIdx.x; c < dim; c += 256) packed[blockIdx.x * ld_packed + c] = hidden[blockIdx.x * ld + c];
}

// Self-check: the products' wait on a barrier that nothing arrives at.
__global__ void xent_timeout_kernel(int* status, const long long budget, int* gave_up) {
    __shared__ __align__(8) unsigned long long bar;
    __shared__ volatile int abort_flag;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(smem_u32(&bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        const bool done = mbar_wait(smem_u32(&bar), 0, &abort_flag, budget);
        if (abort_flag) *status = 1;
        *gave_up = !done && abort_flag;
    }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return (EncodeTiled)p;
    }();
    return fn;
}

// A row-major 16-bit matrix in boxes of 64 columns by box_rows, 128-byte swizzle; reads outside give zeros.
static int make_map(CUtensorMap* map, int dtype, uintptr_t base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiled fn = encode_tiled();
    if (!fn) { set_error("the driver does not offer cuTensorMapEncodeTiled"); return GM_ERR_UNSUPPORTED; }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {(cuuint32_t)kTileK, (cuuint32_t)box_rows};
    const cuuint32_t one[2] = {1, 1};
    const CUresult r = fn(map, dtype == GM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)base, dims, strides,
                          box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed with %d", (int)r); return GM_ERR_CUDA; }
    return GM_OK;
}

// Launches one product or two with as many CTA pairs as fit at once, at most one per turn.
template <int TN, typename First, typename Second = NoProduct>
static int launch_tiles(Device* d, const First& first, int64_t max_turns, int* launched = nullptr, const Second& second = Second()) {
    auto kernel = tile_gemm_kernel<TN, First, Second>;
    bool staging = First::Ops::kStaging;
    if constexpr (Second::kAny) staging = staging || Second::Ops::kStaging;
    const int smem = Ring<TN>::kSmem + (staging ? 8 * kStagingBytes : 0);
    static std::mutex mu;
    static int pairs_of[64] = {0};                   // per device ordinal
    int pairs;
    {
        std::lock_guard<std::mutex> lk(mu);
        int& known = pairs_of[d->ordinal & 63];
        if (known == 0) {
            GM_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)(d->sm_count / 2 * 2));
            cfg.blockDim = dim3(kGemmThreads);
            cfg.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr = {};
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int n = 0;
            GM_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
            if (n < 1) { set_error("no CTA pair of the matrix product fits the device"); return GM_ERR_UNSUPPORTED; }
            known = n;
        }
        pairs = known;
    }
    if (max_turns < pairs) pairs = (int)max_turns;
    if (launched) *launched = pairs;
    GM_CUDA_CHECK(launch_chained(kernel, dim3((unsigned)pairs * 2), dim3(kGemmThreads), smem, d->stream, first, second,
                                 reinterpret_cast<int*>(d->scalars + kXentStatusWord), d->barrier_budget_cycles));
    d->launches++;
    return GM_OK;
}

static int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }   // workspace parts, and rows up to a whole tile

constexpr int64_t kPieceTarget = 512LL << 20;        // bytes of S the recommended workspace holds
constexpr int kFewRows = 128;                        // rows up to which the vocabulary takes the tiles' long side
constexpr int kMostParts = 296;                      // shares of dX's tiles that may be waiting to be added up, 256 KB each

static int64_t split_parts(const gm_linear_xent_t* h) {
    const int64_t all = up256(h->tokens) / kTileM * ((h->dim + kTileN - 1) / kTileN) * 16;
    return all < kMostParts ? all : kMostParts;
}
// m-tiles of the logits' products walked together: as many rows of X as take 32 MB, a quarter of L2
static int logits_group(const gm_linear_xent_t* h) {
    const int64_t g = (32LL << 20) / (kTileM * 2 * h->dim);
    return (int)(g < 8 ? 8 : g > 64 ? 64 : g);
}

struct XentSpace {
    int64_t cap, ld_packed;                          // rows up to a whole tile, stride of the gathered hidden states
    int64_t scalars, rows, target, of_target, packed;  // both passes
    int64_t stats, partial;                          // forward
    int64_t parts, carried, ld_carried, ds, width;   // backward
    int64_t total;
};

static XentSpace common_space(const gm_linear_xent_t* h) {
    XentSpace s = {};
    s.cap = up256(h->tokens);
    s.ld_packed = (h->dim + 7) / 8 * 8;
    s.rows = 256;
    s.target = s.rows + up256(s.cap * 4);
    s.of_target = s.target + up256(s.cap * 4);
    s.packed = s.of_target + up256(s.cap * 4);
    s.total = s.packed + up256(s.cap * s.ld_packed * 2);
    return s;
}

static XentSpace forward_space(const gm_linear_xent_t* h) {
    XentSpace s = common_space(h);
    s.stats = s.total;
    // a few rows: eight pieces per tile of at least 16 entries, and no more tiles than rounds of half the SMs
    const int64_t few_tiles = (h->vocab + 15) / 16 < 1024 ? (h->vocab + 15) / 16 : 1024 + (h->vocab + 127) / 128;
    const int64_t stat_tiles = h->tokens <= kFewRows ? few_tiles * 8 : (h->vocab + kTileN / 2 - 1) / (kTileN / 2);
    s.partial = s.stats + up256(stat_tiles * s.cap * 8);
    s.total = s.partial + up256(s.cap * 4);
    return s;
}

// The widest piece of the vocabulary whose S fits `bytes`; width 0 when not even 256 entries do.
static XentSpace backward_space(const gm_linear_xent_t* h, int64_t bytes) {
    XentSpace s = common_space(h);
    const int64_t all = up256(h->vocab);
    s.parts = s.total;
    s.total = s.parts + split_parts(h) * kTileM * kTileN * 4;
    s.ld_carried = s.ld_packed;
    if (s.total + up256(s.cap * all * 2) <= bytes) {              // one piece: nothing is carried
        s.width = all;
        s.carried = s.ds = s.total;
    } else {
        s.carried = s.total;
        s.ds = s.carried + up256(s.cap * s.ld_carried * 4);
        const int64_t room = bytes - s.ds;
        s.width = room > 0 ? room / (s.cap * 2) / 256 * 256 : 0;
        if (s.width > all) s.width = all;
        // pieces of even size: the last one is not a sliver
        if (s.width > 0) {
            const int64_t pieces = (all + s.width - 1) / s.width;
            s.width = up256((all + pieces - 1) / pieces);
        }
    }
    s.total = s.ds + up256(s.cap * s.width * 2);
    return s;
}

static int64_t backward_bytes(const gm_linear_xent_t* h, bool smallest) {
    XentSpace s = common_space(h);
    const int64_t all = up256(h->vocab);
    s.total += split_parts(h) * kTileM * kTileN * 4;
    int64_t width = smallest ? 256 : kPieceTarget / (s.cap * 2) / 256 * 256;
    if (width < 256) width = 256;
    const int64_t whole = s.total + up256(s.cap * all * 2);       // one piece: nothing is carried
    if (width >= all) return whole;
    const int64_t pieces = (all + width - 1) / width;
    width = up256((all + pieces - 1) / pieces);
    const int64_t pieced = s.total + up256(s.cap * s.ld_packed * 4) + up256(s.cap * width * 2);
    return pieced < whole ? pieced : whole;
}

static int check_xent(const gm_linear_xent_t* h) {
    if (!h) { set_error("loss argument is nil"); return GM_ERR_BAD_ARG; }
    if (h->dtype != GM_F16 && h->dtype != GM_BF16) { set_error("element type %d is not Float16 or BFloat16", h->dtype); return GM_ERR_BAD_ARG; }
    GM_TRY(check_matrix(h->tokens, h->dim, h->ld_hidden, "hidden states"));
    GM_TRY(check_matrix(h->vocab, h->dim, h->ld_weight, "vocabulary table"));
    // One tile of dW is a sum over all rows with a target: 2^26 of them are 2^20 blocks of 64 and 0.3 to 0.4 s, which
    // the waits' default bound of 2^31 cycles (about 1.1 s) covers and 2^28 would not.
    if (h->tokens > (1LL << 26) || h->vocab > (1LL << 28) || h->dim > (1LL << 24)) { set_error("%lld tokens, %lld columns or %lld vocabulary entries are too many", (long long)h->tokens, (long long)h->dim, (long long)h->vocab); return GM_ERR_BAD_SIZE; }
    if (up256(h->tokens) / 256 * (up256(h->vocab) / 256) > 0x3fffffffLL) { set_error("%lld tokens by %lld vocabulary entries are too many", (long long)h->tokens, (long long)h->vocab); return GM_ERR_BAD_SIZE; }
    if (h->ld_weight % 8) { set_error("the table's row stride %lld is not a multiple of 8 elements", (long long)h->ld_weight); return GM_ERR_BAD_ARG; }
    return GM_OK;
}

struct XentCall {
    Device* d;
    const gm_linear_xent_t* h;
    uintptr_t ws;
    XentSpace s;
    XentScalars* sc() const { return (XentScalars*)(ws + s.scalars); }
    int* rows() const { return (int*)(ws + s.rows); }
    int* target() const { return (int*)(ws + s.target); }
    float* of_target() const { return (float*)(ws + s.of_target); }      // the targets' logits, or their entries of softmax - onehot
};

template <typename T>
static int index_and_gather(const XentCall& c, uintptr_t hidden, uintptr_t targets, uintptr_t weight, const float* lse_given, float* losses, float* lse,
                            T* dhidden) {
    const gm_linear_xent_t* h = c.h;
    const bool few = h->tokens <= kFewIndex;
    if (!few) {
        GM_CUDA_CHECK(launch_chained(xent_index_kernel, dim3(1), dim3(kIndexThreads), 0, c.d->stream, (const int*)targets, (int)h->tokens,
                                     (int)h->vocab, c.rows(), c.target(), c.sc()));
        c.d->launches++;
    }
    const bool vec = hidden % 16 == 0 && h->ld_hidden % 8 == 0;
    const bool vec_out = (uintptr_t)dhidden % 16 == 0 && h->ld_hidden % 8 == 0;
    GM_CUDA_CHECK(launch_chained(xent_gather_kernel<T>, dim3((unsigned)c.s.cap), dim3(kGatherThreads), 0, c.d->stream, (const T*)hidden, h->ld_hidden,
                                 (int)h->tokens, (int)h->dim, (int)h->vocab, (const int*)targets, c.rows(), c.target(), c.sc(), few,
                                 (T*)(c.ws + c.s.packed), c.s.ld_packed, (const T*)weight, h->ld_weight, c.of_target(), lse_given, losses, lse, dhidden, vec,
                                 vec_out));
    c.d->launches++;
    return GM_OK;
}

// A few rows: one product that reads W once, and the kernel that joins.
template <typename T, int TN>
static int forward_few(const XentCall& c, uintptr_t hidden, uintptr_t weight, uintptr_t targets, float* losses, float* lse, float* total) {
    const gm_linear_xent_t* h = c.h;
    const XentSpace& s = c.s;
    const bool in_place = hidden % 16 == 0 && h->ld_hidden % 8 == 0;
    const uintptr_t x = in_place ? hidden : c.ws + s.packed;
    // entries per CTA and tile: the rounds that 128 would take, evenly filled
    const int64_t ctas = c.d->sm_count / 2 * 2, rounds = (h->vocab + kHalf * ctas - 1) / (kHalf * ctas);
    const int height = (int)(((h->vocab + rounds * ctas - 1) / (rounds * ctas) + 7) / 8 * 8);
    const int64_t tiles = (h->vocab + 2 * height - 1) / (2 * height);
    CUtensorMap map_w, map_x;
    GM_TRY(make_map(&map_w, h->dtype, weight, h->vocab, h->dim, h->ld_weight, height));
    GM_TRY(make_map(&map_x, h->dtype, x, h->tokens, h->dim, in_place ? h->ld_hidden : s.ld_packed, TN / 2));
    if (!in_place) {
        GM_CUDA_CHECK(launch_chained(xent_copy_kernel<T>, dim3((unsigned)h->tokens), dim3(256), 0, c.d->stream, (const T*)hidden, h->ld_hidden, (int)h->dim,
                                     (T*)x, s.ld_packed));
        c.d->launches++;
    }
    float2* stats = (float2*)(c.ws + s.stats);
    auto product = [&](auto ops) { return launch_tiles<TN>(c.d, Product<decltype(ops), false, false>{map_w, map_x, ops}, tiles); };
    const int n = (int)h->tokens, cap = (int)s.cap, dim = (int)h->dim, vocab = (int)h->vocab;
    if (dim > kOneSum) GM_TRY(product(FewStatsOps<T, TN, true>{c.sc(), (const int*)targets, stats, n, cap, dim, vocab, height, 0, 0}));
    else GM_TRY(product(FewStatsOps<T, TN, false>{c.sc(), (const int*)targets, stats, n, cap, dim, vocab, height, 0, 0}));
    GM_CUDA_CHECK(launch_chained(xent_few_join_kernel<T>, dim3((unsigned)h->tokens), dim3(256), 0, c.d->stream, c.sc(), (const T*)hidden, h->ld_hidden,
                                 (const T*)weight, h->ld_weight, (const int*)targets, (int)h->dim, (int)h->vocab, in_place, stats, (int)s.cap, (int)tiles * 8, losses, lse,
                                 (float*)(c.ws + s.partial), total, h->mean, reinterpret_cast<const int*>(c.d->scalars + kXentStatusWord)));
    c.d->launches++;
    return GM_OK;
}

template <typename T>
static int run_forward(const XentCall& c, uintptr_t hidden, uintptr_t weight, uintptr_t targets, float* losses, float* lse, float* total) {
    const gm_linear_xent_t* h = c.h;
    const XentSpace& s = c.s;
    // 16 x 1,024 x 32,000 takes 20.3, 20.3 and 24.1 us with tiles for 32, 64 and 128 rows and 26.2 us by the way below, 64 rows
    // 20.8 and 25.1 us with tiles for 64 and 128 and 27.5 below, 128 rows 26.0 us and 27.1 below; larger tables: 16 x 4,096 x
    // 131,072 with tiles for 32 and 64 rows 175.6 and 179.6 us
    if (h->tokens <= 32) return forward_few<T, 32>(c, hidden, weight, targets, losses, lse, total);
    if (h->tokens <= 64) return forward_few<T, 64>(c, hidden, weight, targets, losses, lse, total);
    if (h->tokens <= kFewRows) return forward_few<T, kFewRows>(c, hidden, weight, targets, losses, lse, total);
    CUtensorMap map_w, map_x;
    GM_TRY(make_map(&map_w, h->dtype, weight, h->vocab, h->dim, h->ld_weight, kHalf));
    GM_TRY(make_map(&map_x, h->dtype, c.ws + s.packed, s.cap, h->dim, s.ld_packed, kHalf));
    GM_TRY(index_and_gather<T>(c, hidden, targets, weight, nullptr, losses, lse, (T*)nullptr));
    float2* stats = (float2*)(c.ws + s.stats);
    const int64_t n_tiles = (h->vocab + kTileN - 1) / kTileN;
    const int tiles = (int)((h->vocab + kTileN / 2 - 1) / (kTileN / 2));
    auto product = [&](auto ops) { return launch_tiles<kTileN>(c.d, Product<decltype(ops), false, false>{map_x, map_w, ops}, s.cap / kTileM * n_tiles); };
    const int cap = (int)s.cap, dim = (int)h->dim, vocab = (int)h->vocab;
    if (dim > kOneSum) GM_TRY(product(StatsOps<T, true>{c.sc(), c.target(), stats, cap, dim, vocab, logits_group(h), 0, 0}));
    else GM_TRY(product(StatsOps<T, false>{c.sc(), c.target(), stats, cap, dim, vocab, logits_group(h), 0, 0}));
    // a CTA per row up to a few rows per SM, 8 rows per CTA beyond
    auto join = h->tokens <= 1024 ? xent_join_kernel<1> : xent_join_kernel<8>;
    const int64_t ctas = h->tokens <= 1024 ? h->tokens : s.cap / 8;
    GM_CUDA_CHECK(launch_chained(join, dim3((unsigned)ctas), dim3(256), 0, c.d->stream, c.sc(), stats, (int)s.cap, tiles, c.of_target(), c.rows(), losses, lse,
                                 (float*)(c.ws + s.partial), total, h->mean, reinterpret_cast<const int*>(c.d->scalars + kXentStatusWord)));
    c.d->launches++;
    return GM_OK;
}

template <typename T, bool MAP>
static int backward_pieces(const XentCall& c, uintptr_t hidden, uintptr_t weight, uintptr_t targets, const float* lse, const float* scale_device,
                           float grad_scale, uintptr_t dhidden, uintptr_t dweight, bool accumulate) {
    const gm_linear_xent_t* h = c.h;
    const XentSpace& s = c.s;
    const uintptr_t packed = c.ws + s.packed, ds = c.ws + s.ds;
    CUtensorMap x_k, x_mn, w_k, w_mn, ds_k, ds_mn;       // K-major for the logits and dX's S, MN-major for the rest
    CUtensorMap ds_out, dw_out = {};                     // what the epilogues store to
    GM_TRY(make_map(&x_k, h->dtype, packed, s.cap, h->dim, s.ld_packed, kHalf));
    GM_TRY(make_map(&x_mn, h->dtype, packed, s.cap, h->dim, s.ld_packed, kTileK));
    GM_TRY(make_map(&w_k, h->dtype, weight, h->vocab, h->dim, h->ld_weight, kHalf));
    GM_TRY(make_map(&w_mn, h->dtype, weight, h->vocab, h->dim, h->ld_weight, kTileK));
    GM_TRY(make_map(&ds_k, h->dtype, ds, s.cap, s.width, s.width, kHalf));
    GM_TRY(make_map(&ds_mn, h->dtype, ds, s.cap, s.width, s.width, kTileK));
    GM_TRY(make_map(&ds_out, h->dtype, ds, s.cap, s.width, s.width, 32));
    if (MAP) GM_TRY(make_map(&dw_out, h->dtype, dweight, h->vocab, h->dim, h->ld_weight, 32));
    GM_TRY(index_and_gather<T>(c, hidden, targets, weight, lse, nullptr, nullptr, (T*)dhidden));
    const GradScale scale{reinterpret_cast<const int*>(c.d->scalars + kXentStatusWord), scale_device, grad_scale, h->mean, 1.0f / Half16<T>::kUp};
    const int dim = (int)h->dim, vocab = (int)h->vocab;
    const int64_t m_tiles = s.cap / kTileM, d_tiles = (h->dim + kTileN - 1) / kTileN;
    using Hidden = Product<HiddenGradOps<T>, false, true>;
    using Weight = Product<WeightGradOps<T, MAP>, true, true>;
    for (int64_t v = 0; v < vocab; v += s.width) {
        const int v0 = (int)v, v1 = (int)(v + s.width < vocab ? v + s.width : vocab);
        const int64_t v_tiles = (v1 - v0 + kTileN - 1) / kTileN;
        const SoftmaxGradOps<T> grad{c.sc(), c.target(), c.rows(), lse, c.of_target(), ds_out, dim, v0, v1, logits_group(h), 0, v0};
        GM_TRY((launch_tiles<kTileN>(c.d, Product<SoftmaxGradOps<T>, false, false>{x_k, w_k, grad}, m_tiles * v_tiles)));
        const HiddenPlan shape{dim, v0, v1, (int)split_parts(h)};
        const HiddenOut<T> out{(float*)(c.ws + s.carried), s.ld_carried, (T*)dhidden, h->ld_hidden, scale, v0 == 0, v1 == vocab,
                               dhidden % 16 == 0 && h->ld_hidden % 8 == 0};
        float* parts = (float*)(c.ws + s.parts);
        const Hidden dx{ds_k, w_mn, HiddenGradOps<T>{c.sc(), c.rows(), parts, shape, out, 0, v0}};
        const Weight dw{ds_mn, x_mn, WeightGradOps<T, MAP>{c.sc(), dw_out, (T*)dweight, h->ld_weight, scale, dim, v0, v1, 0, 0, accumulate, dweight % 16 == 0}};
        const int64_t x_turns = m_tiles * d_tiles * 16, w_turns = v_tiles * d_tiles;
        int pairs = 0;
        // One launch of both gradients saves a start and an end and fills dX's last round: 39 -> 35 us
        // at 256 x 512 x 10,007, 132 -> 127 us at 6,525 x 1,808 x 1,314.  In many rounds with dX in more than
        // two, its longer turns on a fixed schedule lose more: 4.07 -> 4.15 ms at 8,862 x 1,384 x 55,838.
        const int64_t per_round = c.d->sm_count / 2;
        const bool both = dhidden && dweight && ((m_tiles + v_tiles) * d_tiles <= 16 * per_round || m_tiles * d_tiles <= 2 * per_round);
        if (both) GM_TRY((launch_tiles<kTileN>(c.d, dx, x_turns + w_turns, &pairs, dw)));
        else if (dhidden) GM_TRY((launch_tiles<kTileN>(c.d, dx, x_turns, &pairs)));
        if (dhidden) {
            // how many tiles are split follows from the rows with a target, which only the device knows
            GM_CUDA_CHECK(launch_chained(xent_hidden_join_kernel<T>, dim3((unsigned)c.d->sm_count * 4), dim3(256), 0, c.d->stream, c.sc(), c.rows(), parts, shape,
                                         out, pairs));
            c.d->launches++;
        }
        if (dweight && !both) GM_TRY((launch_tiles<kTileN>(c.d, dw, w_turns)));
    }
    return GM_OK;
}

template <typename T>
static int run_backward(const XentCall& c, uintptr_t hidden, uintptr_t weight, uintptr_t targets, const float* lse, const float* scale_device,
                        float grad_scale, uintptr_t dhidden, uintptr_t dweight, bool accumulate) {
    const bool map = dweight && dweight % 16 == 0 && c.h->dim % 8 == 0 && !accumulate;
    return (map ? backward_pieces<T, true> : backward_pieces<T, false>)(c, hidden, weight, targets, lse, scale_device, grad_scale, dhidden, dweight, accumulate);
}

}  // namespace gm

using namespace gm;

extern "C" {

int64_t gm_linear_xent_workspace_bytes(const gm_linear_xent_t* h, int pass) {
    if (check_xent(h) != GM_OK) return -1;
    if (pass < 0 || pass > 2) { set_error("pass %d is not 0, 1 or 2", pass); return -1; }
    if (pass == 0) return forward_space(h).total;
    if (pass == 2) return backward_bytes(h, true);
    const int64_t f = forward_space(h).total, b = backward_bytes(h, false);
    return f > b ? f : b;
}

int gm_linear_xent_forward_async(uintptr_t device_ptr, const gm_linear_xent_t* h, uintptr_t hidden, uintptr_t weight, uintptr_t targets,
                                 uintptr_t losses, uintptr_t lse, uintptr_t total, uintptr_t workspace, int64_t workspace_bytes) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    GM_TRY(check_xent(h));
    GM_TRY(check_buffer(d, hidden, matrix_bytes(h->tokens, h->dim, h->ld_hidden, 2), 2, "hidden states"));
    GM_TRY(check_buffer(d, weight, matrix_bytes(h->vocab, h->dim, h->ld_weight, 2), 16, "vocabulary table"));
    GM_TRY(check_buffer(d, targets, h->tokens * 4, 4, "targets"));
    GM_TRY(check_buffer(d, losses, h->tokens * 4, 4, "losses"));
    GM_TRY(check_buffer(d, lse, h->tokens * 4, 4, "log-sum-exp"));
    GM_TRY(check_buffer(d, total, 8, 4, "total"));
    const XentCall c{d, h, workspace, forward_space(h)};
    if (workspace_bytes < c.s.total) { set_error("workspace of %lld bytes, the call needs %lld", (long long)workspace_bytes, (long long)c.s.total); return GM_ERR_BAD_SIZE; }
    GM_TRY(check_buffer(d, workspace, c.s.total, 256, "workspace"));
    DeviceGuard g(d);
    if (h->dtype == GM_F16) return run_forward<__half>(c, hidden, weight, targets, (float*)losses, (float*)lse, (float*)total);
    return run_forward<__nv_bfloat16>(c, hidden, weight, targets, (float*)losses, (float*)lse, (float*)total);
}

int gm_linear_xent_backward_async(uintptr_t device_ptr, const gm_linear_xent_t* h, uintptr_t hidden, uintptr_t weight, uintptr_t targets,
                                  uintptr_t lse, uintptr_t scale_device, float grad_scale, uintptr_t dhidden, uintptr_t dweight,
                                  int accumulate, uintptr_t workspace, int64_t workspace_bytes) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    GM_TRY(check_xent(h));
    GM_TRY(check_buffer(d, hidden, matrix_bytes(h->tokens, h->dim, h->ld_hidden, 2), 2, "hidden states"));
    GM_TRY(check_buffer(d, weight, matrix_bytes(h->vocab, h->dim, h->ld_weight, 2), 16, "vocabulary table"));
    GM_TRY(check_buffer(d, targets, h->tokens * 4, 4, "targets"));
    GM_TRY(check_buffer(d, lse, h->tokens * 4, 4, "log-sum-exp"));
    if (scale_device) GM_TRY(check_buffer(d, scale_device, 4, 4, "loss scale"));
    if (!dhidden && !dweight) { set_error("neither gradient is asked for"); return GM_ERR_NIL_BUFFER; }
    if (dhidden) GM_TRY(check_buffer(d, dhidden, matrix_bytes(h->tokens, h->dim, h->ld_hidden, 2), 2, "hidden states' gradient"));
    if (dweight) GM_TRY(check_buffer(d, dweight, matrix_bytes(h->vocab, h->dim, h->ld_weight, 2), 2, "table's gradient"));
    const int64_t need = backward_bytes(h, true);
    if (workspace_bytes < need) { set_error("workspace of %lld bytes, the call needs %lld", (long long)workspace_bytes, (long long)need); return GM_ERR_BAD_SIZE; }
    const XentCall c{d, h, workspace, backward_space(h, workspace_bytes)};
    GM_TRY(check_buffer(d, workspace, c.s.total, 256, "workspace"));
    DeviceGuard g(d);
    if (h->dtype == GM_F16)
        return run_backward<__half>(c, hidden, weight, targets, (const float*)lse, (const float*)scale_device, grad_scale, dhidden, dweight, accumulate != 0);
    return run_backward<__nv_bfloat16>(c, hidden, weight, targets, (const float*)lse, (const float*)scale_device, grad_scale, dhidden, dweight, accumulate != 0);
}

int gm_selftest_xent_timeout(uintptr_t device_ptr, long long budget_cycles, int* gave_up) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    if (!gave_up || budget_cycles <= 0) { set_error("bad self-check arguments"); return GM_ERR_BAD_ARG; }
    DeviceGuard g(d);
    int* words = reinterpret_cast<int*>(d->scalars + kXentStatusWord);       // the status, and a word for the answer
    xent_timeout_kernel<<<1, 32, 0, d->stream>>>(words, budget_cycles, words + 1);
    d->launches++;
    GM_CUDA_CHECK(cudaGetLastError());
    GM_CUDA_CHECK(cudaStreamSynchronize(d->stream));
    GM_CUDA_CHECK(cudaMemcpy(gave_up, words + 1, sizeof(int), cudaMemcpyDeviceToHost));
    return GM_OK;
}

int gm_linear_xent_status(uintptr_t device_ptr) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    DeviceGuard g(d);
    int status = 0;
    GM_CUDA_CHECK(cudaStreamSynchronize(d->stream));
    GM_CUDA_CHECK(cudaMemcpy(&status, d->scalars + kXentStatusWord, sizeof(int), cudaMemcpyDeviceToHost));
    if (!status) return GM_OK;
    GM_CUDA_CHECK(cudaMemset(d->scalars + kXentStatusWord, 0, sizeof(int)));
    set_error("a wait of the vocabulary loss's matrix products ran out; the outputs of that call are not complete");
    return GM_ERR_TIMEOUT;
}

}  // extern "C"
