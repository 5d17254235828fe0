// gm_embedding.cu -- token embedding with scaling and dropout, and its gradient.
//
//   forward   out[t] = drop(scale * table[token_t])      one multiplication, by scale times dropout's factor
//   backward  dtable[v] (+)= scale * sum over t with token_t = v, ascending, of drop(dout[t])
//
// Both are bound by HBM: the forward pass reads and writes one row per token; the backward
// pass reads one row per token and writes every row of the table (or the touched ones).
// The backward sum runs over tokens sorted by {token, position}, which makes it a plain
// sequential sum per row with no float atomics.  The sort is of 64-bit words {token,
// position}: all different, so any correct sort gives the same order.
#include "gm_lm.cuh"

namespace gm {

constexpr int kEmbThreads = 256;
constexpr int kSortTile = 1024;          // words one CTA sorts in registers and shared memory
constexpr int kMergeWays = 8;            // sorted runs that one merge pass joins

// ---------------------------------------------------------------- forward
// A CTA is tx lanes over groups of eight columns times ty tokens; each thread takes ROWS
// tokens and issues all its loads first.  VEC: rows begin on 16-byte boundaries; the last
// dim % 8 columns go element by element.  WHOLE: dim is a multiple of eight, so a group is a block
// of dropout's generator.
template <typename T, bool VEC, bool WHOLE, int ROWS>
__global__ void __launch_bounds__(kEmbThreads, 4)
embedding_forward_kernel(const T* __restrict__ table, const int* __restrict__ tokens, T* __restrict__ out, const int n, const int dim,
                         const int vocab, const int ld_table, const int ld_out, const float scale, const __grid_constant__ Drop d) {
    chain_begin();
    const DropOffset o = drop_begin(d);
    const float up = __fmul_rn(scale, d.up);
    const int groups = (int)(((unsigned)dim + 7u) >> 3);
    const long long t0 = ((long long)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    int tok[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        tok[r] = t0 + r < n ? __ldg(tokens + t0 + r) : -1;
        if (tok[r] >= vocab) tok[r] = -1;
    }
    const int live = n - t0 < ROWS ? (int)(n - t0) : ROWS;           // tokens of this thread (may be none)
    for (int g = blockIdx.y * blockDim.x + threadIdx.x; g < groups; g += gridDim.y * blockDim.x) {
        const int c = g << 3;
        if (WHOLE || c + 8 <= dim) {
            Eight<T, VEC> raw[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (tok[r] >= 0) raw[r].template load<true>(table + (long long)tok[r] * ld_table + c);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (r >= live) break;
                float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (tok[r] >= 0) {
                    widen8<T>(raw[r].r, x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(x[k], up);
                    drop8<WHOLE>(d, o, (unsigned long long)((t0 + r) * dim + c), x);
                }
                Eight<T, VEC>::store(out + (t0 + r) * ld_out + c, x);
            }
        } else {
            for (int r = 0; r < live; ++r) {
                const unsigned keep = tok[r] >= 0 ? drop_mask8(d, o, (unsigned long long)((t0 + r) * dim + c)) : 0u;
                for (int k = 0; k < 8 && k < dim - c; ++k) {
                    float x = 0.0f;
                    if ((keep >> k) & 1u) x = __fmul_rn(to_f32<T>(table[(long long)tok[r] * ld_table + c + k]), up);
                    out[(t0 + r) * ld_out + c + k] = from_f32<T>(x);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- sort
// Tokens without a gradient (out of range, padding) become `vocab` and end up behind the rest.
__device__ __forceinline__ unsigned long long sort_word(const int* tokens, long long i, long long vocab, long long padding) {
    const long long t = tokens[i];
    const unsigned key = t < 0 || t >= vocab || t == padding ? (unsigned)vocab : (unsigned)t;
    return ((unsigned long long)key << 32) | (unsigned)i;
}

// Bitonic sort of 1,024 words, one per thread: strides below a warp by shuffle, the others
// through shared memory.  The same launch clears `used`, one byte per row of the table (a
// multiple of 16 of them), and the number of rows split over chunks; the launch after it, or this one where a tile is all there is, marks
// the rows that tokens point at.
__global__ void __launch_bounds__(kSortTile)
token_sort_tile_kernel(const int* __restrict__ tokens, const long long n, const long long vocab, const long long padding,
                       unsigned long long* __restrict__ out, unsigned char* used, int* split) {
    __shared__ unsigned long long buf[kSortTile];
    const int tid = threadIdx.x;
    const long long i = (long long)blockIdx.x * kSortTile + tid;
    chain_begin();
    unsigned long long key = i < n ? sort_word(tokens, i, vocab, padding) : ~0ull;
    if (i == 0) *split = 0;
    if (used)
        for (long long c = i * 16; c < vocab; c += (long long)gridDim.x * kSortTile * 16) *reinterpret_cast<uint4*>(used + c) = make_uint4(0u, 0u, 0u, 0u);
    for (int size = 2; size <= kSortTile; size <<= 1) {
        const bool up = (tid & size) == 0;
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            unsigned long long other;
            if (stride >= 32) {
                buf[tid] = key;
                __syncthreads();
                other = buf[tid ^ stride];
                __syncthreads();
            } else {
                other = __shfl_xor_sync(0xffffffffu, key, stride);
            }
            const bool low = (tid & stride) == 0;
            const bool take_min = low == up;
            key = take_min ? (other < key ? other : key) : (other > key ? other : key);
        }
    }
    if (i < n) out[i] = key;
    if (used && gridDim.x == 1) {
        __syncthreads();
        if (i < n && (key >> 32) < (unsigned long long)vocab) used[key >> 32] = 1;
    }
}

// The token of a sorted word.
__device__ __forceinline__ unsigned token_at(const unsigned long long* __restrict__ words, long long i) {
    return __ldg(reinterpret_cast<const unsigned*>(words + i) + 1);
}

// First of the words [lo, hi) whose token is not below `key`.
__device__ __forceinline__ long long first_at(const unsigned long long* __restrict__ words, long long lo, long long hi, unsigned key) {
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (token_at(words, mid) < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Joins kMergeWays sorted runs of `run` words (a power of two): a word's place is the number of
// words in front of it in every run of its group, found by bisection, so one pass has no serial
// part.  Runs hold ascending positions, so an equal token of an earlier run comes first and one
// of a later run behind: comparing tokens is enough.  The bisections, chains of dependent loads,
// go in step.
__global__ void __launch_bounds__(128)
token_merge_kernel(const unsigned long long* __restrict__ in, unsigned long long* __restrict__ out, const long long n, const int run,
                   unsigned char* used, const unsigned vocab) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    chain_begin();
    if (i >= n) return;
    const unsigned long long word = __ldg(in + i);
    const unsigned token = (unsigned)(word >> 32);
    if (used && token < vocab) used[token] = 1;
    const long long base = i / ((long long)run * kMergeWays) * ((long long)run * kMergeWays);
    const int mine = (int)((i - base) / run);
    int below[kMergeWays], len[kMergeWays];
#pragma unroll
    for (int j = 0; j < kMergeWays; ++j) {
        const long long left = n - (base + (long long)j * run);
        below[j] = 0;
        len[j] = left <= 0 ? 0 : left < run ? (int)left : run;
    }
    for (int step = run; step > 0; step >>= 1) {
#pragma unroll
        for (int j = 0; j < kMergeWays; ++j)
            if (below[j] + step <= len[j] && token_at(in, base + (long long)j * run + below[j] + step - 1) < token + (j < mine ? 1u : 0u)) below[j] += step;
    }
    long long place = base + (i - base - (long long)mine * run);
#pragma unroll
    for (int j = 0; j < kMergeWays; ++j) place += j == mine ? 0 : below[j];
    out[place] = word;
}

// ---------------------------------------------------------------- backward sums
// The sorted words are cut into chunks of `piece` (at most kPieceMost).  A CTA is up to 128 lanes
// over groups of eight columns times as many chunks as make 128 threads; every thread walks one chunk
// for its columns, eight loads in flight whatever rows they belong to, and writes a row's sum when the
// row's last word has been added.  So all threads have the same work, and a token that fills half the
// batch is spread over the GPU.  A row whose words lie in several chunks leaves a
// partial sum per chunk (slot 2j: chunk j's part of a row that began before it; slot 2j + 1: that
// of a row that begins in it and goes on) and its first chunk in a list, and embedding_join_kernel
// adds them up.  The list's order is chance, the sums are not.
//
// The same launch holds, without ADD, the CTAs that zero the rows no token points at: they have no
// loads to wait for and fill the time of those that do, alternating with them in proportion.
constexpr int kSumThreads = 128;
constexpr int kSumDeep = 8;
constexpr int kPieceMost = 32;
constexpr int kZeroRowsMost = 128;

// What becomes of a finished row: times `up`, added to what is there (ADD) or not.
template <typename G, bool VEC, bool WHOLE, bool ADD>
__device__ __forceinline__ void put_row(G* to, float (&x)[8], const float up, const int cols) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(x[k], up);
    if (WHOLE || cols >= 8) {
        if (ADD) {
            float old[8];
            Eight<G, VEC> there;
            there.template load<false>(to);
            widen8<G>(there.r, old);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = __fadd_rn(old[k], x[k]);
        }
        Eight<G, VEC>::store(to, x);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < cols) to[k] = from_f32<G>(ADD ? __fadd_rn(to_f32<G>(to[k]), x[k]) : x[k]);
    }
}

template <typename T, typename G, bool VEC, bool WHOLE, bool ADD>
__global__ void __launch_bounds__(kSumThreads)
embedding_sum_kernel(const T* __restrict__ dout, const unsigned long long* __restrict__ words, const unsigned char* __restrict__ used,
                     float* __restrict__ pieces, int* split, G* dtable, const int n, const int dim, const int vocab, const int ld_table,
                     const int ld_out, const float scale, const int piece, const int col_ctas, const int sum_ctas, const int zero_rows, const __grid_constant__ Drop d) {
    __shared__ unsigned tok[kSumThreads / 8][kPieceMost], pos[kSumThreads / 8][kPieceMost];
    static_assert(sizeof(tok) >= kZeroRowsMost * sizeof(unsigned), "the zeroing CTAs keep their marks there");
    const int lanes = blockDim.x, tid = threadIdx.y * lanes + threadIdx.x;
    chain_begin();
    const int groups = (int)(((unsigned)dim + 7u) >> 3);
    const long long before = ADD ? blockIdx.x : (long long)blockIdx.x * sum_ctas / gridDim.x;       // summing CTAs in front of this one
    if (!ADD && ((long long)blockIdx.x + 1) * sum_ctas / gridDim.x == before) {
        const long long v0 = (blockIdx.x - before) * zero_rows;
        unsigned* const skip = &tok[0][0];
        if (tid < zero_rows) skip[tid] = v0 + tid < vocab ? used[v0 + tid] : 1u;
        __syncthreads();
        // lanes over the 16-byte words of a row, and several rows at a time where a row is narrow; a row
        // that begins or ends inside a word has those elements zeroed by themselves
        constexpr int PER = 16 / sizeof(G);
        const int words_of_row = (dim + PER - 1) / PER;
        const int wide = words_of_row >= kSumThreads ? kSumThreads : words_of_row > 32 ? 64 : words_of_row > 16 ? 32 : words_of_row > 8 ? 16 : 8;
        const int lane = tid & (wide - 1), step = kSumThreads / wide;
        G* row = dtable + (v0 + tid / wide) * ld_table;
        const long long next = (long long)step * ld_table;
        if (VEC && dim % PER == 0) {
            for (int r = tid / wide; r < zero_rows; r += step, row += next)
                if (!skip[r])
                    for (int w = lane; w < words_of_row; w += wide) __stcs(reinterpret_cast<uint4*>(row) + w, make_uint4(0u, 0u, 0u, 0u));
            return;
        }
        for (int r = tid / wide; r < zero_rows; r += step, row += next) {
            if (skip[r]) continue;
            int head = (int)((16u - (unsigned)(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / (int)sizeof(G);
            if (head > dim) head = dim;
            const int body = (dim - head) / PER, rest = head + body * PER;
            for (int w = lane; w < body; w += wide) __stcs(reinterpret_cast<uint4*>(row + head) + w, make_uint4(0u, 0u, 0u, 0u));
            if (lane < head) row[lane] = from_f32<G>(0.0f);
            if (lane < dim - rest) row[rest + lane] = from_f32<G>(0.0f);
        }
        return;
    }
    const long long row_of_ctas = before / col_ctas, chunk = row_of_ctas * blockDim.y + threadIdx.y, begin = chunk * piece;
    const int most = begin >= n ? 0 : n - begin < piece ? (int)(n - begin) : piece;
    unsigned *const token = tok[threadIdx.y], *const where = pos[threadIdx.y];
    for (int i = threadIdx.x; i < most; i += lanes) {
        const unsigned long long w = __ldg(words + begin + i);
        token[i] = (unsigned)(w >> 32);
        where[i] = (unsigned)w;
    }
    __syncthreads();
    int len = most;                                                   // words without a gradient are behind all others
    while (len > 0 && token[len - 1] >= (unsigned)vocab) --len;
    if (len == 0) return;
    const bool from_before = begin > 0 && token_at(words, begin - 1) == token[0];
    const bool goes_on = begin + len < n && token_at(words, begin + len) == token[len - 1];
    if (threadIdx.x == 0 && goes_on && before == row_of_ctas * col_ctas && !(from_before && token[0] == token[len - 1])) split[1 + atomicAdd(split, 1)] = (int)chunk;
    const DropOffset o = drop_begin(d);
    const float up = __fmul_rn(scale, d.up);
    const int g = (int)(before - row_of_ctas * col_ctas) * lanes + threadIdx.x, c = g << 3;
    if (g >= groups) return;
    const bool full = WHOLE || c + 8 <= dim;
    bool head = from_before;                                          // the current row began in an earlier chunk
    float acc[8] = {};
    constexpr int kDeep = VEC && sizeof(T) == 2 ? kSumDeep : kSumDeep / 2;
    for (int base = 0; base < len; base += kDeep) {
        Eight<T, VEC> raw[kDeep];
        if (full) {
#pragma unroll
            for (int j = 0; j < kDeep; ++j)
                if (base + j < len) raw[j].template load<false>(dout + (long long)where[base + j] * ld_out + c);
        }
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
            if (base + j >= len) break;
            float x[8] = {};
            const long long p = where[base + j];
            if (full) {
                widen8<T>(raw[j].r, x);
            } else {
                for (int k = 0; k < 8 && k < dim - c; ++k) x[k] = to_f32<T>(dout[p * ld_out + c + k]);
            }
            drop8<WHOLE>(d, o, (unsigned long long)(p * dim + c), x);
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] = __fadd_rn(acc[k], x[k]);
            const bool last = base + j + 1 == len;
            if (last || token[base + j + 1] != token[base + j]) {
                if (head || (last && goes_on)) {
                    float4* to = reinterpret_cast<float4*>(pieces + ((2 * chunk + (head ? 0 : 1)) * groups + g) * 8);
                    to[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    to[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                } else {
                    put_row<G, VEC, WHOLE, ADD>(dtable + (long long)token[base + j] * ld_table + c, acc, up, dim - c);
                }
                head = false;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
            }
        }
    }
}

// Adds up the partial sums of the listed rows: a CTA is up to 64 lanes over column groups times as
// many ways as make 256 threads; each way takes a contiguous share of a row's chunks, and the ways are
// joined in order.
constexpr int kJoinThreads = 256, kJoinLanesMost = 64;
template <typename G, bool VEC, bool WHOLE, bool ADD>
__global__ void __launch_bounds__(kJoinThreads)
embedding_join_kernel(const unsigned long long* __restrict__ words, const float* __restrict__ pieces, const int* __restrict__ split, G* dtable,
                      const int n, const int dim, const int ld_table, const float scale, const int piece, const __grid_constant__ Drop d) {
    __shared__ float4 part[2][kJoinThreads];
    const int x = threadIdx.x, y = threadIdx.y, lanes = blockDim.x, ways = blockDim.y, tid = y * lanes + x;
    chain_begin();
    const int groups = (int)(((unsigned)dim + 7u) >> 3), col_blocks = (groups + lanes - 1) / lanes;
    const float up = __fmul_rn(scale, d.up);
    const long long items = (long long)split[0] * col_blocks;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const long long chunk = split[1 + item / col_blocks];
        const int g = (int)(item % col_blocks) * lanes + x;
        const unsigned key = token_at(words, (chunk + 1) * piece);
        // the row's last chunk: chunks whose first word is the row's, 32 looked at together
        long long last = chunk;
        for (;;) {
            const long long at = (last + 1 + (tid & 31)) * piece;
            const unsigned hit = __ballot_sync(0xffffffffu, at < n && token_at(words, at) == key);
            last += hit == 0xffffffffu ? 32 : __ffs((int)~hit) - 1;
            if (hit != 0xffffffffu) break;
        }
        const long long share = (last - chunk + ways) / ways;         // chunks [chunk, last] over the ways
        float acc[8] = {};
        if (g < groups) {
            const long long from = chunk + y * share, to = from + share - 1 < last ? from + share - 1 : last;
#pragma unroll 4
            for (long long j = from; j <= to; ++j) {
                const float4* p = reinterpret_cast<const float4*>(pieces + ((2 * j + (j == chunk ? 1 : 0)) * groups + g) * 8);
                const float4 u = p[0], v = p[1];
                acc[0] = __fadd_rn(acc[0], u.x); acc[1] = __fadd_rn(acc[1], u.y);
                acc[2] = __fadd_rn(acc[2], u.z); acc[3] = __fadd_rn(acc[3], u.w);
                acc[4] = __fadd_rn(acc[4], v.x); acc[5] = __fadd_rn(acc[5], v.y);
                acc[6] = __fadd_rn(acc[6], v.z); acc[7] = __fadd_rn(acc[7], v.w);
            }
        }
        part[0][tid] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        part[1][tid] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        __syncthreads();
        if (y == 0 && g < groups) {
            for (int w = 1; w < ways; ++w) {
                const float4 u = part[0][w * lanes + x], v = part[1][w * lanes + x];
                acc[0] = __fadd_rn(acc[0], u.x); acc[1] = __fadd_rn(acc[1], u.y);
                acc[2] = __fadd_rn(acc[2], u.z); acc[3] = __fadd_rn(acc[3], u.w);
                acc[4] = __fadd_rn(acc[4], v.x); acc[5] = __fadd_rn(acc[5], v.y);
                acc[6] = __fadd_rn(acc[6], v.z); acc[7] = __fadd_rn(acc[7], v.w);
            }
            put_row<G, VEC, WHOLE, ADD>(dtable + (long long)key * ld_table + (g << 3), acc, up, dim - (g << 3));
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
// Sorted words per chunk: 32 in a large call, 16 or 8 where that would leave an SM fewer than 512
// threads: the walk over a chunk is serial, and a small call is as long as one walk (4,095 x 1,000: 46
// us with 8, 50 us with 16; 65,536 x 4,096: 0.32 ms with 32, 0.55 ms with 16, whose partial sums are
// twice as many).  148 is the B200's number of SMs, written in because the workspace's size, which follows
// from the chunks, is told without a device.
static int piece_of(const gm_embedding_t* e) {
    const int64_t walks = e->tokens * ((e->dim + 7) / 8);              // one word each
    return walks >= 32LL * 148 * 512 ? 32 : walks >= 16LL * 148 * 512 ? 16 : 8;
}

// Lanes over column groups: a power of two that covers them, between `least` and `most`.
static int lanes_of(int64_t groups, int least, int most) {
    int x = least;
    while (x < most && x < groups) x <<= 1;
    return x;
}

struct EmbSpace { int64_t words0, words1, used, split, pieces, total; };

static int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

static EmbSpace embedding_space(const gm_embedding_t* e) {
    EmbSpace s;
    s.words0 = 0;
    s.words1 = s.words0 + up256(e->tokens * 8);
    s.used = s.words1 + up256(e->tokens * 8);
    s.split = s.used + up256(e->vocab);
    s.pieces = s.split + up256(((e->tokens + piece_of(e) - 1) / piece_of(e) + 1) * 4);
    s.total = s.pieces + up256(2 * ((e->tokens + piece_of(e) - 1) / piece_of(e)) * ((e->dim + 7) / 8 * 8) * 4);
    return s;
}

static int check_embedding(const gm_embedding_t* e) {
    if (!e) { set_error("embedding argument is nil"); return GM_ERR_BAD_ARG; }
    if (!dtype_bytes(e->dtype)) { set_error("element type %d is not Float32, Float16 or BFloat16", e->dtype); return GM_ERR_BAD_ARG; }
    if (e->vocab > 0x7ffffffeLL) { set_error("vocabulary of %lld rows is too large", (long long)e->vocab); return GM_ERR_BAD_SIZE; }
    GM_TRY(check_matrix(e->vocab, e->dim, e->ld_table, "embedding table"));
    GM_TRY(check_matrix(e->tokens, e->dim, e->ld_out, "embedding output"));
    return GM_OK;
}

template <typename T>
static int launch_embedding_forward(Device* d, const gm_embedding_t* e, uintptr_t table, uintptr_t tokens, uintptr_t out, const Drop& drop) {
    const int lanes = lanes_of((e->dim + 7) / 8, 8, kEmbThreads);
    const dim3 block((unsigned)lanes, (unsigned)(kEmbThreads / lanes));
    // the grid's second axis spreads a wide row over CTAs
    const int64_t y = ((e->dim + 7) / 8 + block.x - 1) / block.x;
    const unsigned gy = (unsigned)(y < 65535 ? y : 65535);
    const bool vec = table % 16 == 0 && out % 16 == 0 && e->ld_table * (int)sizeof(T) % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0;
    // four tokens per thread keep more loads in flight; a call too small for that takes one
    const bool many = e->tokens * gy >= (int64_t)d->sm_count * 8 * block.y;
#define GM_FORWARD(VEC, WHOLE, ROWS)                                                                                                       \
    GM_CUDA_CHECK(launch_chained(embedding_forward_kernel<T, VEC, WHOLE, ROWS>,                                                             \
                                 dim3((unsigned)((e->tokens + block.y * ROWS - 1) / (block.y * ROWS)), gy), block, 0, d->stream,             \
                                 (const T*)table, (const int*)tokens, (T*)out, (int)e->tokens, (int)e->dim, (int)e->vocab, (int)e->ld_table, \
                                 (int)e->ld_out, e->scale, drop))
    const bool whole = e->dim % 8 == 0;
    if (!vec && many) GM_FORWARD(false, false, 2);
    else if (!vec) GM_FORWARD(false, false, 1);
    else if (!whole) GM_FORWARD(true, false, 1);
    else if (many) GM_FORWARD(true, true, 4);
    else GM_FORWARD(true, true, 1);
#undef GM_FORWARD
    d->launches++;
    GM_CUDA_CHECK(cudaGetLastError());
    return GM_OK;
}

template <typename T, typename G>
static int launch_embedding_backward(Device* d, const gm_embedding_t* e, uintptr_t tokens, uintptr_t dout, const Drop& drop,
                                     uintptr_t dtable, bool accumulate, uintptr_t ws) {
    const EmbSpace s = embedding_space(e);
    unsigned long long* words = (unsigned long long*)(ws + s.words0);
    unsigned long long* other = (unsigned long long*)(ws + s.words1);
    unsigned char* used = accumulate ? nullptr : (unsigned char*)(ws + s.used);
    int* split = (int*)(ws + s.split);
    float* pieces = (float*)(ws + s.pieces);
    const int64_t n = e->tokens;
    GM_CUDA_CHECK(launch_chained(token_sort_tile_kernel, dim3((unsigned)((n + kSortTile - 1) / kSortTile)), dim3(kSortTile), 0, d->stream, (const int*)tokens, n,
                                 e->vocab, e->padding_token, words, used, split));
    d->launches++;
    for (int64_t run = kSortTile; run < n; run *= kMergeWays) {
        GM_CUDA_CHECK(launch_chained(token_merge_kernel, dim3((unsigned)((n + 127) / 128)), dim3(128), 0, d->stream, words, other, n, (int)run,
                                     run == kSortTile ? used : nullptr, (unsigned)e->vocab));
        d->launches++;
        unsigned long long* t = words; words = other; other = t;
    }
    const bool vec = dout % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0 && dtable % 16 == 0 && e->ld_table * (int)sizeof(G) % 16 == 0;
    const bool whole = e->dim % 8 == 0;
    const int64_t groups = (e->dim + 7) / 8;
    const int piece = piece_of(e);
    const int lanes = lanes_of(groups, 8, kSumThreads);
    const dim3 sum_block((unsigned)lanes, (unsigned)(kSumThreads / lanes));
    const int64_t chunks = (n + piece - 1) / piece, col_ctas = (groups + lanes - 1) / lanes;
    const int64_t sum_ctas = (chunks + sum_block.y - 1) / sum_block.y * col_ctas;
    // a zeroing CTA has about 64 KB to write
    const int64_t fit = (64 << 10) / (e->dim * (int64_t)sizeof(G));
    const int zero_rows = (int)(fit < 16 ? 16 : fit > kZeroRowsMost ? kZeroRowsMost : fit);
    const int64_t zero_ctas = accumulate ? 0 : (e->vocab + zero_rows - 1) / zero_rows;
    if (sum_ctas + zero_ctas > 0x7fffffff) { set_error("%lld tokens of %lld columns are too many", (long long)n, (long long)e->dim); return GM_ERR_BAD_SIZE; }
    // narrow tables: more ways, the longest row's share is the time; wide ones: fewer, wider CTAs (0.322
    // against 0.336 ms at 65,536 x 4,096)
    const int join_lanes = lanes_of(groups, 8, groups >= 256 ? kJoinLanesMost : kJoinLanesMost / 2);
    const dim3 join_block((unsigned)join_lanes, (unsigned)(kJoinThreads / join_lanes));
    const int64_t join_most = chunks * ((groups + join_lanes - 1) / join_lanes);
    const unsigned join_grid = (unsigned)(join_most < d->sm_count * 8 ? join_most : d->sm_count * 8);
#define GM_SUM(VEC, WHOLE, ADD)                                                                                                              \
    do {                                                                                                                                     \
        GM_CUDA_CHECK(launch_chained(embedding_sum_kernel<T, G, VEC, WHOLE, ADD>, dim3((unsigned)(sum_ctas + zero_ctas)), sum_block,        \
                                     0, d->stream, (const T*)dout, words, used, pieces, split, (G*)dtable, (int)n, (int)e->dim,              \
                                     (int)e->vocab, (int)e->ld_table, (int)e->ld_out, e->scale, piece, (int)col_ctas, (int)sum_ctas,    \
                                     zero_rows, drop));                                                                                  \
        if (chunks > 1)                                                                                                                      \
            GM_CUDA_CHECK(launch_chained(embedding_join_kernel<G, VEC, WHOLE, ADD>, dim3(join_grid), join_block, 0, d->stream, words,        \
                                         pieces, split, (G*)dtable, (int)n, (int)e->dim, (int)e->ld_table, e->scale, piece, drop));          \
    } while (0)
    if (accumulate) {
        if (vec && whole) GM_SUM(true, true, true);
        else if (vec) GM_SUM(true, false, true);
        else GM_SUM(false, false, true);
    } else {
        if (vec && whole) GM_SUM(true, true, false);
        else if (vec) GM_SUM(true, false, false);
        else GM_SUM(false, false, false);
    }
#undef GM_SUM
    d->launches += chunks > 1 ? 2 : 1;
    return GM_OK;
}

}  // namespace gm

using namespace gm;

extern "C" {

int gm_embedding_forward_async(uintptr_t device_ptr, const gm_embedding_t* e, uintptr_t table, uintptr_t tokens, uintptr_t out,
                               const gm_dropout_t* dropout) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    GM_TRY(check_embedding(e));
    const int eb = dtype_bytes(e->dtype);
    GM_TRY(check_buffer(d, table, matrix_bytes(e->vocab, e->dim, e->ld_table, eb), eb, "embedding table"));
    GM_TRY(check_buffer(d, tokens, e->tokens * 4, 4, "tokens"));
    GM_TRY(check_buffer(d, out, matrix_bytes(e->tokens, e->dim, e->ld_out, eb), eb, "embedding output"));
    Drop drop;
    GM_TRY(make_drop(d, dropout, &drop));
    DeviceGuard g(d);
    if (e->dtype == GM_F32) return launch_embedding_forward<float>(d, e, table, tokens, out, drop);
    if (e->dtype == GM_F16) return launch_embedding_forward<__half>(d, e, table, tokens, out, drop);
    return launch_embedding_forward<__nv_bfloat16>(d, e, table, tokens, out, drop);
}

int64_t gm_embedding_workspace_bytes(const gm_embedding_t* e) {
    return check_embedding(e) == GM_OK ? embedding_space(e).total : -1;
}

int gm_embedding_backward_async(uintptr_t device_ptr, const gm_embedding_t* e, uintptr_t tokens, uintptr_t dout,
                                const gm_dropout_t* dropout, uintptr_t dtable, int grad_dtype, int accumulate,
                                uintptr_t workspace, int64_t workspace_bytes) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    GM_TRY(check_embedding(e));
    if (grad_dtype != GM_F32 && grad_dtype != e->dtype) { set_error("the gradient's type %d is neither Float32 nor that of dout", grad_dtype); return GM_ERR_BAD_ARG; }
    const int eb = dtype_bytes(e->dtype), gb = dtype_bytes(grad_dtype);
    GM_TRY(check_buffer(d, tokens, e->tokens * 4, 4, "tokens"));
    GM_TRY(check_buffer(d, dout, matrix_bytes(e->tokens, e->dim, e->ld_out, eb), eb, "embedding output gradient"));
    GM_TRY(check_buffer(d, dtable, matrix_bytes(e->vocab, e->dim, e->ld_table, gb), gb, "embedding table gradient"));
    const int64_t need = embedding_space(e).total;
    if (workspace_bytes < need) { set_error("workspace of %lld bytes, the call needs %lld", (long long)workspace_bytes, (long long)need); return GM_ERR_BAD_SIZE; }
    GM_TRY(check_buffer(d, workspace, need, 256, "workspace"));
    Drop drop;
    GM_TRY(make_drop(d, dropout, &drop));
    DeviceGuard g(d);
    const bool acc = accumulate != 0;
    if (e->dtype == GM_F32) return launch_embedding_backward<float, float>(d, e, tokens, dout, drop, dtable, acc, workspace);
    if (e->dtype == GM_F16) {
        if (grad_dtype == GM_F32) return launch_embedding_backward<__half, float>(d, e, tokens, dout, drop, dtable, acc, workspace);
        return launch_embedding_backward<__half, __half>(d, e, tokens, dout, drop, dtable, acc, workspace);
    }
    if (grad_dtype == GM_F32) return launch_embedding_backward<__nv_bfloat16, float>(d, e, tokens, dout, drop, dtable, acc, workspace);
    return launch_embedding_backward<__nv_bfloat16, __nv_bfloat16>(d, e, tokens, dout, drop, dtable, acc, workspace);
}

}  // extern "C"
