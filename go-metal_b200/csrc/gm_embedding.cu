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
constexpr int kPiece = 32;               // sorted words whose sum is one piece of a long row

// ---------------------------------------------------------------- forward
// A CTA is tx lanes over groups of eight columns times ty tokens; each thread takes ROWS
// tokens and issues all its loads first.  VEC: rows begin on 16-byte boundaries; the last
// dim % 8 columns, and everything without VEC, go element by element.  WHOLE: dim is a multiple
// of eight, so a group is a block of dropout's generator.
template <typename T, bool VEC, bool WHOLE, int ROWS>
__global__ void __launch_bounds__(kEmbThreads, 4)
embedding_forward_kernel(const T* __restrict__ table, const int* __restrict__ tokens, T* __restrict__ out, const int n, const int dim,
                         const int vocab, const int ld_table, const int ld_out, const float scale, const __grid_constant__ Drop d) {
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
        if (VEC && (WHOLE || c + 8 <= dim)) {
            Raw8<T> raw[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (tok[r] >= 0) raw[r] = load8<T, true>(table + (long long)tok[r] * ld_table + c);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (r >= live) break;
                float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                if (tok[r] >= 0) {
                    widen8<T>(raw[r], x);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = __fmul_rn(x[k], up);
                    drop8<WHOLE>(d, o, (unsigned long long)((t0 + r) * dim + c), x);
                }
                store8<T>(out + (t0 + r) * ld_out + c, x);
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
// through shared memory.
__global__ void __launch_bounds__(kSortTile)
token_sort_tile_kernel(const int* __restrict__ tokens, const long long n, const long long vocab, const long long padding,
                       unsigned long long* __restrict__ out) {
    __shared__ unsigned long long buf[kSortTile];
    const int tid = threadIdx.x;
    const long long i = (long long)blockIdx.x * kSortTile + tid;
    unsigned long long key = i < n ? sort_word(tokens, i, vocab, padding) : ~0ull;
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
token_merge_kernel(const unsigned long long* __restrict__ in, unsigned long long* __restrict__ out, const long long n, const int run) {
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= n) return;
    const unsigned long long word = __ldg(in + i);
    const unsigned token = (unsigned)(word >> 32);
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

// first[v] = number of sorted words whose token is below v, for v in [0, vocab].
__global__ void __launch_bounds__(256)
token_first_kernel(const unsigned long long* __restrict__ words, const long long n, const long long vocab, int* __restrict__ first) {
    const long long v = (long long)blockIdx.x * 256 + threadIdx.x;
    if (v <= vocab) first[v] = (int)first_at(words, 0, n, (unsigned)v);
}

// ---------------------------------------------------------------- backward sums
// Adds the rows of dout that words [a, b) name, in order, to acc: COLS groups of eight columns,
// `apart` groups from one to the next, the first one g.  COLS x DEEP loads are in flight.
template <typename T, bool VEC, bool WHOLE, int COLS, int DEEP>
__device__ __forceinline__ void add_rows(const T* __restrict__ dout, const unsigned long long* __restrict__ words, long long a, const long long b,
                                         const int g, const int apart, const int dim, const int ld_out, const Drop& d, const DropOffset& o,
                                         float (&acc)[COLS][8]) {
    const int c0 = g << 3;
    if (VEC && (WHOLE || c0 + 8 <= dim)) {                            // without WHOLE there is one group per thread
        while (a < b) {
            Raw8<T> raw[DEEP][COLS];
            unsigned pos[DEEP];
            const int m = b - a < DEEP ? (int)(b - a) : DEEP;
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
                if (j < m) {
                    pos[j] = __ldg(reinterpret_cast<const unsigned*>(words + a + j));
                    const T* row = dout + (long long)pos[j] * ld_out + c0;
#pragma unroll
                    for (int q = 0; q < COLS; ++q)
                        if (q == 0 || c0 + q * apart * 8 < dim) raw[j][q] = load8<T, false>(row + q * apart * 8);
                }
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
                if (j < m) {
#pragma unroll
                    for (int q = 0; q < COLS; ++q)
                        if (q == 0 || c0 + q * apart * 8 < dim) {
                            float x[8];
                            widen8<T>(raw[j][q], x);
                            drop8<WHOLE>(d, o, (unsigned long long)((long long)pos[j] * dim + c0 + q * apart * 8), x);
#pragma unroll
                            for (int k = 0; k < 8; ++k) acc[q][k] = __fadd_rn(acc[q][k], x[k]);
                        }
                }
            a += m;
        }
    } else {
        for (; a < b; ++a) {
            const long long p = __ldg(reinterpret_cast<const unsigned*>(words + a));
            const unsigned keep = drop_mask8(d, o, (unsigned long long)(p * dim + c0));
            for (int k = 0; k < 8 && k < dim - c0; ++k)
                if ((keep >> k) & 1u) acc[0][k] = __fadd_rn(acc[0][k], to_f32<T>(dout[p * ld_out + c0 + k]));
        }
    }
}

// The row of table that a word with this token belongs to: its words are [a, b).
__device__ __forceinline__ void row_of(const unsigned long long* __restrict__ words, const int* __restrict__ first, const long long n,
                                       const unsigned key, long long* a, long long* b) {
    if (first) {
        *a = __ldg(first + key);
        *b = __ldg(first + key + 1);
    } else {
        *a = first_at(words, 0, n, key);
        *b = first_at(words, *a, n, key + 1u);
    }
}

// A row of more than kPiece words is summed in pieces of kPiece, counted from its first word, so
// that a token that fills half the batch is still spread over the GPU.  A piece that begins at
// word s leaves its sum in slot 2 (s / kPiece), the row's first piece in the slot behind that:
// among kPiece neighbouring words there begin at most one first piece and one other.
template <typename T, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(128)
embedding_pieces_kernel(const T* __restrict__ dout, const unsigned long long* __restrict__ words, const int* __restrict__ first,
                        float* __restrict__ pieces, const int n, const int dim, const int vocab, const int ld_out, const __grid_constant__ Drop d) {
    __shared__ long long from[2], to[2];
    const int tid = threadIdx.x;
    const long long begin = (long long)blockIdx.x * kPiece;
    if (tid < 2) from[tid] = -1;
    __syncthreads();
    if (tid < kPiece && begin + tid < n) {
        const long long i = begin + tid;
        const unsigned key = token_at(words, i);
        // a row of more than kPiece words has a word of its own kPiece places on or back
        const bool maybe = key < (unsigned)vocab && ((i + kPiece < n && token_at(words, i + kPiece) == key) || (i >= kPiece && token_at(words, i - kPiece) == key));
        if (maybe) {
            long long a, b;
            row_of(words, first, n, key, &a, &b);
            if ((i - a) % kPiece == 0) {
                const int side = i == a ? 1 : 0;
                from[side] = i;
                to[side] = i + kPiece < b ? i + kPiece : b;
            }
        }
    }
    __syncthreads();
    if (from[0] < 0 && from[1] < 0) return;
    const DropOffset o = drop_begin(d);
    const int groups = (int)(((unsigned)dim + 7u) >> 3);
    for (int g = blockIdx.y * 128 + tid; g < groups; g += gridDim.y * 128) {
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            if (from[side] < 0) continue;
            float acc[1][8] = {};
            add_rows<T, VEC, WHOLE, 1, 8>(dout, words, from[side], to[side], g, 0, dim, ld_out, d, o, acc);
            float4* p = reinterpret_cast<float4*>(pieces + ((2 * (long long)blockIdx.x + side) * groups + g) * 8);
            p[0] = make_float4(acc[0][0], acc[0][1], acc[0][2], acc[0][3]);
            p[1] = make_float4(acc[0][4], acc[0][5], acc[0][6], acc[0][7]);
        }
    }
}

// HEADS false: items are the table's rows, every one is written.  HEADS true (accumulate): items
// are the sorted words; one that begins a row adds to it, the others are passed over.  A CTA is
// tx lanes, each with COLS groups of eight columns, times ty items at a time, kRowTurns times.
constexpr int kRowTurns = 8;
constexpr int kRowLanesLeast = 8;
template <typename T, typename G, bool VEC, bool WHOLE, bool HEADS, int COLS>
__global__ void __launch_bounds__(kEmbThreads, 3)
embedding_rows_kernel(const T* __restrict__ dout, const unsigned long long* __restrict__ words, const int* __restrict__ first,
                      const float* __restrict__ pieces, G* dtable, const int n, const int dim, const int vocab, const int ld_table,
                      const int ld_out, const float scale, const __grid_constant__ Drop d) {
    // where the CTA's rows begin and end (its words' tokens, and the one before), read at once
    __shared__ int mark[kEmbThreads / kRowLanesLeast * kRowTurns + 1];
    const int items = blockDim.y * kRowTurns;
    const long long item0 = (long long)blockIdx.x * items;
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i <= items; i += kEmbThreads) {
        const long long at = HEADS ? item0 + i - 1 : item0 + i;
        if (HEADS) mark[i] = at >= 0 && at < n ? (int)token_at(words, at) : vocab;
        else mark[i] = at <= vocab ? __ldg(first + at) : 0;
    }
    __syncthreads();
    const DropOffset o = drop_begin(d);
    const int groups = (int)(((unsigned)dim + 7u) >> 3), lanes = blockDim.x;
    const float up = __fmul_rn(scale, d.up);
#pragma unroll 1
    for (int turn = 0; turn < kRowTurns; ++turn) {
        const int slot = turn * blockDim.y + threadIdx.y;
        const long long item = item0 + slot;
        int v;
        long long a, b;
        if (HEADS) {
            if (item >= n) return;
            v = mark[slot + 1];
            if (v >= vocab || (item > 0 && mark[slot] == v)) continue;
            a = item;
            b = item + 1;
            if (b < n && token_at(words, b) == (unsigned)v) b = first_at(words, b, n, (unsigned)v + 1u);
        } else {
            if (item >= vocab) return;
            v = (int)item;
            a = mark[slot];
            b = mark[slot + 1];
        }
        G* const row = dtable + (long long)v * ld_table;
        for (int g = blockIdx.y * lanes * COLS + threadIdx.x; g < groups; g += gridDim.y * lanes * COLS) {
            const int c = g << 3;
            if (!HEADS && VEC && WHOLE && a == b) {                       // a row of zeros, most of them in a large table
#pragma unroll
                for (int q = 0; q < COLS; ++q)
                    if (q == 0 || c + q * lanes * 8 < dim) {
                        uint4* to = reinterpret_cast<uint4*>(row + c + q * lanes * 8);
                        __stcs(to, make_uint4(0u, 0u, 0u, 0u));
                        if (sizeof(G) == 4) __stcs(to + 1, make_uint4(0u, 0u, 0u, 0u));
                    }
                continue;
            }
            float acc[COLS][8] = {};
            if (b - a > kPiece) {
#pragma unroll 2
                for (long long s = a; s < b; s += kPiece) {
                    const float* p = pieces + (2 * (s / kPiece) + (s == a ? 1 : 0)) * groups * 8 + c;
#pragma unroll
                    for (int q = 0; q < COLS; ++q)
                        if (q == 0 || c + q * lanes * 8 < dim) {
                            const float4* at = reinterpret_cast<const float4*>(p + q * lanes * 8);
                            const float4 x = at[0], y = at[1];
                            acc[q][0] = __fadd_rn(acc[q][0], x.x); acc[q][1] = __fadd_rn(acc[q][1], x.y);
                            acc[q][2] = __fadd_rn(acc[q][2], x.z); acc[q][3] = __fadd_rn(acc[q][3], x.w);
                            acc[q][4] = __fadd_rn(acc[q][4], y.x); acc[q][5] = __fadd_rn(acc[q][5], y.y);
                            acc[q][6] = __fadd_rn(acc[q][6], y.z); acc[q][7] = __fadd_rn(acc[q][7], y.w);
                        }
                }
            } else if (b > a) {
                constexpr int DEEP = COLS == 1 ? (sizeof(T) == 2 ? 8 : 4) : (sizeof(T) == 2 ? 2 : 1);
                add_rows<T, VEC, WHOLE, COLS, DEEP>(dout, words, a, b, g, lanes, dim, ld_out, d, o, acc);
            }
#pragma unroll
            for (int q = 0; q < COLS; ++q) {
                if (q > 0 && c + q * lanes * 8 >= dim) break;
                G* to = row + c + q * lanes * 8;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[q][k] = __fmul_rn(acc[q][k], up);
                if (VEC && (WHOLE || c + 8 <= dim)) {
                    if (HEADS) {
                        float old[8];
                        widen8<G>(load8<G, false>(to), old);
#pragma unroll
                        for (int k = 0; k < 8; ++k) acc[q][k] = __fadd_rn(old[k], acc[q][k]);
                    }
                    store8<G>(to, acc[q]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < dim - c) to[k] = from_f32<G>(HEADS ? __fadd_rn(to_f32<G>(to[k]), acc[q][k]) : acc[q][k]);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- host side
struct EmbSpace { int64_t words0, words1, first, pieces, total; };

static int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }

static EmbSpace embedding_space(const gm_embedding_t* e) {
    EmbSpace s;
    s.words0 = 0;
    s.words1 = s.words0 + up256(e->tokens * 8);
    s.first = s.words1 + up256(e->tokens * 8);
    s.pieces = s.first + up256((e->vocab + 1) * 4);
    s.total = s.pieces + up256(2 * ((e->tokens + kPiece - 1) / kPiece) * ((e->dim + 7) / 8 * 8) * 4);
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

// CTA of tx lanes, each with `cols` column groups, and ty rows; the grid's second axis for wide rows.
static void row_shape(int64_t dim, int cols, dim3* block, unsigned* grid_y) {
    const int64_t groups = ((dim + 7) / 8 + cols - 1) / cols;
    int tx = kRowLanesLeast;
    while (tx < kEmbThreads && tx < groups) tx <<= 1;
    *block = dim3((unsigned)tx, (unsigned)(kEmbThreads / tx));
    const int64_t y = (groups + tx - 1) / tx;
    *grid_y = (unsigned)(y < 65535 ? y : 65535);
}

template <typename T>
static int launch_embedding_forward(Device* d, const gm_embedding_t* e, uintptr_t table, uintptr_t tokens, uintptr_t out, const Drop& drop) {
    dim3 block;
    unsigned gy = 1;
    row_shape(e->dim, 1, &block, &gy);
    const bool vec = table % 16 == 0 && out % 16 == 0 && e->ld_table * (int)sizeof(T) % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0;
    // four tokens per thread keep more loads in flight; a call too small for that takes one
    const bool many = e->tokens * gy >= (int64_t)d->sm_count * 8 * block.y;
#define GM_FORWARD(VEC, WHOLE, ROWS)                                                                                                            \
    embedding_forward_kernel<T, VEC, WHOLE, ROWS><<<dim3((unsigned)((e->tokens + block.y * ROWS - 1) / (block.y * ROWS)), gy), block, 0, d->stream>>>( \
        (const T*)table, (const int*)tokens, (T*)out, (int)e->tokens, (int)e->dim, (int)e->vocab, (int)e->ld_table, (int)e->ld_out, e->scale, drop)
    const bool whole = e->dim % 8 == 0;
    if (!vec) GM_FORWARD(false, false, 1);
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
    int* first = (int*)(ws + s.first);
    float* pieces = (float*)(ws + s.pieces);
    const int64_t n = e->tokens;
    token_sort_tile_kernel<<<(unsigned)((n + kSortTile - 1) / kSortTile), kSortTile, 0, d->stream>>>((const int*)tokens, n, e->vocab, e->padding_token, words);
    d->launches++;
    for (int64_t run = kSortTile; run < n; run *= kMergeWays) {
        token_merge_kernel<<<(unsigned)((n + 127) / 128), 128, 0, d->stream>>>(words, other, n, (int)run);
        d->launches++;
        unsigned long long* t = words; words = other; other = t;
    }
    if (!accumulate) {
        token_first_kernel<<<(unsigned)((e->vocab + 256) / 256), 256, 0, d->stream>>>(words, n, e->vocab, first);
        d->launches++;
    }
    const bool vec = dout % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0 && dtable % 16 == 0 && e->ld_table * (int)sizeof(G) % 16 == 0;
    const bool whole = e->dim % 8 == 0;
    const int64_t groups = (e->dim + 7) / 8;
    if (n > kPiece) {
        const int64_t y = (groups + 127) / 128;
        const dim3 grid((unsigned)((n + kPiece - 1) / kPiece), (unsigned)(y < 65535 ? y : 65535));
        if (vec && whole) embedding_pieces_kernel<T, true, true><<<grid, 128, 0, d->stream>>>((const T*)dout, words, accumulate ? nullptr : first, pieces, (int)n, (int)e->dim, (int)e->vocab, (int)e->ld_out, drop);
        else if (vec) embedding_pieces_kernel<T, true, false><<<grid, 128, 0, d->stream>>>((const T*)dout, words, accumulate ? nullptr : first, pieces, (int)n, (int)e->dim, (int)e->vocab, (int)e->ld_out, drop);
        else embedding_pieces_kernel<T, false, false><<<grid, 128, 0, d->stream>>>((const T*)dout, words, accumulate ? nullptr : first, pieces, (int)n, (int)e->dim, (int)e->vocab, (int)e->ld_out, drop);
        d->launches++;
    }
    // four groups per lane where that still fills a warp: the bookkeeping of a row is paid less often
    const bool wide = vec && whole && groups >= 128;
    dim3 block;
    unsigned gy = 1;
    row_shape(e->dim, wide ? 4 : 1, &block, &gy);
    const int64_t items = accumulate ? n : e->vocab;
    const int64_t per_cta = (int64_t)block.y * kRowTurns;
    const dim3 grid((unsigned)((items + per_cta - 1) / per_cta), gy);
#define GM_ROWS(VEC, WHOLE, HEADS, COLS)                                                                                        \
    embedding_rows_kernel<T, G, VEC, WHOLE, HEADS, COLS><<<grid, block, 0, d->stream>>>(                                         \
        (const T*)dout, words, first, pieces, (G*)dtable, (int)n, (int)e->dim, (int)e->vocab, (int)e->ld_table, (int)e->ld_out, e->scale, drop)
    if (accumulate) {
        if (wide) GM_ROWS(true, true, true, 4);
        else if (vec && whole) GM_ROWS(true, true, true, 1);
        else if (vec) GM_ROWS(true, false, true, 1);
        else GM_ROWS(false, false, true, 1);
    } else {
        if (wide) GM_ROWS(true, true, false, 4);
        else if (vec && whole) GM_ROWS(true, true, false, 1);
        else if (vec) GM_ROWS(true, false, false, 1);
        else GM_ROWS(false, false, false, 1);
    }
#undef GM_ROWS
    d->launches++;
    GM_CUDA_CHECK(cudaGetLastError());
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
    GM_TRY(make_drop(dropout, &drop));
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
    GM_TRY(make_drop(dropout, &drop));
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
