// gm_embedding.cu -- token embedding with scaling and dropout, and its gradient.
//
//   forward   out[t] = drop(scale * table[token_t])
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
constexpr int kMergeWays = 32;           // sorted runs that one merge pass joins
constexpr int kPiece = 64;               // sorted tokens whose sum is one piece of a long row

// ---------------------------------------------------------------- forward
// A CTA is tx lanes over groups of eight columns times ty tokens; each thread takes ROWS
// tokens and issues all its loads first.  VEC: rows begin on 16-byte boundaries; the last
// dim % 8 columns, and everything without VEC, go element by element.
template <typename T, bool VEC, int ROWS>
__global__ void __launch_bounds__(kEmbThreads)
embedding_forward_kernel(const T* __restrict__ table, const int* __restrict__ tokens, T* __restrict__ out,
                         const long long n, const long long dim, const long long vocab, const long long ld_table,
                         const long long ld_out, const float scale, Drop d) {
    drop_begin(d);
    const long long groups = (dim + 7) >> 3;
    const long long t0 = ((long long)blockIdx.x * blockDim.y + threadIdx.y) * ROWS;
    long long tok[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        tok[r] = t0 + r < n ? (long long)__ldg(tokens + t0 + r) : -1;
        if (tok[r] >= vocab) tok[r] = -1;
    }
    for (long long g = (long long)blockIdx.y * blockDim.x + threadIdx.x; g < groups; g += (long long)gridDim.y * blockDim.x) {
        const long long c = g << 3;
        if (VEC && c + 8 <= dim) {
            Raw8<T> raw[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (tok[r] >= 0) raw[r] = load8<T, true>(table + tok[r] * ld_table + c);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const long long t = t0 + r;
                if (t >= n) break;
                float x[8];
                if (tok[r] >= 0) {
                    widen8<T>(raw[r], x);
                    const unsigned keep = drop_mask8(d, (unsigned long long)(t * dim + c));
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = (keep >> k) & 1u ? __fmul_rn(__fmul_rn(x[k], scale), d.up) : 0.0f;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = 0.0f;
                }
                store8<T>(out + t * ld_out + c, x);
            }
        } else {
            for (int r = 0; r < ROWS; ++r) {
                const long long t = t0 + r;
                if (t >= n) break;
                const unsigned keep = tok[r] >= 0 ? drop_mask8(d, (unsigned long long)(t * dim + c)) : 0u;
                for (int k = 0; k < 8 && c + k < dim; ++k) {
                    float x = 0.0f;
                    if ((keep >> k) & 1u) x = __fmul_rn(__fmul_rn(to_f32<T>(table[tok[r] * ld_table + c + k]), scale), d.up);
                    out[t * ld_out + c + k] = from_f32<T>(x);
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

__device__ __forceinline__ long long lower_bound(const unsigned long long* __restrict__ a, long long lo, long long hi, unsigned long long x) {
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (__ldg(a + mid) < x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Joins kMergeWays sorted runs of `run` words: a word's place is the number of smaller words
// in every run of its group, found by bisection, so one pass has no serial part.
__global__ void __launch_bounds__(256)
token_merge_kernel(const unsigned long long* __restrict__ in, unsigned long long* __restrict__ out, const long long n, const long long run) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const unsigned long long key = __ldg(in + i);
    const long long base = i / (run * kMergeWays) * (run * kMergeWays);
    const long long mine = base + (i - base) / run * run;
    long long rank = i - mine;
    for (int q = 0; q < kMergeWays; ++q) {
        const long long a = base + q * run;
        if (a >= n) break;
        if (a == mine) continue;
        const long long b = a + run < n ? a + run : n;
        rank += lower_bound(in, a, b, key) - a;
    }
    out[base + rank] = key;
}

// first[v] = number of sorted words whose token is below v, for v in [0, vocab].
__global__ void __launch_bounds__(256)
token_first_kernel(const unsigned long long* __restrict__ words, const long long n, const long long vocab, int* __restrict__ first) {
    const long long v = (long long)blockIdx.x * 256 + threadIdx.x;
    if (v <= vocab) first[v] = (int)lower_bound(words, 0, n, (unsigned long long)v << 32);
}

// ---------------------------------------------------------------- backward sums
// Adds the rows of dout that words [a, b) name, in order, to acc: eight columns from c.
template <typename T, bool VEC>
__device__ __forceinline__ void add_rows(const T* __restrict__ dout, const unsigned long long* __restrict__ words, long long a, const long long b,
                                         const long long c, const long long dim, const long long ld_out, const Drop& d, float (&acc)[8]) {
    if (VEC && c + 8 <= dim) {
        constexpr int DEEP = 8;
        while (a < b) {
            Raw8<T> raw[DEEP];
            unsigned pos[DEEP];
            const int m = b - a < DEEP ? (int)(b - a) : DEEP;
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
                if (j < m) {
                    pos[j] = (unsigned)__ldg(words + a + j);
                    raw[j] = load8<T, false>(dout + (long long)pos[j] * ld_out + c);
                }
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
                if (j < m) {
                    float x[8];
                    widen8<T>(raw[j], x);
                    const unsigned keep = drop_mask8(d, (unsigned long long)((long long)pos[j] * dim + c));
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[k] = __fadd_rn(acc[k], (keep >> k) & 1u ? x[k] : 0.0f);
                }
            a += m;
        }
    } else {
        for (; a < b; ++a) {
            const long long p = (long long)(unsigned)__ldg(words + a);
            const unsigned keep = drop_mask8(d, (unsigned long long)(p * dim + c));
            for (int k = 0; k < 8 && c + k < dim; ++k)
                if ((keep >> k) & 1u) acc[k] = __fadd_rn(acc[k], to_f32<T>(dout[p * ld_out + c + k]));
        }
    }
}

// A row whose sorted words lie in more than one chunk of kPiece words is summed in pieces, one
// per chunk, so that a token that fills half the batch is still spread over the GPU.  Slot 2j
// holds chunk j's part of a row that began before it, slot 2j + 1 that of a row that begins in
// it and goes on.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128)
embedding_pieces_kernel(const T* __restrict__ dout, const unsigned long long* __restrict__ words, float* __restrict__ pieces,
                        const long long n, const long long dim, const long long vocab, const long long ld_out, Drop d) {
    __shared__ unsigned tok[kPiece];
    const int tid = threadIdx.x;
    const long long begin = (long long)blockIdx.x * kPiece;
    const int len = n - begin < kPiece ? (int)(n - begin) : kPiece;
    if (tid < len) tok[tid] = (unsigned)(__ldg(words + begin + tid) >> 32);
    __syncthreads();
    const unsigned head = tok[0], tail = tok[len - 1];
    const bool from_before = begin > 0 && head < vocab && (unsigned)(__ldg(words + begin - 1) >> 32) == head;
    const bool goes_on = begin + len < n && tail < vocab && (unsigned)(__ldg(words + begin + len) >> 32) == tail;
    if (!from_before && !goes_on) return;
    const int n_head = __syncthreads_count(tid < len && tok[tid] == head);
    const int n_tail = __syncthreads_count(tid < len && tok[tid] == tail);
    drop_begin(d);
    const long long groups = (dim + 7) >> 3;
    for (long long g = (long long)blockIdx.y * 128 + tid; g < groups; g += (long long)gridDim.y * 128) {
        const long long c = g << 3;
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            if (side == 0 ? !from_before : !goes_on || (from_before && n_head == len)) continue;
            float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            add_rows<T, VEC>(dout, words, side == 0 ? begin : begin + len - n_tail, side == 0 ? begin + n_head : begin + len, c, dim, ld_out, d, acc);
            float* p = pieces + (2 * (long long)blockIdx.x + side) * (groups * 8) + c;
            reinterpret_cast<float4*>(p)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        }
    }
}

// HEADS false: one item per row of the table, every row is written.  HEADS true (accumulate):
// one item per sorted word, those that begin a row add to it, the others leave.
template <typename T, typename G, bool VEC, bool HEADS>
__global__ void __launch_bounds__(kEmbThreads)
embedding_rows_kernel(const T* __restrict__ dout, const unsigned long long* __restrict__ words, const int* __restrict__ first,
                      const float* __restrict__ pieces, G* dtable, const long long n, const long long dim, const long long vocab,
                      const long long ld_table, const long long ld_out, const float scale, Drop d) {
    const long long item = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    long long v, a, b;
    if (HEADS) {
        if (item >= n) return;
        const unsigned key = (unsigned)(__ldg(words + item) >> 32);
        if (key >= vocab || (item > 0 && (unsigned)(__ldg(words + item - 1) >> 32) == key)) return;
        v = key;
        a = item;
        b = lower_bound(words, item + 1, n, (unsigned long long)(key + 1u) << 32);
    } else {
        if (item >= vocab) return;
        v = item;
        a = __ldg(first + v);
        b = __ldg(first + v + 1);
    }
    drop_begin(d);
    const long long groups = (dim + 7) >> 3;
    const float up = __fmul_rn(scale, d.up);
    const long long ca = a / kPiece, cb = b > a ? (b - 1) / kPiece : ca;
    for (long long g = (long long)blockIdx.y * blockDim.x + threadIdx.x; g < groups; g += (long long)gridDim.y * blockDim.x) {
        const long long c = g << 3;
        float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (b > a) {
            if (ca == cb) {
                add_rows<T, VEC>(dout, words, a, b, c, dim, ld_out, d, acc);
            } else {
                // a row that begins on a chunk's first word left that chunk's part in the odd slot
#pragma unroll 4
                for (long long j = ca; j <= cb; ++j) {
                    const float4* p = reinterpret_cast<const float4*>(pieces + (2 * j + (j == ca ? 1 : 0)) * (groups * 8) + c);
                    const float4 x = p[0], y = p[1];
                    acc[0] = __fadd_rn(acc[0], x.x); acc[1] = __fadd_rn(acc[1], x.y);
                    acc[2] = __fadd_rn(acc[2], x.z); acc[3] = __fadd_rn(acc[3], x.w);
                    acc[4] = __fadd_rn(acc[4], y.x); acc[5] = __fadd_rn(acc[5], y.y);
                    acc[6] = __fadd_rn(acc[6], y.z); acc[7] = __fadd_rn(acc[7], y.w);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] = __fmul_rn(acc[k], up);
        }
        G* to = dtable + v * ld_table + c;
        if (VEC && c + 8 <= dim) {
            if (HEADS) {
                float old[8];
                widen8<G>(load8<G, false>(to), old);
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] = __fadd_rn(old[k], acc[k]);
            }
            store8<G>(to, acc);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < dim) to[k] = from_f32<G>(HEADS ? __fadd_rn(to_f32<G>(to[k]), acc[k]) : acc[k]);
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

// CTA of tx lanes over the column groups and ty rows, and the grid's second axis for wide rows.
static void row_shape(int64_t dim, dim3* block, unsigned* grid_y) {
    const int64_t groups = (dim + 7) / 8;
    int tx = 8;
    while (tx < kEmbThreads && tx < groups) tx <<= 1;
    *block = dim3((unsigned)tx, (unsigned)(kEmbThreads / tx));
    const int64_t y = (groups + tx - 1) / tx;
    *grid_y = (unsigned)(y < 65535 ? y : 65535);
}

template <typename T>
static int launch_embedding_forward(Device* d, const gm_embedding_t* e, uintptr_t table, uintptr_t tokens, uintptr_t out, const Drop& drop) {
    dim3 block;
    unsigned gy = 1;
    row_shape(e->dim, &block, &gy);
    const bool vec = table % 16 == 0 && out % 16 == 0 && e->ld_table * (int)sizeof(T) % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0;
    const dim3 grid((unsigned)((e->tokens + block.y - 1) / block.y), gy);
    if (vec) embedding_forward_kernel<T, true, 1><<<grid, block, 0, d->stream>>>((const T*)table, (const int*)tokens, (T*)out, e->tokens, e->dim, e->vocab, e->ld_table, e->ld_out, e->scale, drop);
    else embedding_forward_kernel<T, false, 1><<<grid, block, 0, d->stream>>>((const T*)table, (const int*)tokens, (T*)out, e->tokens, e->dim, e->vocab, e->ld_table, e->ld_out, e->scale, drop);
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
        token_merge_kernel<<<(unsigned)((n + 255) / 256), 256, 0, d->stream>>>(words, other, n, run);
        d->launches++;
        unsigned long long* t = words; words = other; other = t;
    }
    if (!accumulate) {
        token_first_kernel<<<(unsigned)((e->vocab + 256) / 256), 256, 0, d->stream>>>(words, n, e->vocab, first);
        d->launches++;
    }
    const bool vec = dout % 16 == 0 && e->ld_out * (int)sizeof(T) % 16 == 0 && dtable % 16 == 0 && e->ld_table * (int)sizeof(G) % 16 == 0;
    const int64_t groups = (e->dim + 7) / 8;
    if (n > kPiece) {
        const int64_t y = (groups + 127) / 128;
        const dim3 grid((unsigned)((n + kPiece - 1) / kPiece), (unsigned)(y < 65535 ? y : 65535));
        if (vec) embedding_pieces_kernel<T, true><<<grid, 128, 0, d->stream>>>((const T*)dout, words, pieces, n, e->dim, e->vocab, e->ld_out, drop);
        else embedding_pieces_kernel<T, false><<<grid, 128, 0, d->stream>>>((const T*)dout, words, pieces, n, e->dim, e->vocab, e->ld_out, drop);
        d->launches++;
    }
    dim3 block;
    unsigned gy = 1;
    row_shape(e->dim, &block, &gy);
    const int64_t items = accumulate ? n : e->vocab;
    const dim3 grid((unsigned)((items + block.y - 1) / block.y), gy);
#define GM_ROWS(VEC, HEADS)                                                                                                   \
    embedding_rows_kernel<T, G, VEC, HEADS><<<grid, block, 0, d->stream>>>((const T*)dout, words, first, pieces, (G*)dtable, n, \
                                                                           e->dim, e->vocab, e->ld_table, e->ld_out, e->scale, drop)
    if (accumulate) { if (vec) GM_ROWS(true, true); else GM_ROWS(false, true); }
    else { if (vec) GM_ROWS(true, false); else GM_ROWS(false, false); }
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
