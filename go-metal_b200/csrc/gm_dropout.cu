// gm_dropout.cu -- dropout from a counter-based generator, with an optional residual:
//     y = residual + x * keep / (1 - p)
// The mask is a function of {seed, offset, element}, so it is never stored: the backward
// pass is the same call on the gradient.  Bound by HBM: one read of x (and of the residual),
// one write of y, 4 to 12 bytes per element.
#include "gm_lm.cuh"

namespace gm {

int make_drop(const Device* d, const gm_dropout_t* in, Drop* out) {
    *out = Drop{};
    out->up = 1.0f;
    if (!in) return GM_OK;
    if (!(in->p >= 0.0f && in->p <= 1.0f)) { set_error("dropout probability %g is outside [0, 1]", (double)in->p); return GM_ERR_BAD_ARG; }
    if (in->offset_device) GM_TRY(check_buffer(d, in->offset_device, 8, 8, "device offset of dropout"));
    for (int r = 0; r < 10; ++r) {
        out->key[2 * r] = (unsigned)in->seed + (unsigned)r * 0x9E3779B9u;
        out->key[2 * r + 1] = (unsigned)(in->seed >> 32) + (unsigned)r * 0xBB67AE85u;
    }
    out->o0 = (unsigned)in->offset;
    out->o1 = (unsigned)(in->offset >> 32);
    out->more = (const unsigned long long*)in->offset_device;
    out->cut = (unsigned)floor((double)in->p * 65536.0 + 0.5);
    out->up = out->cut < 65536u ? (float)(65536.0 / (65536.0 - (double)out->cut)) : 0.0f;
    return GM_OK;
}

int check_buffer(const Device* d, uintptr_t p, int64_t need, int64_t align, const char* what) {
    if (!p) { set_error("%s is nil", what); return GM_ERR_NIL_BUFFER; }
    if (p % (uintptr_t)align) { set_error("%s is not %lld-byte aligned", what, (long long)align); return GM_ERR_BAD_ARG; }
    const int ord = registered_ordinal(p);
    if (ord >= 0 && ord != d->ordinal) { set_error("%s lies on device %d, the handle's device is %d", what, ord, d->ordinal); return GM_ERR_BAD_ARG; }
    return buffer_holds(p, need, what) ? GM_OK : GM_ERR_BAD_SIZE;
}

int check_matrix(int64_t rows, int64_t cols, int64_t ld, const char* what) {
    if (rows <= 0 || cols <= 0 || rows > 0x7fffffffLL || cols > (1LL << 30)) {
        set_error("%s: size %lld x %lld is outside [1, 2^31) x [1, 2^30]", what, (long long)rows, (long long)cols);
        return GM_ERR_BAD_SIZE;
    }
    if (ld > 0x7fffffffLL) { set_error("%s: row stride %lld is outside [1, 2^31)", what, (long long)ld); return GM_ERR_BAD_SIZE; }
    if (ld < cols) { set_error("%s: row stride %lld is smaller than its %lld columns", what, (long long)ld, (long long)cols); return GM_ERR_BAD_ARG; }
    if (rows * ld > (1LL << 60)) { set_error("%s: %lld rows of stride %lld hold more than 2^60 elements", what, (long long)rows, (long long)ld); return GM_ERR_BAD_SIZE; }
    return GM_OK;
}

// One thread takes kDropVec groups of eight elements, a CTA's width apart, and issues their
// loads before it runs the generator.  Flat: the matrices are contiguous and a group may cross rows.
// Rows: a group lies inside a row and is a block of the generator (cols is a multiple of
// eight).  Odd: a group lies inside a row and may begin inside a block, which costs the generator
// twice.  The elements behind the last whole group, of the matrix or of each row, go one by one.
// VEC: rows begin on 16-byte boundaries.  bf16 without a residual, 16,384 x 4,096: 57 us flat, 70 us by
// rows, 84 us flat at an odd address, 123 us with 4,091 columns (all element by element: 176 and 188 us).
constexpr int kDropThreads = 256;
constexpr int kDropVec = 2;
enum class Walk { Flat, Rows, Odd };

template <typename T, bool RES, Walk WALK, bool VEC>
__global__ void __launch_bounds__(kDropThreads)
dropout_kernel(const T* x, const T* res, T* y, const long long n, const int cols, const int row_groups,
               const long long ld_x, const long long ld_r, const long long ld_y, const __grid_constant__ Drop d) {
    chain_begin();
    const DropOffset o = drop_begin(d);
    const long long g0 = (long long)blockIdx.x * (kDropThreads * kDropVec) + threadIdx.x;
    Eight<T, VEC> xv[kDropVec], rv[kDropVec];
    long long row[kDropVec], col[kDropVec];
    int live[kDropVec];                                                    // elements of the group, at most eight
#pragma unroll
    for (int i = 0; i < kDropVec; ++i) {
        const long long g = g0 + (long long)i * kDropThreads;
        if (WALK == Walk::Flat) {
            row[i] = 0;
            col[i] = g * 8;
            live[i] = col[i] + 8 <= n ? 8 : col[i] < n ? (int)(n - col[i]) : 0;
        } else {
            row[i] = g / row_groups;
            col[i] = (g - row[i] * row_groups) * 8;
            live[i] = row[i] * cols >= n ? 0 : WALK == Walk::Rows || col[i] + 8 <= cols ? 8 : (int)(cols - col[i]);
        }
        if (live[i] < 8) continue;
        xv[i].template load<false>(x + row[i] * ld_x + col[i]);
        if (RES) rv[i].template load<false>(res + row[i] * ld_r + col[i]);
    }
#pragma unroll
    for (int i = 0; i < kDropVec; ++i) {
        const unsigned long long first = (unsigned long long)(WALK == Walk::Flat ? col[i] : row[i] * cols + col[i]);
        if (WALK != Walk::Rows && live[i] < 8) {
            if (live[i] == 0) continue;
            const unsigned keep = drop_mask8(d, o, first);
            for (int k = 0; k < live[i]; ++k) {
                float v = (keep >> k) & 1u ? __fmul_rn(to_f32<T>(x[row[i] * ld_x + col[i] + k]), d.up) : 0.0f;
                if (RES) v = __fadd_rn(to_f32<T>(res[row[i] * ld_r + col[i] + k]), v);
                y[row[i] * ld_y + col[i] + k] = from_f32<T>(v);
            }
            continue;
        }
        if (WALK == Walk::Rows && live[i] == 0) continue;
        float v[8], r[8];
        widen8<T>(xv[i].r, v);
        if (RES) widen8<T>(rv[i].r, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __fmul_rn(v[k], d.up);
        drop8<WALK != Walk::Odd>(d, o, first, v);                         // a dropped NaN is dropped
        if (RES) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(r[k], v[k]);
        }
        Eight<T, VEC>::store(y + row[i] * ld_y + col[i], v);
    }
}

template <typename T, bool RES>
static int launch_dropout(Device* d, int64_t rows, int64_t cols, uintptr_t x, int64_t ld_x, uintptr_t r, int64_t ld_r,
                          uintptr_t y, int64_t ld_y, const Drop& drop) {
    const int64_t n = rows * cols;
    const int eb = (int)sizeof(T);
    const bool flat = rows == 1 || (ld_x == cols && ld_y == cols && (!RES || ld_r == cols));
    const bool strides = flat || (ld_x * eb % 16 == 0 && ld_y * eb % 16 == 0 && (!RES || ld_r * eb % 16 == 0));
    const bool vec = strides && x % 16 == 0 && y % 16 == 0 && (!RES || r % 16 == 0);
    const int64_t row_groups = (cols + 7) / 8, groups = flat ? (n + 7) / 8 : rows * row_groups;
    const int64_t grid = (groups + kDropThreads * kDropVec - 1) / (kDropThreads * kDropVec);
    if (grid > 0x7fffffff) { set_error("%lld x %lld elements are too many", (long long)rows, (long long)cols); return GM_ERR_BAD_SIZE; }
#define GM_DROP(WALK, VEC)                                                                                                             \
    GM_CUDA_CHECK(launch_chained(dropout_kernel<T, RES, WALK, VEC>, dim3((unsigned)grid), dim3(kDropThreads), 0, d->stream, (const T*)x, \
                                 (const T*)r, (T*)y, n, (int)cols, (int)row_groups, ld_x, ld_r, ld_y, drop))
    if (flat && vec) GM_DROP(Walk::Flat, true);
    else if (flat) GM_DROP(Walk::Flat, false);
    else if (cols % 8 == 0 && vec) GM_DROP(Walk::Rows, true);
    else if (cols % 8 == 0) GM_DROP(Walk::Rows, false);
    else if (vec) GM_DROP(Walk::Odd, true);
    else GM_DROP(Walk::Odd, false);
#undef GM_DROP
    d->launches++;
    return GM_OK;
}

}  // namespace gm

using namespace gm;

extern "C" int gm_dropout_async(uintptr_t device_ptr, int dtype, int64_t rows, int64_t cols, uintptr_t x, int64_t ld_x,
                                uintptr_t residual, int64_t ld_residual, uintptr_t y, int64_t ld_y, const gm_dropout_t* dropout) {
    Device* d = as_device(device_ptr);
    if (!d) return GM_ERR_NIL_DEVICE;
    const int eb = dtype_bytes(dtype);
    if (!eb) { set_error("element type %d is not Float32, Float16 or BFloat16", dtype); return GM_ERR_BAD_ARG; }
    if (!dropout) { set_error("dropout argument is nil"); return GM_ERR_BAD_ARG; }
    GM_TRY(check_matrix(rows, cols, ld_x, "dropout input"));
    GM_TRY(check_matrix(rows, cols, ld_y, "dropout output"));
    if (residual) GM_TRY(check_matrix(rows, cols, ld_residual, "dropout residual"));
    GM_TRY(check_buffer(d, x, matrix_bytes(rows, cols, ld_x, eb), eb, "dropout input"));
    GM_TRY(check_buffer(d, y, matrix_bytes(rows, cols, ld_y, eb), eb, "dropout output"));
    if (residual) GM_TRY(check_buffer(d, residual, matrix_bytes(rows, cols, ld_residual, eb), eb, "dropout residual"));
    if ((y == x && ld_y != ld_x) || (residual && y == residual && ld_y != ld_residual)) {
        set_error("an in-place call needs equal row strides");
        return GM_ERR_BAD_ARG;
    }
    Drop drop;
    GM_TRY(make_drop(d, dropout, &drop));
    DeviceGuard g(d);
    if (dtype == GM_F32) return residual ? launch_dropout<float, true>(d, rows, cols, x, ld_x, residual, ld_residual, y, ld_y, drop)
                                         : launch_dropout<float, false>(d, rows, cols, x, ld_x, 0, 0, y, ld_y, drop);
    if (dtype == GM_F16) return residual ? launch_dropout<__half, true>(d, rows, cols, x, ld_x, residual, ld_residual, y, ld_y, drop)
                                         : launch_dropout<__half, false>(d, rows, cols, x, ld_x, 0, 0, y, ld_y, drop);
    return residual ? launch_dropout<__nv_bfloat16, true>(d, rows, cols, x, ld_x, residual, ld_residual, y, ld_y, drop)
                    : launch_dropout<__nv_bfloat16, false>(d, rows, cols, x, ld_x, 0, 0, y, ld_y, drop);
}
