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
    return GM_OK;
}

// One thread takes kDropVec groups of eight elements, a CTA's width apart, and issues their
// loads before it runs the generator.  FLAT: the matrices are contiguous and a group may cross
// rows, the last n % 8 elements go one by one; otherwise a group lies inside a row (cols is a
// multiple of eight).
constexpr int kDropThreads = 256;
constexpr int kDropVec = 2;

template <typename T, bool RES, bool FLAT>
__global__ void __launch_bounds__(kDropThreads)
dropout_vec_kernel(const T* x, const T* res, T* y, const long long n, const int row_groups,
                   const long long ld_x, const long long ld_r, const long long ld_y, const __grid_constant__ Drop d) {
    chain_begin();
    const DropOffset o = drop_begin(d);
    const long long groups = n >> 3;
    const long long g0 = (long long)blockIdx.x * (kDropThreads * kDropVec) + threadIdx.x;
    Raw8<T> xv[kDropVec], rv[kDropVec];
    long long row[kDropVec];
    long long col[kDropVec];
#pragma unroll
    for (int i = 0; i < kDropVec; ++i) {
        const long long g = g0 + (long long)i * kDropThreads;
        if (g >= groups) break;
        if (FLAT) { row[i] = 0; col[i] = g * 8; }
        else { row[i] = g / row_groups; col[i] = (g - row[i] * row_groups) * 8; }
        xv[i] = load8<T, false>(x + row[i] * ld_x + col[i]);
        if (RES) rv[i] = load8<T, false>(res + row[i] * ld_r + col[i]);
    }
#pragma unroll
    for (int i = 0; i < kDropVec; ++i) {
        const long long g = g0 + (long long)i * kDropThreads;
        if (FLAT && g == groups) {
            const unsigned keep = drop_mask8(d, o, (unsigned long long)groups * 8);
            for (long long e = groups * 8; e < n; ++e) {
                float v = (keep >> (e & 7)) & 1u ? __fmul_rn(to_f32<T>(x[e]), d.up) : 0.0f;
                if (RES) v = __fadd_rn(to_f32<T>(res[e]), v);
                y[e] = from_f32<T>(v);
            }
        }
        if (g >= groups) break;
        float v[8], r[8];
        widen8<T>(xv[i], v);
        if (RES) widen8<T>(rv[i], r);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __fmul_rn(v[k], d.up);
        drop_block(d, o, (unsigned long long)g, v);                       // a dropped NaN is dropped
        if (RES) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __fadd_rn(r[k], v[k]);
        }
        store8<T>(y + row[i] * ld_y + col[i], v);
    }
}

// Any strides and alignment: one thread per group of eight logical elements, element by element.
template <typename T, bool RES>
__global__ void __launch_bounds__(kDropThreads)
dropout_any_kernel(const T* x, const T* res, T* y, const long long n, const long long cols,
                   const long long ld_x, const long long ld_r, const long long ld_y, const __grid_constant__ Drop d) {
    chain_begin();
    const DropOffset o = drop_begin(d);
    const long long g = (long long)blockIdx.x * kDropThreads + threadIdx.x;
    if (g * 8 >= n) return;
    const unsigned keep = drop_mask8(d, o, (unsigned long long)g * 8);
    long long row = g * 8 / cols, col = g * 8 - row * cols;
    for (int k = 0; k < 8 && g * 8 + k < n; ++k) {
        float v = (keep >> k) & 1u ? __fmul_rn(to_f32<T>(x[row * ld_x + col]), d.up) : 0.0f;
        if (RES) v = __fadd_rn(to_f32<T>(res[row * ld_r + col]), v);
        y[row * ld_y + col] = from_f32<T>(v);
        if (++col == cols) { col = 0; ++row; }
    }
}

template <typename T, bool RES>
static int launch_dropout(Device* d, int64_t rows, int64_t cols, uintptr_t x, int64_t ld_x, uintptr_t r, int64_t ld_r,
                          uintptr_t y, int64_t ld_y, const Drop& drop) {
    const T *px = (const T*)x, *pr = (const T*)r;
    T* py = (T*)y;
    const int64_t n = rows * cols;
    const int eb = (int)sizeof(T);
    const bool flat = rows == 1 || (ld_x == cols && ld_y == cols && (!RES || ld_r == cols));
    const bool aligned = x % 16 == 0 && y % 16 == 0 && (!RES || r % 16 == 0);
    const bool rowwise = cols % 8 == 0 && ld_x * eb % 16 == 0 && ld_y * eb % 16 == 0 && (!RES || ld_r * eb % 16 == 0);
    const bool vec = aligned && (flat || rowwise);
    const int64_t per_cta = kDropThreads * (vec ? kDropVec : 1);
    const int64_t grid = ((n + 7) / 8 + per_cta - 1) / per_cta;
    if (grid > 0x7fffffff) { set_error("%lld x %lld elements are too many", (long long)rows, (long long)cols); return GM_ERR_BAD_SIZE; }
    const dim3 g((unsigned)grid), t(kDropThreads);
    if (vec && flat) GM_CUDA_CHECK(launch_chained(dropout_vec_kernel<T, RES, true>, g, t, 0, d->stream, px, pr, py, n, 0, 0, 0, 0, drop));
    else if (vec) GM_CUDA_CHECK(launch_chained(dropout_vec_kernel<T, RES, false>, g, t, 0, d->stream, px, pr, py, n, (int)(cols / 8), ld_x, ld_r, ld_y, drop));
    else GM_CUDA_CHECK(launch_chained(dropout_any_kernel<T, RES>, g, t, 0, d->stream, px, pr, py, n, cols, ld_x, ld_r, ld_y, drop));
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
