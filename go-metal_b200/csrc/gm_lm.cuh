// gm_lm.cuh -- what the language-model operators share: element types, eight-element
// vectors, the counter-based generator of dropout, and argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "gm_internal.h"

namespace gm {

// ---- element types: arithmetic is in binary32, one rounding at the store ----
template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two neighbours of a 16-bit type in one 32-bit word (low half first).
template <typename T> __device__ __forceinline__ unsigned pack2(float lo, float hi);
template <> __device__ __forceinline__ unsigned pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }

// Eight elements as they lie in memory: one 16-byte word of a 16-bit type, two of fp32.
template <typename T> struct Raw8 { uint4 a; };
template <> struct Raw8<float> { uint4 a, b; };

// CACHED: the line may be wanted again soon (table rows of frequent tokens, partial sums);
// otherwise it is streamed.
template <typename T, bool CACHED> __device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
    const uint4* q = reinterpret_cast<const uint4*>(p);
    r.a = CACHED ? *q : __ldcs(q);
    if constexpr (sizeof(T) == 4) r.b = CACHED ? q[1] : __ldcs(q + 1);
    return r;
}

template <typename T> __device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const unsigned w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(w[k]);
    } else {
        const unsigned w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2<T>(w[k]);
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}

template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    uint4* q = reinterpret_cast<uint4*>(p);
    if constexpr (sizeof(T) == 4) {
        __stcs(q, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
        __stcs(q + 1, make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])));
    } else {
        __stcs(q, make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])));
    }
}

// Eight elements at any address, read as the 16-byte words that hold them (each word holds at least
// one of the eight, so nothing outside their 16-byte words is touched, and no page that holds none of
// them) and shifted into place when they are used; what else those words hold, which a neighbour may be writing,
// falls out there.  Matrices whose rows do not begin on 16-byte boundaries come this way: element
// by element the same traffic took 4 times as long.
template <typename T> struct Any8 {
    uint4 a, b, c;               // c: fp32 only
    unsigned off;                // bytes from a's begin to the first element
};

template <typename T> __device__ __forceinline__ Any8<T> load8_any(const T* p) {
    Any8<T> r;
    r.off = (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u);
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
    r.a = q[0];
    if (sizeof(T) == 4) {
        r.b = q[1];
        r.c = r.off ? q[2] : make_uint4(0u, 0u, 0u, 0u);
    } else {
        r.b = r.off ? q[1] : make_uint4(0u, 0u, 0u, 0u);
        r.c = make_uint4(0u, 0u, 0u, 0u);
    }
    return r;
}

template <typename T> __device__ __forceinline__ void widen8(const Any8<T>& r, float (&x)[8]) {
    unsigned w[12] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w, r.c.x, r.c.y, r.c.z, r.c.w};
    constexpr int N = sizeof(T) == 4 ? 8 : 4;                        // words of eight elements
    if (r.off & 8u) {
#pragma unroll
        for (int k = 0; k < N + 2; ++k) w[k] = w[k + 2];
    }
    if (r.off & 4u) {
#pragma unroll
        for (int k = 0; k < N + 1; ++k) w[k] = w[k + 1];
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(w[k]);
    } else {
        const unsigned bits = (r.off & 2u) * 8u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2<T>(__funnelshift_r(w[k], w[k + 1], bits));
            x[2 * k] = f.x;
            x[2 * k + 1] = f.y;
        }
    }
}

// Eight elements to any address, in 32-bit stores and two of 16 bits where they straddle.
template <typename T> __device__ __forceinline__ void store8_any(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = x[k];
    } else if ((reinterpret_cast<uintptr_t>(p) & 2u) == 0) {
        unsigned* q = reinterpret_cast<unsigned*>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
    } else {
        p[0] = from_f32<T>(x[0]);
        unsigned* q = reinterpret_cast<unsigned*>(p + 1);
#pragma unroll
        for (int k = 0; k < 3; ++k) q[k] = pack2<T>(x[2 * k + 1], x[2 * k + 2]);
        p[7] = from_f32<T>(x[7]);
    }
}

// Both kinds under one name: VEC says that the address is a multiple of 16 bytes.
template <typename T, bool VEC> struct Eight;
template <typename T> struct Eight<T, true> {
    Raw8<T> r;
    template <bool CACHED> __device__ __forceinline__ void load(const T* p) { r = load8<T, CACHED>(p); }
    static __device__ __forceinline__ void store(T* p, const float (&x)[8]) { store8<T>(p, x); }
};
template <typename T> struct Eight<T, false> {
    Any8<T> r;
    template <bool CACHED> __device__ __forceinline__ void load(const T* p) { r = load8_any<T>(p); }
    static __device__ __forceinline__ void store(T* p, const float (&x)[8]) { store8_any<T>(p, x); }
};

// ---- dropout's generator ----
// Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): counter {element / 8 (64 bits), offset (64 bits)}, key = seed.  The
// 128 bits of one answer serve eight elements, 16 bits each, so the generator costs a quarter
// of a multiply-pair per element and round; an element stays when its 16 bits, as a number,
// reach `cut` = round(p * 65536).  What stays is multiplied by 65536 / (65536 - cut), which
// makes the expectation exact for the probability that is really used, cut / 65536.
struct Drop {
    unsigned key[20];                    // the ten rounds' keys: the seed, and after each round the Weyl constants on top
    unsigned o0, o1;                     // offset
    const unsigned long long* more;      // null, or a device word that is added to the offset
    unsigned cut;                        // 0: everything stays, no generator
    float up;
};

// The offset this launch uses.
struct DropOffset { unsigned o0, o1; };
__device__ __forceinline__ DropOffset drop_begin(const Drop& d) {
    if (d.cut == 0u || d.more == nullptr) return {d.o0, d.o1};
    const unsigned long long o = (((unsigned long long)d.o1 << 32) | d.o0) + *d.more;
    return {(unsigned)o, (unsigned)(o >> 32)};
}

// The 128 bits of one block, elements 2k and 2k + 1 in the low and high half of word k.
__device__ __forceinline__ void drop_words(const Drop& d, const DropOffset& o, const unsigned long long block, unsigned (&w)[4]) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = o.o0, c3 = o.o1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)0xD2511F53u * c0, b = (unsigned long long)0xCD9E8D57u * c2;
        c0 = (unsigned)(b >> 32) ^ c1 ^ d.key[2 * r];
        c1 = (unsigned)b;
        c2 = (unsigned)(a >> 32) ^ c3 ^ d.key[2 * r + 1];
        c3 = (unsigned)a;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// Zeroes the dropped ones of a whole block of eight elements.  A half reaches the cut when the
// word that has it on top reaches the cut shifted up: two compares and one shift per word.
__device__ __forceinline__ void drop_block(const Drop& d, const DropOffset& o, const unsigned long long block, float (&x)[8]) {
    if (d.cut == 0u) return;
    if (d.cut > 0xffffu) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = 0.0f;
        return;
    }
    unsigned w[4];
    drop_words(d, o, block, w);
    const unsigned top = d.cut << 16;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        x[2 * k] = (w[k] << 16) >= top ? x[2 * k] : 0.0f;
        x[2 * k + 1] = w[k] >= top ? x[2 * k + 1] : 0.0f;
    }
}

// Bit k: element 8 * block + k stays.
__device__ __forceinline__ unsigned drop_bits(const Drop& d, const DropOffset& o, const unsigned long long block) {
    unsigned w[4];
    drop_words(d, o, block, w);
    unsigned keep = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        keep |= ((w[k] & 0xffffu) >= d.cut ? 1u : 0u) << (2 * k);
        keep |= ((w[k] >> 16) >= d.cut ? 1u : 0u) << (2 * k + 1);
    }
    return keep;
}

// Bit k: element first + k stays, for eight elements that may begin inside a block.
__device__ __forceinline__ unsigned drop_mask8(const Drop& d, const DropOffset& o, const unsigned long long first) {
    if (d.cut == 0u) return 0xffu;
    unsigned keep = drop_bits(d, o, first >> 3);
    const unsigned skip = (unsigned)first & 7u;
    if (skip != 0u) keep = (keep | (drop_bits(d, o, (first >> 3) + 1) << 8)) >> skip;
    return keep & 0xffu;
}

// Zeroes the dropped ones of eight elements from `first` on; WHOLE: they are a block.
template <bool WHOLE>
__device__ __forceinline__ void drop8(const Drop& d, const DropOffset& o, const unsigned long long first, float (&x)[8]) {
    if (WHOLE) {
        drop_block(d, o, first >> 3, x);
    } else {
        const unsigned keep = drop_mask8(d, o, first);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = (keep >> k) & 1u ? x[k] : 0.0f;
    }
}

__device__ __forceinline__ void chain_begin() {
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
}

// ---- host side ----
inline int dtype_bytes(int dtype) { return dtype == GM_F32 ? 4 : dtype == GM_F16 || dtype == GM_BF16 ? 2 : 0; }

// Fills the kernel's form of a dropout argument (null: none).  Returns GM_OK or a code.
int make_drop(const Device* d, const gm_dropout_t* in, Drop* out);

// A buffer of at least `need` bytes on this device, aligned to `align`; need 0 checks the rest.
int check_buffer(const Device* d, uintptr_t p, int64_t need, int64_t align, const char* what);

// Rows and row stride below 2^31, at most 2^30 columns (column arithmetic is in 32 bits), a stride
// that covers the columns, and at most 2^60 elements, so that no count of bytes passes 64 bits (a wrapped
// one would let a small buffer pass for large enough).
int check_matrix(int64_t rows, int64_t cols, int64_t ld, const char* what);

// Bytes from a matrix's first element to behind its last one.
inline int64_t matrix_bytes(int64_t rows, int64_t cols, int64_t ld, int eb) { return rows > 0 ? ((rows - 1) * ld + cols) * eb : 0; }

// A launch that may begin while the kernel before it in the stream ends (programmatic stream
// serialization).  The kernel calls chain_begin() before it touches memory: it waits for the kernel
// before, and lets the one behind start its own wait.
template <typename... P, typename... A>
inline cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

#define GM_TRY(expr)                      \
    do {                                  \
        const int rc__ = (expr);          \
        if (rc__ != GM_OK) return rc__;   \
    } while (0)

}  // namespace gm
