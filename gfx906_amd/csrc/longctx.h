// What the kernels of the 4-bit cache (kv4_kernel.hip) and of sparse attention
// (sparse_kernel.hip) share: element types, matrix and lane operations on the
// device, error messages and checks on the host. Internal to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

namespace gfx906_amd {
namespace longctx {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
// Running max (log2 units) of a row that has seen no key: finite, so that a score
// of -inf weighs 0 and not exp2(-inf + inf), and below every score of a key.
constexpr float kNoMax = -3.0e38f;

#if defined(__HIP_DEVICE_COMPILE__)
template <class T>
struct Elem;
template <>
struct Elem<f16> {
    using x2 = f16x2;
    using x8 = f16x8;
    static __device__ __forceinline__ f32x4 mma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ x2 cvt2(float a, float b) {
        return __builtin_convertvector(f32x2{a, b}, x2);
    }
};
template <>
struct Elem<bf16> {
    using x2 = bf16x2;
    using x8 = bf16x8;
    static __device__ __forceinline__ f32x4 mma16(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ x2 cvt2(float a, float b) {
        return __builtin_convertvector(f32x2{a, b}, x2);
    }
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// Scale of an E8M0 byte in the form the cvt_scalef32 instructions take it: they
// use its exponent field, 0 for 2^-127 and 255 for NaN.
__device__ __forceinline__ float e8m0(unsigned byte) { return __uint_as_float(byte << 23); }
#endif

// Error message of the calling thread; `what` per file.
struct LastError {
    char text[256];
    int fail(const char* fmt, ...) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(text, sizeof text, fmt, ap);
        va_end(ap);
        return 1;
    }
    // 0, or 2 with a message, after the launches of a call.
    int launched(const char* what, hipError_t e) {
        if (e == hipSuccess) return 0;
        fail("%s: launch failed: %s", what, hipGetErrorString(e));
        return 2;
    }
    const char* get() const { return text[0] ? text : nullptr; }
};

// |scale| in log2 units, as the kernels multiply scores by it. Never 0, so that a masked score
// stays -inf and not NaN; the smallest fp32 number, as scores of bf16 rows reach 3e38: times it
// they are below 1e-6 and weigh alike. (Kernels are built with fp32 denormals.)
inline float log2_scale(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1.4e-45f); }
// Whether a scale is a number and finite in these units (a score of 0 would be NaN, else).
inline bool good_scale(float scale) { return scale == scale && log2_scale(scale) < INFINITY; }

// Whether HIP launches so many workgroups (fewer than 2^32 threads in x).
inline bool launchable(long long groups, int threads) { return groups < (1LL << 32) / threads; }

inline bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Whether rows of D elements at the strides s[0..n) over sizes e[0..n) lie apart:
// taken by growing stride, each stride reaches past the span of those below it.
// (Stricter than needed for interleaved layouts, which no tensor view here has.)
inline bool rows_apart(const long long* s, const long long* e, int n, int D) {
    bool used[4] = {};
    long long span = D;
    for (int k = 0; k < n; ++k) {
        int best = -1;
        for (int i = 0; i < n; ++i)
            if (!used[i] && (best < 0 || s[i] < s[best])) best = i;
        used[best] = true;
        if (e[best] <= 1) continue;
        if (s[best] < span) return false;
        span += (e[best] - 1) * s[best];
    }
    return true;
}

}  // namespace longctx
}  // namespace gfx906_amd
