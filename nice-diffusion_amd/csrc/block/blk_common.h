// Shared helpers of libnd_block.so, the transformer-block operators (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "nd_block.h"

namespace ndb {

void set_error(const char* fmt, ...);

inline int fail_arg(const char* fn, const char* what) {
    set_error("%s: %s", fn, what);
    return ND_E_ARG;
}

inline int check_launch(const char* fn) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("%s: launch failed: %s", fn, hipGetErrorString(e));
        return ND_E_LAUNCH;
    }
    return ND_OK;
}

// Raise a kernel's dynamic-LDS limit to the CU's 160 KiB, once per (kernel, device): `flags` is one static array per kernel
// instantiation.  Two threads that race here both set the same attribute.
constexpr int kMaxDevices = 64;
inline int ensure_max_lds(const void* kern, bool (&flags)[kMaxDevices], const char* fn) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) dev = kMaxDevices - 1;
    if (flags[dev] && dev != kMaxDevices - 1) return ND_OK;
    hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) {
        set_error("%s: hipFuncSetAttribute: %s", fn, hipGetErrorString(e));
        return ND_E_LAUNCH;
    }
    flags[dev] = true;
    return ND_OK;
}

#define NDB_REQUIRE(cond, fn, msg)                  \
    do {                                            \
        if (!(cond)) return ndb::fail_arg(fn, msg); \
    } while (0)

// a launch counts its threads in 32 bits
inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads < (1LL << 32); }

inline bool aligned_to(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// N consecutive elements as one vector access (the caller guarantees N * sizeof(T) alignment, at most 16 bytes each)
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
    constexpr int BYTES = N * (int)sizeof(T);
    constexpr int STEP = BYTES > 16 ? 16 / (int)sizeof(T) : N;
    typedef T vec __attribute__((ext_vector_type(STEP)));
#pragma unroll
    for (int i = 0; i < N; i += STEP) {
        if constexpr (STEP == 1) {
            v[i] = (float)p[i];
        } else {
            const vec t = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
            for (int j = 0; j < STEP; ++j) v[i + j] = (float)t[j];
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
    constexpr int BYTES = N * (int)sizeof(T);
    constexpr int STEP = BYTES > 16 ? 16 / (int)sizeof(T) : N;
    typedef T vec __attribute__((ext_vector_type(STEP)));
#pragma unroll
    for (int i = 0; i < N; i += STEP) {
        if constexpr (STEP == 1) {
            p[i] = (T)v[i];
        } else {
            vec t;
#pragma unroll
            for (int j = 0; j < STEP; ++j) t[j] = (T)v[i + j];
            *reinterpret_cast<vec*>(p + i) = t;
        }
    }
}

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// c += a b over one 16-byte piece a lane of either operand: 16 k in bf16 (lane half lh holds k = 8 lh + 0 .. 7), 8 k in fp32
// (4 lh + 0 .. 3; instruction j takes one k of either half)
template <typename T>
__device__ __forceinline__ f32x16 mma_step(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (sizeof(T) == 2) {
        union { u32x4 u; bf16x8 h; } x, y;
        x.u = a, y.u = b;
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.h, y.h, c, 0, 0, 0);
    } else {
        union { u32x4 u; float f[4]; } x, y;
        x.u = a, y.u = b;
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.f[j], y.f[j], c, 0, 0, 0);
        return c;
    }
}

}  // namespace ndb
