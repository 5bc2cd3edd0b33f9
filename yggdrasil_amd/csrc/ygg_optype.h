// The operators' three element types: conversions, and loads and stores of 16 bytes at any element's address.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ygg {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct bf16_t { uint16_t bits; };
struct f16_t { _Float16 v; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __builtin_bit_cast(float, (uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v.v; }

// rounded to nearest, ties to even
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
    return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)};
}
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) { return f16_t{(_Float16)v}; }

// 16 bytes from an address of T's alignment
template <class T> __device__ __forceinline__ u32x4 load16(const T *p) {
    typedef uint32_t any __attribute__((ext_vector_type(4), aligned(1)));
    return *(const any *)p;
}
// of which the first n elements exist; the others come as zero
template <class T> __device__ __forceinline__ u32x4 load16(const T *p, int n) {
    constexpr int kE = 16 / sizeof(T);
    if (n >= kE) return load16(p);
    u32x4 v = {0, 0, 0, 0};
    if (n <= 0) return v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 3; j++)
            if (j < n) v[j] = ((const uint32_t *)p)[j];
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 7; j++)
            if (j < n) v[j / 2] |= (uint32_t)((const uint16_t *)p)[j] << 16 * (j % 2);
    } else {
#pragma unroll
        for (int j = 0; j < 15; j++)
            if (j < n) v[j / 4] |= (uint32_t)((const uint8_t *)p)[j] << 8 * (j % 4);
    }
    return v;
}

// The same without a branch, so that loads that follow are not held up, for rows of 16 bytes or more: p is n elements (any
// number, also none or less) before its row's end. The row's last 16 bytes are loaded where fewer are left, and moved down.
template <class T> __device__ __forceinline__ u32x4 load16_end(const T *p, int n) {
    constexpr int kE = 16 / sizeof(T);
    const u32x4 v = load16(p + min(n - kE, 0));
    const int bits = max(kE - n, 0) * 8 * (int)sizeof(T);
    const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    uint64_t a = bits < 64 ? lo >> (bits & 63) | (hi << 1) << (~bits & 63) : hi >> (bits & 63), b = bits < 64 ? hi >> (bits & 63) : 0;
    if (bits >= 128) a = 0;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
}
// the values of 16 bytes
__device__ __forceinline__ void unpack(u32x4 v, float *f, float) {
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = __builtin_bit_cast(float, (uint32_t)v[j]);
}
__device__ __forceinline__ void unpack(u32x4 v, float *f, bf16_t) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[2 * j] = __builtin_bit_cast(float, v[j] << 16);
        f[2 * j + 1] = __builtin_bit_cast(float, v[j] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(u32x4 v, float *f, f16_t) {
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[j / 2] >> 16 * (j % 2)));
}

// kN consecutive values rounded to T at an address of T's alignment, of which the first `left` exist
template <class T, int kN, class V> __device__ __forceinline__ void store_run(T *p, const V *v, int left) {
    constexpr int kE = kN * sizeof(T) < 16 ? kN : 16 / sizeof(T);
    typedef uint32_t any __attribute__((ext_vector_type(kE * sizeof(T) / 4), aligned(1)));
    if (left >= kN) {
#pragma unroll
        for (int k = 0; k < kN; k += kE) {
            T t[kE];
#pragma unroll
            for (int j = 0; j < kE; j++) t[j] = from_f32<T>(v[k + j]);
            any a;
            __builtin_memcpy(&a, t, sizeof(a));
            *(any *)(p + k) = a;
        }
    } else {
#pragma unroll
        for (int k = 0; k < kN; k++)
            if (k < left) p[k] = from_f32<T>(v[k]);
    }
}

}  // namespace ygg
