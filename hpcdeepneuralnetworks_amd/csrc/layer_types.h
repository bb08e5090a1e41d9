// Element types of the layer operators (FP32, FP16, BF16): 16-byte vectors, conversions to and from FP32.
#pragma once

#include "common.h"

namespace hpcdnn {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));

// Values of T in 16 bytes: what one lane loads or stores at a time.
template <class T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));

// Four words at any address that a value of two bytes may have.
typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes from an address that is aligned to T only (rows of odd length start anywhere): one global_load_dwordx4 all the
// same, global memory instructions take any alignment on this target.
template <class T>
__device__ __forceinline__ v4u load16(const T* p) {
    return *reinterpret_cast<const v4u_any*>(p);
}
template <class T>
__device__ __forceinline__ void store16(T* p, v4u v) {
    *reinterpret_cast<v4u_any*>(p) = v;
}

// The first `n` values of such a vector, 0 < n < kVec<T>; zeros behind them.
template <class T>
__device__ __forceinline__ v4u load_part(const T* p, int n) {
    union {
        T t[kVec<T>];
        v4u u;
    } r;
    r.u = v4u{0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kVec<T> - 1; ++i)
        if (i < n) r.t[i] = p[i];
    return r.u;
}
template <class T>
__device__ __forceinline__ void store_part(T* p, v4u v, int n) {
    union {
        v4u u;
        T t[kVec<T>];
    } r;
    r.u = v;
#pragma unroll
    for (int i = 0; i < kVec<T> - 1; ++i)
        if (i < n) p[i] = r.t[i];
}

// Vector at column `col` of a row of `cols` columns: whole, cut at the end of the row, or zeros behind it.
template <class T>
__device__ __forceinline__ v4u load_row(const T* row, int col, int cols) {
    if (col + kVec<T> <= cols) return load16(row + col);
    if (col < cols) return load_part(row + col, cols - col);
    return v4u{0u, 0u, 0u, 0u};
}
template <class T>
__device__ __forceinline__ void store_row(T* row, int col, int cols, v4u v) {
    if (col + kVec<T> <= cols) store16(row + col, v);
    else if (col < cols) store_part(row + col, v, cols - col);
}

template <class T>
__device__ __forceinline__ void unpack(v4u u, float (&f)[kVec<T>]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, static_cast<unsigned>(u[i]));  // the cast makes a value of the element
    } else if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_bit_cast(float, u[i] << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, u[i] & 0xffff0000u);
        }
    } else {
        typedef f16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v2h h = __builtin_bit_cast(v2h, static_cast<unsigned>(u[i]));
            f[2 * i] = static_cast<float>(h.x);
            f[2 * i + 1] = static_cast<float>(h.y);
        }
    }
}

// Round to nearest, ties to even, once per value.
template <class T>
__device__ __forceinline__ v4u pack(const float (&f)[kVec<T>]) {
    v4u u;
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(unsigned, f[i]);
    } else {
        typedef T v2t __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v2t h = {static_cast<T>(f[2 * i]), static_cast<T>(f[2 * i + 1])};
            u[i] = __builtin_bit_cast(unsigned, h);
        }
    }
    return u;
}

// Sum over the wave, in every lane (a scalar register: the value is read from lane 63).
__device__ __forceinline__ float wave_allsum(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_lane63(v)), 63));
}

inline size_t type_bytes(int type) { return type == HPCDNN_F32 ? 4 : 2; }
inline bool type_valid(int type) { return type == HPCDNN_F32 || type == HPCDNN_F16 || type == HPCDNN_BF16; }
// Pointers are aligned to their element.
inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Calls f with a null pointer of the C++ type that `type` names.
template <class F>
auto with_type(int type, F&& f) {
    switch (type) {
        case HPCDNN_F16: return f(static_cast<f16*>(nullptr));
        case HPCDNN_BF16: return f(static_cast<bf16*>(nullptr));
        default: return f(static_cast<float*>(nullptr));
    }
}

}  // namespace hpcdnn
