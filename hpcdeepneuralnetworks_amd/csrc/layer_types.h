// Element types of the layer operators (FP32, FP16, BF16): 16-byte vectors, conversions to and from FP32.
#pragma once

#include "common.h"

namespace hpcdnn {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef unsigned v4u __attribute__((ext_vector_type(4)));

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
// One float through a descriptor.
__device__ __forceinline__ float buffer_load_f(__amdgpu_buffer_rsrc_t rs, int byte_offset) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, byte_offset, 0, 0));
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

// Vector at column `col` of a row of `cols` columns: whole, cut at the end of the row, or zeros behind it.
template <class T>
__device__ __forceinline__ v4u load_row(const T* row, int col, int cols) {
    if (col + kVec<T> <= cols) return load16(row + col);
    if (col < cols) return load_part(row + col, cols - col);
    return v4u{0u, 0u, 0u, 0u};
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

// A row of `cols` values (0: no row at all) as a buffer descriptor, wave-uniform.  Loads give zeros behind the end and
// stores there are dropped, without a branch.  That is worth more than the instructions it saves: loads and stores share one
// in-order counter, and behind a store in a branch the wait for an older load has to be one for every store as well.
// 16 bytes at a time need a row on a 4-byte address that holds whole dwords (the range check is per dword).
template <class T, bool kDwords>
struct row_buffer {
    __amdgpu_buffer_rsrc_t rs;
    int skew;  // bytes by which the row starts behind a 4-byte address (rows that are read by single values)
    __device__ __forceinline__ row_buffer(const T* row, int cols) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row);
        skew = kDwords ? 0 : static_cast<int>(at & 2);
        const int64_t bytes = static_cast<int64_t>(cols) * static_cast<int64_t>(sizeof(T));
        rs = make_rsrc(reinterpret_cast<const float*>(at - skew), kDwords ? bytes : cols > 0 ? bytes + skew : 0);
    }
    __device__ __forceinline__ v4u load16(int col) const {
        return __builtin_amdgcn_raw_buffer_load_b128(rs, col * static_cast<int>(sizeof(T)), 0, 0);
    }
    __device__ __forceinline__ void store16(int col, v4u v) const {
        __builtin_amdgcn_raw_buffer_store_b128(v, rs, col * static_cast<int>(sizeof(T)), 0, 0);
    }
    // non-temporal: a large result that nothing on the way reads again
    __device__ __forceinline__ void store16_once(int col, v4u v) const {
        __builtin_amdgcn_raw_buffer_store_b128(v, rs, col * static_cast<int>(sizeof(T)), 0, 2);
    }
    __device__ __forceinline__ T load1(int col) const {
        return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rs, col * 2 + skew, 0, 0));
    }
    __device__ __forceinline__ void store1(int col, T v) const {
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rs, col * 2 + skew, 0, 0);
    }
};

// How the threads that share a row hold its values, NV vectors of kVec each.
//  kDwordRows   rows on 4-byte addresses that hold whole dwords: vector v of thread t is columns (v n + t) kVec ..., through a
//               descriptor that ends it.
//  kOverlapRows any other row of at least kVec values (16-bit rows of odd length, or at odd addresses): the same vectors from
//               any address, and those that would pass the end of the row are moved back to end with it.  What such a vector
//               shares with its neighbour is not its own: left out of every sum, and stored twice with the same value.  So
//               there is no branch here either.
//  kSingleRows  shorter ones, value by value through the descriptor.
enum row_kind { kDwordRows, kOverlapRows, kSingleRows };

template <class T, int NV, row_kind kKind>
struct row_values {
    static_assert(kKind == kDwordRows || sizeof(T) == 2, "FP32 rows are whole dwords");
    int t, n, cols;
    v4u u[kKind == kSingleRows ? 1 : NV];
    T single[kKind == kSingleRows ? NV * kVec<T> : 1];
    __device__ __forceinline__ row_values(int thread, int threads, int columns) : t(thread), n(threads), cols(columns) {}
    __device__ __forceinline__ int first_own(int v) const { return (v * n + t) * kVec<T>; }
    __device__ __forceinline__ int column(int v, int i) const {
        if constexpr (kKind == kSingleRows) return (v * kVec<T> + i) * n + t;
        else if constexpr (kKind == kOverlapRows) return min(first_own(v), cols - kVec<T>) + i;
        else return first_own(v) + i;
    }
    __device__ __forceinline__ bool own(int v, int i) const {
        return kKind == kOverlapRows ? column(v, i) >= first_own(v) : column(v, i) < cols;
    }
    // Row `row` of the matrix at m.  Behind its last row: zeros (kOverlapRows: the last row).
    __device__ __forceinline__ void load(const T* m, int64_t ld, int64_t row, int64_t rows) {
        const bool is = row < rows;
        if constexpr (kKind == kOverlapRows) {
            const T* r = m + (is ? row : rows - 1) * ld;
#pragma unroll
            for (int v = 0; v < NV; ++v) u[v] = load16(r + column(v, 0));
        } else {
            const row_buffer<T, kKind == kDwordRows> b(m + (is ? row : 0) * ld, is ? cols : 0);
            if constexpr (kKind == kDwordRows) {
#pragma unroll
                for (int v = 0; v < NV; ++v) u[v] = b.load16(column(v, 0));
            } else {
#pragma unroll
                for (int k = 0; k < NV * kVec<T>; ++k) single[k] = b.load1(k * n + t);
            }
        }
    }
    __device__ __forceinline__ void clear() {
        if constexpr (kKind == kSingleRows) {
#pragma unroll
            for (int k = 0; k < NV * kVec<T>; ++k) single[k] = static_cast<T>(0.f);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) u[v] = v4u{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void get(float (&f)[NV][kVec<T>]) const {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if constexpr (kKind == kSingleRows) {
#pragma unroll
                for (int i = 0; i < kVec<T>; ++i) f[v][i] = static_cast<float>(single[v * kVec<T> + i]);
            } else {
                unpack<T>(u[v], f[v]);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[NV][kVec<T>]) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if constexpr (kKind == kSingleRows) {
#pragma unroll
                for (int i = 0; i < kVec<T>; ++i) single[v * kVec<T> + i] = static_cast<T>(f[v][i]);
            } else {
                u[v] = pack<T>(f[v]);
            }
        }
    }
    // Behind the last row: dropped (kOverlapRows: to the last row, whose values they are).
    __device__ __forceinline__ void store(T* m, int64_t ld, int64_t row, int64_t rows) const {
        const bool is = row < rows;
        if constexpr (kKind == kOverlapRows) {
            T* r = m + (is ? row : rows - 1) * ld;
#pragma unroll
            for (int v = 0; v < NV; ++v) __builtin_nontemporal_store(u[v], reinterpret_cast<v4u_any*>(r + column(v, 0)));
        } else {
            const row_buffer<T, kKind == kDwordRows> b(m + (is ? row : 0) * ld, is ? cols : 0);
            if constexpr (kKind == kDwordRows) {
#pragma unroll
                for (int v = 0; v < NV; ++v) b.store16_once(column(v, 0), u[v]);
            } else {
#pragma unroll
                for (int k = 0; k < NV * kVec<T>; ++k) b.store1(k * n + t, single[k]);
            }
        }
    }
};

// Host: whether rows of this matrix are whole dwords, and the kind of a call all of whose matrices are (or are not).
inline bool rows_are_dwords(const void* p, int64_t ld, int cols, size_t elem) {
    return reinterpret_cast<uintptr_t>(p) % 4 == 0 && (ld * static_cast<int64_t>(elem)) % 4 == 0 && (cols * elem) % 4 == 0;
}
inline row_kind kind_of(bool all_dwords, int cols) { return all_dwords ? kDwordRows : cols >= kVec<f16> ? kOverlapRows : kSingleRows; }

// Put behind loads whose values are for the next turn of a loop: memory might have changed, as far as the compiler knows, so
// it cannot move them (as it does with plain loads) to where that turn uses them, and they stay in flight over this one.
__device__ __forceinline__ void loads_start_here() { asm volatile("" ::: "memory"); }

// Sum over the wave, in every lane (a scalar register: the value is read from lane 63).
__device__ __forceinline__ float wave_allsum(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_lane63(v)), 63));
}

// The value of the first lane, for one that is the same in all: a scalar register.
__device__ __forceinline__ float wave_first(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
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
