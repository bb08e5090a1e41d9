// Products of a few tokens with a matrix of 4-bit weights, y[t][m] = alpha * sum_n W[m][n] x[t][n] + beta * y[t][m], where
// W[m][n] = (q[m][n] - z[m][n / group]) * s[m][n / group]; and the packing of such a matrix on the host.
//
// Bound by the stream of weights: half a byte each, read once, against 2 operations per token.  The weights of a row are
// therefore read 16 bytes (32 columns, never more than one group) per lane, and everything else is kept cheap:
//  - a nibble becomes a 16-bit float in one step, by placing it in the mantissa of 16.0: 16 + q is exact in FP16 and in
//    BF16, and two of them (columns c and c + 4 of eight) are made by one shift and one and-or.  The products are summed
//    in FP32 by two-term dot instructions; the offset is taken out per 32 columns, with the group's zero point,
//      sum (q - z) x = sum (16 + q) x - (16 + z) sum x,
//    and only then scaled.  The smallest power of two whose mantissa takes a nibble in both types keeps what cancels there
//    within a factor of about five of the result.  FP32 tokens use byte-to-float conversions and q itself.
//  - x lies in LDS in the order in which the lanes need it, its sums over 32 columns beside it.
#include <algorithm>
#include <cmath>

#include "layer_types.h"
#ifndef W4MIN
#define W4MIN 5
#endif
#ifndef W4TW
#define W4TW kW4TileWaves
#endif
#ifndef W4BPC
#define W4BPC 1
#endif
#ifndef W4ROWS
#define W4ROWS
#endif
#ifndef W4RT
#define W4RT 1
#endif

namespace hpcdnn {

constexpr int kW4Cols = 32;                      // columns of one lane and load
constexpr int kW4Piece = kW4Cols * kWave;        // columns of a wave and load
constexpr int kW4MaxWaves = 16;                  // waves of a workgroup
constexpr int kW4LdsBytes = 65536;

template <class T>
constexpr int kW4Parts = kW4Cols / kVec<T>;      // 16-byte parts of a lane's x

// 16-bit pairs for the dot instruction: dword p = columns (p, p + 4) of eight.
__device__ __forceinline__ v4u pair_order(v4u d) {
    return v4u{__builtin_amdgcn_perm(d[2], d[0], 0x05040100u), __builtin_amdgcn_perm(d[2], d[0], 0x07060302u),
               __builtin_amdgcn_perm(d[3], d[1], 0x05040100u), __builtin_amdgcn_perm(d[3], d[1], 0x07060302u)};
}

// The eight nibbles of w as 16 + q in T, columns (p, p + 4) in dword p.
template <class T>
__device__ __forceinline__ v4u nibbles_plus_16(unsigned w) {
    if constexpr (std::is_same_v<T, f16>) {      // 16.0 = 0x4C00, q in bits 6 .. 9 of the mantissa
        constexpr unsigned mask = 0x03C003C0u, one = 0x4C004C00u;
        return v4u{((w << 6) & mask) | one, ((w << 2) & mask) | one, ((w >> 2) & mask) | one, ((w >> 6) & mask) | one};
    } else {                                     // 16.0 = 0x4180, q in bits 3 .. 6
        constexpr unsigned mask = 0x00780078u, one = 0x41804180u;
        return v4u{((w << 3) & mask) | one, ((w >> 1) & mask) | one, ((w >> 5) & mask) | one, ((w >> 9) & mask) | one};
    }
}

template <class T>
__device__ __forceinline__ float dot2(unsigned a, unsigned b, float c) {
    typedef T v2t __attribute__((ext_vector_type(2)));
    if constexpr (std::is_same_v<T, f16>) return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2t, a), __builtin_bit_cast(v2t, b), c, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2t, a), __builtin_bit_cast(v2t, b), c, false);
}

// x of one panel of columns into LDS: part i of the 32 columns of lane l and piece p of token t at
// ((t * pieces + p) * parts + i) * 1024 + l * 16 bytes, so a wave reads a part without bank conflicts; sums of 32 behind.
template <class T, int TB>
__device__ __forceinline__ void stage_x(char* lds, float* sums, int pieces, const T* __restrict__ x, int64_t ldx, int tokens, int n0, int N) {
    const int chunks = pieces * kWave;
    for (int i = threadIdx.x; i < TB * chunks; i += blockDim.x) {
        const int t = i / chunks, c = i - t * chunks;
        const int col = n0 + c * kW4Cols;
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < kW4Parts<T>; ++p) {
            v4u v = {0u, 0u, 0u, 0u};
            if (t < tokens) v = load_row(x + t * ldx, col + p * kVec<T>, N);
            float f[kVec<T>];
            unpack<T>(v, f);
#pragma unroll
            for (int k = 0; k < kVec<T>; ++k) sum += f[k];
            if constexpr (sizeof(T) == 2) v = pair_order(v);
            *reinterpret_cast<v4u*>(lds + (((t * pieces + c / kWave) * kW4Parts<T> + p) * kWave + c % kWave) * 16) = v;
        }
        sums[i] = sum;
    }
}

// A wave takes kRows rows at a time through all columns, kPieces pieces of 2048 columns to a step; TB tokens at a time
// (blockIdx.y counts groups of them).  While one step is computed the next one's weights, scales and zero points are on
// their way, also into the next rows and panel; the first are requested before x is staged.  kRows * kPieces = 4 keeps 4 KiB
// per wave in flight whatever the shape: sixteen waves of a CU then cover the 50 KiB that the memory's latency asks for.
template <class T, int TB, int kRows, int kPieces, bool kZeros>
__global__ __launch_bounds__(kW4MaxWaves * kWave) void w4_gemv_kernel(int batch, int M, int N, int group_shift, float alpha,
                                                                      const unsigned char* __restrict__ q, int64_t ldq,
                                                                      const T* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                                                      int64_t ldg, const T* __restrict__ x, int64_t ldx, float beta,
                                                                      T* __restrict__ y, int64_t ldy, int rows_per_block, int panel) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int stride = blockDim.x / kWave * kRows;  // rows that the workgroup takes at a time
    const int pieces = panel / kW4Piece;
    float* sums = reinterpret_cast<float*>(lds + static_cast<size_t>(TB) * panel * sizeof(T));
    const int t0 = blockIdx.y * TB, tokens = min(TB, batch - t0);
    x += t0 * ldx;
    y += t0 * ldy;
    const int row_bytes = ((N + 1) / 2 + 3) & ~3;  // whole dwords: the last may hold bytes behind the row, whose x is zero
    const int first = blockIdx.x * rows_per_block, last = min(M, first + rows_per_block);

    // rows r0 ... of the workgroup, columns from n0 + p0 * 2048 on
    v4u w[kRows][kPieces];
    T s[kRows][kPieces];
    unsigned char z[kRows][kPieces];
    auto load = [&](int r0, int n0, int p0) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int m = r0 + wave * kRows + r;
            const bool is = m < last;
            const int64_t at = is ? m : first;
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const float*>(q + at * ldq), is ? row_bytes : 0);
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
                const int col = n0 + (p0 + u) * kW4Piece + lane * kW4Cols;
                w[r][u] = __builtin_amdgcn_raw_buffer_load_b128(rs, col / 2, 0, 0);
                const int64_t g = at * ldg + (min(col, N - 1) >> group_shift);  // behind the last column: x is zero
                s[r][u] = scales[g];
                if (kZeros) z[r][u] = zeros[g];
            }
        }
    };
    if (first < last && N > 0) load(first, 0, 0);
    bool staged = false;
    for (int r0 = first; r0 < last; r0 += stride) {
        float acc[kRows][TB];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) acc[r][t] = 0.f;
        for (int n0 = 0; n0 < N; n0 += panel) {
            if (!staged || panel < N) {
                __syncthreads();
                stage_x<T, TB>(lds, sums, pieces, x, ldx, tokens, n0, N);
                __syncthreads();
                staged = true;
            }
            for (int p0 = 0; p0 < pieces; p0 += kPieces) {
                v4u now[kRows][kPieces];
                float scale[kRows][kPieces], offset[kRows][kPieces];
                constexpr float kOffset = sizeof(T) == 2 ? 16.f : 0.f;
#pragma unroll
                for (int r = 0; r < kRows; ++r)
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) {
                        now[r][u] = w[r][u];
                        scale[r][u] = static_cast<float>(s[r][u]);
                        offset[r][u] = kOffset + (kZeros ? static_cast<float>(z[r][u]) : 8.f);
                    }
                const bool panel_end = p0 + kPieces >= pieces, row_end = panel_end && n0 + panel >= N;
                load(row_end ? r0 + stride : r0, !panel_end ? n0 : row_end ? 0 : n0 + panel, panel_end ? 0 : p0 + kPieces);
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    if (p0 + u >= pieces) break;
                    float dot[kRows][TB];
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
#pragma unroll
                        for (int t = 0; t < TB; ++t) dot[r][t] = 0.f;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {  // eight columns
                        if constexpr (sizeof(T) == 2) {
                            v4u xv[TB];
#pragma unroll
                            for (int t = 0; t < TB; ++t)
                                xv[t] = *reinterpret_cast<const v4u*>(lds + (((t * pieces + p0 + u) * kW4Parts<T> + d) * kWave + lane) * 16);
#pragma unroll
                            for (int r = 0; r < kRows; ++r) {
                                const v4u wq = nibbles_plus_16<T>(now[r][u][d]);
#pragma unroll
                                for (int t = 0; t < TB; ++t)
#pragma unroll
                                    for (int k = 0; k < 4; ++k) dot[r][t] = dot2<T>(wq[k], xv[t][k], dot[r][t]);
                            }
                        } else {
                            v4f xv[TB][2];
#pragma unroll
                            for (int t = 0; t < TB; ++t)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    xv[t][h] = *reinterpret_cast<const v4f*>(lds + (((t * pieces + p0 + u) * kW4Parts<T> + 2 * d + h) * kWave + lane) * 16);
#pragma unroll
                            for (int r = 0; r < kRows; ++r) {
                                const unsigned even = now[r][u][d] & 0x0f0f0f0fu, odd = (now[r][u][d] >> 4) & 0x0f0f0f0fu;
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float wk = static_cast<float>((((k & 1) ? odd : even) >> (8 * (k / 2))) & 0xffu);
#pragma unroll
                                    for (int t = 0; t < TB; ++t) dot[r][t] = __builtin_fmaf(wk, xv[t][k / 4][k & 3], dot[r][t]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int t = 0; t < TB; ++t) {
                        const float sx = sums[(t * pieces + p0 + u) * kWave + lane];
#pragma unroll
                        for (int r = 0; r < kRows; ++r)
                            acc[r][t] = __builtin_fmaf(scale[r][u], __builtin_fmaf(-offset[r][u], sx, dot[r][t]), acc[r][t]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const int m = r0 + wave * kRows + r;
                const float v = alpha * wave_allsum(acc[r][t]);
                if (lane == r * TB + t && m < last && t < tokens) {
                    T* dst = y + t * ldy + m;
                    *dst = static_cast<T>(beta == 0.f ? v : __builtin_fmaf(beta, static_cast<float>(*dst), v));
                }
            }
    }
}

// ---- matrix-core form -------------------------------------------------------
// For more tokens the products go to the matrix cores: a 16 x 16 tile of y (16 tokens by 16 rows of W) takes 32 columns per
// instruction, and the nibbles cost the same few instructions for one token or sixteen.  A workgroup has kRowTiles tiles of
// rows by kTokTiles of tokens; its waves split the columns between them, in runs of units of 128, and their sums meet in
// LDS at the end (in wave order): so a narrow matrix still keeps every CU loading.
//
// Lane l reads 16 bytes (32 columns) of row l % 16 from quarter l / 16 of the unit.  An instruction sums over the four
// quarters of the lanes, so the dwords are first exchanged between the quarters (a 4 x 4 transposition in four lane swaps):
// dword d of the lanes is then columns 32 d + 8 (l / 16) ... of the unit, and every instruction stays inside one group.
// The sums over x that take out the offset of the nibbles come from the same instruction with a matrix of ones.
constexpr int kW4Unit = 128;
constexpr int kW4TileWaves = 16;

typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef bf16 v8b __attribute__((ext_vector_type(8)));

template <class T>
__device__ __forceinline__ v4f mfma_16x16x32(v4u a, v4u b, v4f c) {
    if constexpr (std::is_same_v<T, f16>)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// dword d of quarter j  <->  dword j of quarter d
__device__ __forceinline__ v4u transpose_quarters(v4u w) {
    const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return v4u{c[0], c[1], d[0], d[1]};
}

template <class T, int kRowTiles, int kTokTiles, int kGroupSteps, bool kZeros>
__global__ __launch_bounds__(W4TW * kWave) void w4_tile_kernel(int batch, int M, int N, float alpha,
                                                                       const unsigned char* __restrict__ q, int64_t ldq,
                                                                       const T* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                                                       int64_t ldg, const T* __restrict__ x, int64_t ldx, float beta,
                                                                       T* __restrict__ y, int64_t ldy, int units_per_wave) {
    extern __shared__ __align__(16) float part[];  // [wave][tile][4][lane]
    constexpr int kGroup = 32 * kGroupSteps, kGroups = 4 / kGroupSteps;  // columns of a group, groups of a unit
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int waves = blockDim.x / kWave;
    const int row = lane & 15, quarter = lane >> 4;
    const int m0 = blockIdx.x * kRowTiles * 16, t0 = blockIdx.y * kTokTiles * 16;
    const int full = N / kW4Unit, units = (N + kW4Unit - 1) / kW4Unit, groups = (N + kGroup - 1) / kGroup;
    const int begin = wave * units_per_wave, end = min(full & ~1, begin + units_per_wave);  // units_per_wave is even
    const unsigned char* wp[kRowTiles];
    const T* sp[kRowTiles];
    const unsigned char* zp[kRowTiles];
    const T* xp[kTokTiles];
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r) {
        const int64_t m = min(m0 + r * 16 + row, M - 1);
        wp[r] = q + m * ldq + quarter * 16;
        sp[r] = scales + m * ldg;
        zp[r] = kZeros ? zeros + m * ldg : nullptr;
    }
#pragma unroll
    for (int t = 0; t < kTokTiles; ++t) xp[t] = x + static_cast<int64_t>(min(t0 + t * 16 + row, batch - 1)) * ldx + quarter * 8;

    v4f total[kTokTiles][kRowTiles];
#pragma unroll
    for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) total[t][r] = v4f{0.f, 0.f, 0.f, 0.f};

    // one unit: 32 columns at a time, the scale applied where a group ends
    auto unit_products = [&](const v4u (&wt)[kRowTiles], const float (&scale)[kRowTiles][kGroups], const float (&offset)[kRowTiles][kGroups],
                             const v4u (&xv)[kTokTiles][4]) {
        constexpr unsigned kOne = std::is_same_v<T, f16> ? 0x3C003C00u : 0x3F803F80u;
        const v4u ones = {kOne, kOne, kOne, kOne};
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            v4f acc[kTokTiles][kRowTiles], sum[kTokTiles];
#pragma unroll
            for (int k = 0; k < kGroupSteps; ++k) {
                const int d = g * kGroupSteps + k;
                const v4f zero = {0.f, 0.f, 0.f, 0.f};
                v4u xo[kTokTiles];
#pragma unroll
                for (int t = 0; t < kTokTiles; ++t) {
                    xo[t] = pair_order(xv[t][d]);
                    sum[t] = mfma_16x16x32<T>(xo[t], ones, k == 0 ? zero : sum[t]);
                }
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    const v4u wq = nibbles_plus_16<T>(wt[r][d]);
#pragma unroll
                    for (int t = 0; t < kTokTiles; ++t) acc[t][r] = mfma_16x16x32<T>(xo[t], wq, k == 0 ? zero : acc[t][r]);
                }
            }
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
                for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        total[t][r][i] = __builtin_fmaf(scale[r][g], __builtin_fmaf(-offset[r][g], sum[t][i], acc[t][r][i]), total[t][r][i]);
        }
    };
    v4u wt[kRowTiles];
    float scale[kRowTiles][kGroups], offset[kRowTiles][kGroups];

    if (begin < end) {
        // Units go in pairs (begin and end are even).  Everything of a pair is requested one pair ahead and in the order of
        // its use, since loads return in order; the scales of a pair are consecutive, one load per row.
        typedef T pair_scales __attribute__((ext_vector_type(2 * kGroups)));
        typedef unsigned char pair_zeros __attribute__((ext_vector_type(2 * kGroups)));
        typedef pair_scales pair_scales_any __attribute__((aligned(2)));
        typedef pair_zeros pair_zeros_any __attribute__((aligned(1)));
        v4u w[2][kRowTiles], xv[2][kTokTiles][4];
        pair_scales sv[kRowTiles];
        pair_zeros zv[kRowTiles];
        // past the wave's last pair the loads repeat it: without a branch they stay in flight
        auto load_scales = [&](int u) {
            const int64_t g = static_cast<int64_t>(min(u, end - 2)) * kGroups;
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
                sv[r] = *reinterpret_cast<const pair_scales_any*>(sp[r] + g);
                if (kZeros) zv[r] = *reinterpret_cast<const pair_zeros_any*>(zp[r] + g);
            }
        };
        auto load_unit = [&](int u, int k) {
            const int64_t at = min(u, end - 2) + k;
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) w[k][r] = load16(reinterpret_cast<const T*>(wp[r] + at * (kW4Unit / 2)));
#pragma unroll
            for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                for (int d = 0; d < 4; ++d) xv[k][t][d] = load16(xp[t] + at * kW4Unit + d * 32);
        };
        load_scales(begin);
        load_unit(begin, 0);
        load_unit(begin, 1);
        for (int u = begin; u < end; u += 2) {
            float pair_scale[2][kRowTiles][kGroups], pair_offset[2][kRowTiles][kGroups];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        pair_scale[k][r][g] = static_cast<float>(sv[r][k * kGroups + g]);
                        pair_offset[k][r][g] = 16.f + (kZeros ? static_cast<float>(zv[r][k * kGroups + g]) : 8.f);
                    }
            load_scales(u + 2);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) wt[r] = transpose_quarters(w[k][r]);
                unit_products(wt, pair_scale[k], pair_offset[k], xv[k]);
                load_unit(u + 2, k);
            }
        }
    }
    // the last, odd unit and the columns behind the last whole one, one at a time
    for (int u = max(full & ~1, wave * units_per_wave); u < min(units, (wave + 1) * units_per_wave); ++u) {
        v4u xv[kTokTiles][4];
        const int row_bytes = (N + 1) / 2, at = u * (kW4Unit / 2) + quarter * 16;
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
            v4u w;
#pragma unroll
            for (int d = 0; d < 4; ++d)  // whole dwords: the last may hold bytes behind the row, whose x is zero
                w[d] = at + 4 * d < row_bytes ? *reinterpret_cast<const unsigned*>(wp[r] + u * (kW4Unit / 2) + 4 * d) : 0u;
            wt[r] = transpose_quarters(w);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int64_t i = min(u * kGroups + g, groups - 1);  // behind the last column: x is zero
                scale[r][g] = static_cast<float>(sp[r][i]);
                offset[r][g] = 16.f + (kZeros ? static_cast<float>(zp[r][i]) : 8.f);
            }
        }
#pragma unroll
        for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) xv[t][d] = load_row(xp[t] - quarter * 8, u * kW4Unit + d * 32 + quarter * 8, N);
        unit_products(wt, scale, offset, xv);
    }

    constexpr int kTiles = kTokTiles * kRowTiles;
#pragma unroll
    for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[((wave * kTiles + t * kRowTiles + r) * 4 + i) * kWave + lane] = total[t][r][i];
    __syncthreads();
    for (int o = threadIdx.x; o < kTiles * 4 * kWave; o += blockDim.x) {
        float v = part[o];
        for (int k = 1; k < waves; ++k) v += part[k * kTiles * 4 * kWave + o];
        const int l = o & (kWave - 1), i = (o / kWave) & 3, tile = o / (4 * kWave);
        const int m = m0 + (tile % kRowTiles) * 16 + (l & 15), t = t0 + (tile / kRowTiles) * 16 + 4 * (l >> 4) + i;
        if (m < M && t < batch) {
            T* dst = y + t * ldy + m;
            v *= alpha;
            *dst = static_cast<T>(beta == 0.f ? v : __builtin_fmaf(beta, static_cast<float>(*dst), v));
        }
    }
}

namespace {

// Columns of x that LDS holds for TB tokens, a multiple of 2048; panels of equal size where one does not hold all.
int panel_of(int N, int tb, size_t elem) {
    const int most = static_cast<int>(kW4LdsBytes / (tb * (kW4Piece * elem + kWave * sizeof(float))));
    const int pieces = std::max(1, static_cast<int>(ceil_div(N, kW4Piece)));
    const int panels = static_cast<int>(ceil_div(pieces, most));
    return static_cast<int>(ceil_div(pieces, panels)) * kW4Piece;
}

template <class T, bool kZeros>
int launch_w4(int batch, int M, int N, int group_shift, float alpha, const unsigned char* q, int64_t ldq, const void* scales,
              const unsigned char* zeros, int64_t ldg, const void* x, int64_t ldx, float beta, void* y, int64_t ldy, hipStream_t stream) {
    const int cus = device_cus();
    auto go = [&](auto tb, auto rows) {
        constexpr int TB = decltype(tb)::value, kRows = decltype(rows)::value, kPieces = kRows < 4 ? 4 / kRows : 1;
        const int panel = panel_of(N, TB, sizeof(T));
        const size_t lds = static_cast<size_t>(TB) * panel * sizeof(T) + static_cast<size_t>(TB) * panel / kW4Cols * sizeof(float);
        // one workgroup of sixteen waves per CU; fewer waves while there are not enough rows for that
        int waves = kW4MaxWaves;
        while (waves > 4 && ceil_div(M, waves * kRows) < cus) waves /= 2;
        const int unit = waves * kRows;
        const int per_block = static_cast<int>(ceil_div(ceil_div(M, unit), cus * (W4BPC))) * unit;
        const dim3 grid(static_cast<unsigned>(ceil_div(M, per_block)), static_cast<unsigned>(ceil_div(batch, TB)));
        w4_gemv_kernel<T, TB, kRows, kPieces, kZeros><<<grid, waves * kWave, lds, stream>>>(
            batch, M, N, group_shift, alpha, q, ldq, static_cast<const T*>(scales), zeros, ldg, static_cast<const T*>(x), ldx, beta,
            static_cast<T*>(y), ldy, per_block, panel);
    };
    using std::integral_constant;
    if constexpr (sizeof(T) == 2)
        if (batch >= W4MIN && N > 0) {
            auto tile = [&](auto row_tiles, auto tok_tiles) {
                constexpr int kRowTiles = decltype(row_tiles)::value, kTokTiles = decltype(tok_tiles)::value;
                const int units = static_cast<int>(ceil_div(N, kW4Unit));
                const int per_wave = static_cast<int>(ceil_div(units, 2 * W4TW)) * 2;
                const int waves = static_cast<int>(ceil_div(units, per_wave));
                const size_t lds = static_cast<size_t>(waves) * kRowTiles * kTokTiles * 4 * kWave * sizeof(float);
                const dim3 grid(static_cast<unsigned>(ceil_div(M, 16 * kRowTiles)), static_cast<unsigned>(ceil_div(batch, 16 * kTokTiles)));
                auto of_group = [&](auto steps) {
                w4_tile_kernel<T, kRowTiles, kTokTiles, decltype(steps)::value, kZeros><<<grid, waves * kWave, lds, stream>>>(
                    batch, M, N, alpha, q, ldq, static_cast<const T*>(scales), zeros, ldg, static_cast<const T*>(x), ldx, beta,
                    static_cast<T*>(y), ldy, per_wave);
                };
                if (group_shift == 5) of_group(integral_constant<int, 1>{});
                else if (group_shift == 6) of_group(integral_constant<int, 2>{});
                else of_group(integral_constant<int, 4>{});
            };
            tile(integral_constant<int, W4RT>{}, integral_constant<int, 1>{});
            return launch_status();
        }
    // rows per wave and step: as many as leave every CU its sixteen waves
    auto by_rows = [&](auto tb) {
        if (M >= 64 * cus W4ROWS) go(tb, integral_constant<int, 4>{});
        else if (M >= 32 * cus W4ROWS) go(tb, integral_constant<int, 2>{});
        else go(tb, integral_constant<int, 1>{});
    };
    if (batch == 1) by_rows(integral_constant<int, 1>{});
    else if (batch == 2) by_rows(integral_constant<int, 2>{});
    else by_rows(integral_constant<int, 4>{});
    return launch_status();
}

int shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

}  // namespace
}  // namespace hpcdnn

extern "C" int hpcdnn_w4_gemv(int type, int batch, int M, int N, int group, float alpha, const uint8_t* q, int64_t ldq,
                              const void* scales, const uint8_t* zeros, int64_t ldg, const void* x, int64_t ldx, float beta, void* y,
                              int64_t ldy, void* stream) {
    using namespace hpcdnn;
    const int shift = shift_of(group);
    if (!type_valid(type) || batch < 0 || M < 0 || N < 0 || shift < 0 || N > HPCDNN_W4_MAX_COLS || batch > HPCDNN_W4_MAX_BATCH)
        return HPCDNN_ERR_INVALID_VALUE;
    if (batch == 0 || M == 0) return HPCDNN_OK;
    const size_t e = type_bytes(type);
    if (y == nullptr || ldy < M || !aligned(y, e)) return HPCDNN_ERR_INVALID_VALUE;
    if (N > 0 && (q == nullptr || !aligned(q, 4) || ldq % 4 != 0 || ldq < (N + 1) / 2 || scales == nullptr || !aligned(scales, e) ||
                  ldg < ceil_div(N, group) || x == nullptr || !aligned(x, e) || ldx < N))
        return HPCDNN_ERR_INVALID_VALUE;
    return with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (zeros != nullptr)
            return launch_w4<T, true>(batch, M, N, shift, alpha, q, ldq, scales, zeros, ldg, x, ldx, beta, y, ldy, static_cast<hipStream_t>(stream));
        return launch_w4<T, false>(batch, M, N, shift, alpha, q, ldq, scales, zeros, ldg, x, ldx, beta, y, ldy, static_cast<hipStream_t>(stream));
    });
}

// Host packing.  Symmetric (zeros == NULL): s = max |w| / 7 over the group, q = 8 + w / s rounded to nearest, ties to even,
// within 0 .. 15.  With zero points: s = (max - min) / 15 with 0 inside the range, z = -min / s rounded, q = z + w / s rounded.
// s is rounded to `type` first and q follows from the rounded one.
extern "C" int hpcdnn_w4_quantize(int type, int M, int N, int group, const float* W, int64_t ldw, uint8_t* q, int64_t ldq, void* scales,
                                  uint8_t* zeros, int64_t ldg) {
    using namespace hpcdnn;
    if (!type_valid(type) || M < 0 || N < 0 || shift_of(group) < 0) return HPCDNN_ERR_INVALID_VALUE;
    if (M == 0 || N == 0) return HPCDNN_OK;
    if (W == nullptr || ldw < N || q == nullptr || ldq < (N + 1) / 2 || scales == nullptr || ldg < ceil_div(N, group))
        return HPCDNN_ERR_INVALID_VALUE;
    return with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        for (int m = 0; m < M; ++m) {
            const float* w = W + m * ldw;
            uint8_t* out = q + m * ldq;
            std::fill(out, out + (N + 1) / 2, static_cast<uint8_t>(0));
            for (int g = 0; g * group < N; ++g) {
                const int n0 = g * group, n1 = std::min(N, n0 + group);
                float lo = 0.f, hi = 0.f;
                for (int n = n0; n < n1; ++n) {
                    if (!std::isfinite(w[n])) return HPCDNN_ERR_INVALID_VALUE;
                    lo = std::min(lo, w[n]);
                    hi = std::max(hi, w[n]);
                }
                const T scale = static_cast<T>(zeros ? hi / 15.f - lo / 15.f : std::max(hi, -lo) / 7.f);
                const float s = static_cast<float>(scale);
                if (!std::isfinite(s)) return HPCDNN_ERR_INVALID_VALUE;
                const float z = !zeros ? 8.f : s == 0.f ? 0.f : std::min(15.f, std::nearbyint(-lo / s));
                static_cast<T*>(scales)[m * ldg + g] = scale;
                if (zeros) zeros[m * ldg + g] = static_cast<uint8_t>(z);
                for (int n = n0; n < n1; ++n) {
                    const float v = s == 0.f ? z : std::max(0.f, std::min(15.f, std::nearbyint(w[n] / s) + z));
                    out[n / 2] = static_cast<uint8_t>(out[n / 2] | (static_cast<unsigned>(v) << (4 * (n & 1))));
                }
            }
        }
        return HPCDNN_OK;
    });
}
