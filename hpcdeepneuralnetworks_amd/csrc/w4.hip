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
//    within a factor of about five of the result.  FP32 tokens use byte-to-float conversions and q itself, on the matrix
//    cores q - z, which BF16 holds, and three BF16 in the place of each FP32 value.
//  - x lies in LDS in the order in which the lanes need it, its sums over 32 columns beside it.
// Dot and matrix instructions take 16-bit values below the smallest normal number as they are, so these count in full and
// cancel against the sums, which are formed from conversions in one form and by the matrix cores in the other.
// Measured, one token: 16384 x 16384 FP16 in groups of 64 with zero points 28 us (5.2 TB/s), 4096 x 4096 BF16 5.3 us.
#include <algorithm>
#include <cmath>

#include "layer_types.h"

namespace hpcdnn {

constexpr int kW4Cols = 32;                      // columns of one lane and load
constexpr int kW4Piece = kW4Cols * kWave;        // columns of a wave and load
constexpr int kW4MaxWaves = 16;                  // waves of a workgroup
constexpr size_t kW4LdsBytes = 163840;           // of a CU

template <class T>
constexpr int kW4Parts = kW4Cols / kVec<T>;      // 16-byte parts of a lane's x

// 16-bit pairs for the dot instruction: dword p = columns (p, p + 4) of eight.
__device__ __forceinline__ v4u pair_order(v4u d) {
    return v4u{__builtin_amdgcn_perm(d[2], d[0], 0x05040100u), __builtin_amdgcn_perm(d[2], d[0], 0x07060302u),
               __builtin_amdgcn_perm(d[3], d[1], 0x05040100u), __builtin_amdgcn_perm(d[3], d[1], 0x07060302u)};
}

// The eight nibbles of w as 16 + q in T, columns (p, p + 4) in dword p: a shift and an and-or each.  An instruction takes
// one constant from a scalar register and none from the instruction stream beside it, so the second has to be a vector
// register; left to itself the compiler uses two instructions with a literal each instead.
template <class T>
struct nibble_maker {
    static constexpr unsigned kMask = std::is_same_v<T, f16> ? 0x03C003C0u : 0x00780078u;  // where q stands in the mantissa of 16.0
    unsigned one = std::is_same_v<T, f16> ? 0x4C004C00u : 0x41804180u;
    __device__ __forceinline__ nibble_maker() { asm("" : "+v"(one)); }
    __device__ __forceinline__ unsigned put(unsigned w) const { return (w & kMask) | (one & ~kMask); }
    __device__ __forceinline__ v4u operator()(unsigned w) const {
        if constexpr (std::is_same_v<T, f16>) return v4u{put(w << 6), put(w << 2), put(w >> 2), put(w >> 6)};
        else return v4u{put(w << 3), put(w >> 1), put(w >> 5), put(w >> 9)};
    }
};

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

    [[maybe_unused]] const nibble_maker<std::conditional_t<sizeof(T) == 2, T, f16>> nibbles;

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
                w[r][u] = __builtin_amdgcn_raw_buffer_load_b128(rs, col / 2, 0, 2);  // non-temporal: read once (4 % faster)
                const int64_t g = at * ldg + (min(col, N - 1) >> group_shift);  // behind the last column: x is zero
                s[r][u] = scales[g];
                if (kZeros) z[r][u] = zeros[g];
            }
        }
        loads_start_here();
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
                                const v4u wq = nibbles(now[r][u][d]);
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
// LDS at the end (in wave order).  Columns are not split over workgroups: a matrix of fewer than 16 rows per CU leaves CUs
// without work (sixteen BF16 tokens by 1024 x 8192 7.6 us, on 64 of them), and every 16 or 32 tokens unpack the weights again
// (2048 BF16 tokens by 16384 x 16384 2.8 ms, 390 TFLOP/s, a third of a plain product's rate).
//
// What limits it is the number of cache lines and 64-byte pieces that the loads touch: neighbouring lanes therefore load
// neighbouring 16 bytes (four lanes a row's unit of weights, four lanes 64 bytes of a token), and the order that the
// instructions want, row or token l % 16 and part l / 16 in lane l, comes about in LDS, each wave for itself.  (Loaded in that
// order right away, thirteen tokens by 6143 x 8200 took 20 us; scales go through LDS as well, sixteen of a row at a time.)
//
// An instruction sums over the four quarters of the lanes, so the dwords of the weights are exchanged between the quarters (a
// 4 x 4 transposition in four lane swaps): dword d is then columns 32 d + 8 (l / 16) ... of the unit, and every instruction
// stays inside one group.  The sums over x that take out the offset of the nibbles come from the same instruction with a
// matrix of ones.
//
// FP32 tokens are taken apart into three BF16 each, exactly, and multiplied by q - z, which BF16 holds: three instructions of
// 32 columns in the place of eight of four columns, each twice as long, and the products are exact as well.  (Sixteen tokens
// by 16384 x 16384 63 us, with the FP32 instruction 115; seven by 6143 x 8201 26 and 37.)
constexpr int kW4Unit = 128;
// Tokens from which this form is taken.  16-bit: two cost the other form 32 us on 16384 x 16384 and this one 35, four 45 and 36.
// FP32: three by 16384 x 16384 53 us and 60, by 4224 x 9408 22 and 26; four by 9984 x 11287 75 and 38, by 8192 x 8192 25 and 22.
template <class T>
constexpr int kW4TileTokens = sizeof(T) == 2 ? 3 : 4;
constexpr int kW4TileWaves = 8;
constexpr int kW4Segment = 16;  // scales of a row that a wave keeps in LDS at a time
template <class T>
constexpr int kW4Exchange = kWave * 8 * static_cast<int>(sizeof(T));  // 8 values of every lane

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

// Bits 16 ... 31 of eight FP32 values, which for values that BF16 holds is their conversion.
__device__ __forceinline__ v4u upper_halves(const float (&f)[8]) {
    v4u u;
#pragma unroll
    for (int p = 0; p < 4; ++p)
        u[p] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, f[2 * p + 1]), __builtin_bit_cast(unsigned, f[2 * p]), 0x07060302u);
    return u;
}

// Eight FP32 values as three BF16 each, which add up to them: 24 bits are eight of the value, eight of what is left and
// eight of what is left then.
__device__ __forceinline__ void three_bf16(v4u lo, v4u hi, v4u (&out)[3]) {
    float f[8], left[8];
    auto upper = [](float v) { return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & 0xffff0000u); };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        f[i] = __builtin_bit_cast(float, static_cast<unsigned>(i < 4 ? lo[i & 3] : hi[i & 3]));
        left[i] = f[i] - upper(f[i]);
    }
    out[0] = upper_halves(f);
    out[1] = upper_halves(left);
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] -= upper(left[i]);
    out[2] = upper_halves(left);
}

// q - z of the eight nibbles of w: at most eight bits, so BF16 holds it.
__device__ __forceinline__ v4u exact_weights(unsigned w, float z) {
    const unsigned even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<float>((((j & 1) ? odd : even) >> (8 * (j / 2))) & 0xffu) - z;
    return upper_halves(f);
}

// LDS of a wave of the kernel below: its parts, or its sums at the end.
template <class T>
constexpr int w4_tile_lds(int row_tiles, int tok_tiles) {
    const int parts = kW4Exchange<T> + row_tiles * 16 * kW4Segment * (static_cast<int>(sizeof(T)) + 1), sums = row_tiles * tok_tiles * 4 * kWave * 4;
    return parts > sums ? parts : sums;
}

template <class T, int kRowTiles, int kTokTiles, int kGroupSteps, bool kZeros>
__global__ __launch_bounds__(kW4TileWaves * kWave) void w4_tile_kernel(int batch, int M, int N, float alpha,
                                                                       const unsigned char* __restrict__ q, int64_t ldq,
                                                                       const T* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                                                       int64_t ldg, const T* __restrict__ x, int64_t ldx, float beta,
                                                                       T* __restrict__ y, int64_t ldy, int units_per_wave) {
    extern __shared__ __align__(16) float part[];  // the waves' own parts, at the end their sums [wave][tile][4][lane]
    constexpr int kGroup = 32 * kGroupSteps, kGroups = 4 / kGroupSteps;  // columns of a group, groups of a unit
    constexpr bool kF32 = std::is_same_v<T, float>;
    constexpr int kXParts = kF32 ? 8 : 4;          // 16-byte parts of x that a lane has of a unit
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int waves = blockDim.x / kWave;
    const int row = lane & 15, quarter = lane >> 4;
    const int m0 = blockIdx.x * kRowTiles * 16, t0 = blockIdx.y * kTokTiles * 16;
    const int full = N / kW4Unit, units = (N + kW4Unit - 1) / kW4Unit, groups = (N + kGroup - 1) / kGroup;
    const int begin = wave * units_per_wave, end = min(full & ~1, begin + units_per_wave);  // units_per_wave is even
    // rows of the lane as the instructions want them (row) and as they are loaded (lane / 4)
    auto row_at = [&](int tile, int i) { return static_cast<int64_t>(min(m0 + tile * 16 + i, M - 1)); };
    const unsigned char* wp[kRowTiles];
    const T* sp[kRowTiles];
    const unsigned char* zp[kRowTiles];
    const T* xp[kTokTiles];
    const int load_row_of = lane >> 2, load_part = lane & 3;
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r) {
        const int64_t m = row_at(r, load_row_of);
        wp[r] = q + m * ldq + load_part * 16;
        sp[r] = scales + m * ldg;
        zp[r] = kZeros ? zeros + m * ldg : nullptr;
    }
    // LDS of the wave: 16 bytes of every lane on their way to another, scales and zero points of a segment
    char* const mine = reinterpret_cast<char*>(part) + wave * w4_tile_lds<T>(kRowTiles, kTokTiles);
    T* const my_s = reinterpret_cast<T*>(mine + kW4Exchange<T>);
    unsigned char* const my_z = reinterpret_cast<unsigned char*>(my_s + kRowTiles * 16 * kW4Segment);
#pragma unroll
    for (int t = 0; t < kTokTiles; ++t) xp[t] = x + static_cast<int64_t>(min(t0 + t * 16 + load_row_of, batch - 1)) * ldx + load_part * kVec<T>;

    v4f total[kTokTiles][kRowTiles];
#pragma unroll
    for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) total[t][r] = v4f{0.f, 0.f, 0.f, 0.f};

    [[maybe_unused]] const nibble_maker<std::conditional_t<kF32, f16, T>> nibbles;
    // one unit: 32 columns at a time, the scale applied where a group ends
    auto unit_products = [&](const v4u (&wt)[kRowTiles], const float (&scale)[kRowTiles][kGroups], const float (&offset)[kRowTiles][kGroups],
                             const v4u (&xv)[kTokTiles][kXParts]) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            v4f acc[kTokTiles][kRowTiles];
            [[maybe_unused]] v4f sum[kTokTiles];
#pragma unroll
            for (int t = 0; t < kTokTiles; ++t) {
                sum[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) acc[t][r] = v4f{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int d = g * kGroupSteps; d < (g + 1) * kGroupSteps; ++d) {
                if constexpr (kF32) {
                    v4u xo[kTokTiles][3];
#pragma unroll
                    for (int t = 0; t < kTokTiles; ++t) three_bf16(xv[t][2 * d], xv[t][2 * d + 1], xo[t]);
#pragma unroll
                    for (int r = 0; r < kRowTiles; ++r) {
                        const v4u wq = exact_weights(wt[r][d], offset[r][g]);
#pragma unroll
                        for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                            for (int k = 0; k < 3; ++k) acc[t][r] = mfma_16x16x32<bf16>(xo[t][k], wq, acc[t][r]);
                    }
                } else {
                    constexpr unsigned kOne = std::is_same_v<T, f16> ? 0x3C003C00u : 0x3F803F80u;
                    const v4u ones = {kOne, kOne, kOne, kOne};
                    v4u xo[kTokTiles];
#pragma unroll
                    for (int t = 0; t < kTokTiles; ++t) {
                        xo[t] = pair_order(xv[t][d]);
                        sum[t] = mfma_16x16x32<T>(xo[t], ones, sum[t]);
                    }
#pragma unroll
                    for (int r = 0; r < kRowTiles; ++r) {
                        const v4u wq = nibbles(wt[r][d]);
#pragma unroll
                        for (int t = 0; t < kTokTiles; ++t) acc[t][r] = mfma_16x16x32<T>(xo[t], wq, acc[t][r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
                for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float dot = kF32 ? acc[t][r][i] : __builtin_fmaf(-offset[r][g], sum[t][i], acc[t][r][i]);
                        total[t][r][i] = __builtin_fmaf(scale[r][g], dot, total[t][r][i]);
                    }
        }
    };
    // Part p of row i stands at (p ^ i / 2 % 4): eight lanes meet no bank twice, neither writing nor reading (a third of the
    // conflicts counted with i / 4 or without).  A wave's LDS accesses are carried out in order, so one place does for all.
    auto to_instruction_order = [&](v4u v) {
        *reinterpret_cast<v4u*>(mine + load_row_of * 64 + ((load_part ^ (load_row_of >> 1)) & 3) * 16) = v;
        __builtin_amdgcn_wave_barrier();
        const v4u got = *reinterpret_cast<const v4u*>(mine + row * 64 + ((quarter ^ (row >> 1)) & 3) * 16);
        __builtin_amdgcn_wave_barrier();
        return got;
    };
    // FP32: the eight parts of a step's 32 columns, of which a lane wants parts 2 (l / 16) and the next; part p of token i at
    // (p ^ i / 2 % 8).
    [[maybe_unused]] auto to_instruction_order2 = [&](v4u lo, v4u hi, v4u& first, v4u& second) {
        char* const put = mine + load_row_of * 128;
        const int put_at = (load_row_of >> 1) & 7, get_at = (row >> 1) & 7;
        *reinterpret_cast<v4u*>(put + (load_part ^ put_at) * 16) = lo;
        *reinterpret_cast<v4u*>(put + ((load_part + 4) ^ put_at) * 16) = hi;
        __builtin_amdgcn_wave_barrier();
        first = *reinterpret_cast<const v4u*>(mine + row * 128 + ((2 * quarter) ^ get_at) * 16);
        second = *reinterpret_cast<const v4u*>(mine + row * 128 + ((2 * quarter + 1) ^ get_at) * 16);
        __builtin_amdgcn_wave_barrier();
    };
    constexpr float kOffset = kF32 ? 0.f : 16.f;   // what stands on a weight beside its zero point
    v4u wt[kRowTiles];
    float scale[kRowTiles][kGroups], offset[kRowTiles][kGroups];

    if (begin < end) {
        // Units go in pairs (begin and end are even).  Everything of a pair is requested one pair ahead, and in the order of
        // its use, since loads return in order.
        typedef T scales4 __attribute__((ext_vector_type(4)));
        typedef unsigned char zeros4 __attribute__((ext_vector_type(4)));
        typedef scales4 scales4_any __attribute__((aligned(2)));
        typedef zeros4 zeros4_any __attribute__((aligned(1)));
        constexpr int kSegmentUnits = kW4Segment / kGroups;
        v4u w[2][kRowTiles], xv[2][kTokTiles][kXParts];
        scales4 sv[kRowTiles];
        zeros4 zv[kRowTiles];
        // four scales of the lane's row from unit u on; behind the row's last one that one again (of no use)
        auto load_scales = [&](int u) {
            const int g = u * kGroups + 4 * load_part;
            const bool whole = (u + kSegmentUnits) * kGroups <= groups;  // the same for all lanes
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
                if (whole) {
                    sv[r] = *reinterpret_cast<const scales4_any*>(sp[r] + g);
                    if (kZeros) zv[r] = *reinterpret_cast<const zeros4_any*>(zp[r] + g);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sv[r][i] = sp[r][min(g + i, groups - 1)];
                        if (kZeros) zv[r][i] = zp[r][min(g + i, groups - 1)];
                    }
                }
            }
            loads_start_here();
        };
        // past the wave's last pair the loads repeat it: without a branch they stay in flight
        auto load_unit = [&](int u, int k) {
            const int64_t at = min(u, end - 2) + k;
#pragma unroll
            for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                for (int i = 0; i < kXParts; ++i) xv[k][t][i] = load16(xp[t] + at * kW4Unit + i * 4 * kVec<T>);
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) w[k][r] = load16(reinterpret_cast<const T*>(wp[r] + at * (kW4Unit / 2)));
            loads_start_here();
        };
        load_scales(begin);
        load_unit(begin, 0);
        load_unit(begin, 1);
        for (int u0 = begin; u0 < end; u0 += kSegmentUnits) {
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
                *reinterpret_cast<scales4*>(my_s + (r * 16 + load_row_of) * kW4Segment + 4 * load_part) = sv[r];
                if (kZeros) *reinterpret_cast<zeros4*>(my_z + (r * 16 + load_row_of) * kW4Segment + 4 * load_part) = zv[r];
            }
            __builtin_amdgcn_wave_barrier();
            load_scales(min(u0 + kSegmentUnits, end - 1));
            for (int u = u0; u < min(end, u0 + kSegmentUnits); u += 2) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    v4u xo[kTokTiles][kXParts];
#pragma unroll
                    for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            if constexpr (kF32) to_instruction_order2(xv[k][t][2 * d], xv[k][t][2 * d + 1], xo[t][2 * d], xo[t][2 * d + 1]);
                            else xo[t][d] = to_instruction_order(xv[k][t][d]);
                        }
#pragma unroll
                    for (int r = 0; r < kRowTiles; ++r) {
                        wt[r] = transpose_quarters(to_instruction_order(w[k][r]));
#pragma unroll
                        for (int g = 0; g < kGroups; ++g) {
                            const int at = (r * 16 + row) * kW4Segment + (u + k - u0) * kGroups + g;
                            scale[r][g] = static_cast<float>(my_s[at]);
                            offset[r][g] = kOffset + (kZeros ? static_cast<float>(my_z[at]) : 8.f);
                        }
                    }
                    load_unit(u + 2, k);
                    unit_products(wt, scale, offset, xo);
                }
            }
        }
    }
    // the last, odd unit and the columns behind the last whole one, one at a time
    for (int u = max(full & ~1, begin); u < min(units, begin + units_per_wave); ++u) {
        v4u xv[kTokTiles][kXParts];
        const int row_bytes = (N + 1) / 2, at = u * (kW4Unit / 2) + quarter * 16;
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
            const int64_t m = row_at(r, row);
            v4u w;
#pragma unroll
            for (int d = 0; d < 4; ++d)  // whole dwords: the last may hold bytes behind the row, whose x is zero
                w[d] = at + 4 * d < row_bytes ? *reinterpret_cast<const unsigned*>(q + m * ldq + at + 4 * d) : 0u;
            wt[r] = transpose_quarters(w);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int64_t i = min(u * kGroups + g, groups - 1);  // behind the last column: x is zero
                scale[r][g] = static_cast<float>(scales[m * ldg + i]);
                offset[r][g] = kOffset + (kZeros ? static_cast<float>(zeros[m * ldg + i]) : 8.f);
            }
        }
#pragma unroll
        for (int t = 0; t < kTokTiles; ++t)
#pragma unroll
            for (int i = 0; i < kXParts; ++i) {
                const int col = u * kW4Unit + (kF32 ? (i / 2) * 32 + quarter * 8 + (i & 1) * 4 : i * 32 + quarter * 8);
                xv[t][i] = load_row(x + static_cast<int64_t>(min(t0 + t * 16 + row, batch - 1)) * ldx, col, N);
            }
        unit_products(wt, scale, offset, xv);
    }

    __syncthreads();  // the waves' sums take the place of x
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

// Columns of x that LDS holds for TB tokens, a multiple of 2048; panels of equal size where one does not hold all.  A
// workgroup may take all of a CU's LDS (two FP32 tokens by 4224 x 9408 17 us, in two panels of 64 KiB at most 26).
int panel_of(int N, int tb, size_t elem) {
    const int most = static_cast<int>(kW4LdsBytes / (tb * (kW4Piece * elem + kWave * sizeof(float))));
    const int pieces = std::max(1, static_cast<int>(ceil_div(N, kW4Piece)));
    const int panels = static_cast<int>(ceil_div(pieces, most));
    return static_cast<int>(ceil_div(pieces, panels)) * kW4Piece;
}

template <class T, bool kZeros>
int launch_w4(int batch, int M, int N, int group_shift, float alpha, const unsigned char* q, int64_t ldq, const void* scales,
              const unsigned char* zeros, int64_t ldg, const void* x, int64_t ldx, float beta, void* y, int64_t ldy, hipStream_t stream) {
    using std::integral_constant;
    const int cus = device_cus();
    auto tile = [&](auto row_tiles, auto tok_tiles, auto steps) {
        constexpr int kRowTiles = decltype(row_tiles)::value, kTokTiles = decltype(tok_tiles)::value;
        const int units = static_cast<int>(ceil_div(N, kW4Unit));
        const int per_wave = static_cast<int>(ceil_div(units, 2 * kW4TileWaves)) * 2;
        const int waves = static_cast<int>(ceil_div(units, per_wave));
        const size_t lds = static_cast<size_t>(waves) * w4_tile_lds<T>(kRowTiles, kTokTiles);
        const dim3 grid(static_cast<unsigned>(ceil_div(M, 16 * kRowTiles)), static_cast<unsigned>(ceil_div(batch, 16 * kTokTiles)));
        w4_tile_kernel<T, kRowTiles, kTokTiles, decltype(steps)::value, kZeros><<<grid, waves * kWave, lds, stream>>>(
            batch, M, N, alpha, q, ldq, static_cast<const T*>(scales), zeros, ldg, static_cast<const T*>(x), ldx, beta, static_cast<T*>(y),
            ldy, per_wave);
    };
    auto of_group = [&](auto row_tiles, auto tok_tiles) {
        if (group_shift == 5) tile(row_tiles, tok_tiles, integral_constant<int, 1>{});
        else if (group_shift == 6) tile(row_tiles, tok_tiles, integral_constant<int, 2>{});
        else tile(row_tiles, tok_tiles, integral_constant<int, 4>{});
    };
    if (batch >= kW4TileTokens<T> && N > 0) {
        // Row tiles of a workgroup: it reads all of x once, which costs about as much as one of them, and the CU with the
        // most workgroups decides.  (Thirteen tokens, one / two / three / four tiles: 4096 x 8192 9.8 / 12.3 / - / 17.8 us,
        // 8192 x 8192 16.5 / 13.7 / 16.9 / 19.2 us; six by 9879 x 9920 25.0 / 30.5 / 23.9 / 28.4 us; sixteen by
        // 16384 x 16384 64 / 44 / 53 / 39 us.)  The rule does not see that four tiles pass the registers in some forms of the
        // small groups: FP16 in groups of 32 without zero points spills 45 (sixteen by 16384 x 16384 71 us, BF16 39), FP32
        // with zero points 17 in groups of 32 and 3 in groups of 64 (70 and 61 us, in groups of 128 57).
        auto cost = [&](int row_tiles, int tok_tiles) {
            return ceil_div(ceil_div(M, 16 * row_tiles) * ceil_div(batch, 16 * tok_tiles), cus) * (row_tiles + 1);
        };
        auto by_cost = [&](auto most_rows, auto tok_tiles) {
            constexpr int kTok = decltype(tok_tiles)::value, kMost = decltype(most_rows)::value;
            int best = 1;
            for (int r = 2; r <= kMost; ++r)
                if (cost(r, kTok) <= cost(best, kTok)) best = r;
            if (best == 1) of_group(integral_constant<int, 1>{}, tok_tiles);
            else if (best == 2) of_group(integral_constant<int, 2>{}, tok_tiles);
            else if constexpr (kMost > 2) {
                if (best == 3) of_group(integral_constant<int, 3>{}, tok_tiles);
                else of_group(integral_constant<int, 4>{}, tok_tiles);
            }
        };
        // Thirty-two 16-bit tokens go as two tiles of one workgroup: 8192 x 8192 18.1 us, as two workgroups 21.0.
        bool pairs = false;
        if constexpr (sizeof(T) == 2) {
            pairs = batch > 16;
            if (pairs) by_cost(integral_constant<int, 2>{}, integral_constant<int, 2>{});
        }
        if (!pairs) by_cost(integral_constant<int, 4>{}, integral_constant<int, 1>{});
        return launch_status();
    }
    auto go = [&](auto tb, auto rows) {
        constexpr int TB = decltype(tb)::value, kRows = decltype(rows)::value, kPieces = kRows < 4 ? 4 / kRows : 1;
        const int panel = panel_of(N, TB, sizeof(T));
        const size_t lds = static_cast<size_t>(TB) * panel * sizeof(T) + static_cast<size_t>(TB) * panel / kW4Cols * sizeof(float);
        // A CU holds sixteen waves.  As one workgroup they share x; as four of four waves, each with its own copy of x, they
        // follow M more closely: taken where that spares the CU with the most rows more than a quarter of them and the copies
        // fit (4149 x 8320 10.8 us, as one workgroup 11.4; 9000 x 2000 6.1 and 6.8; two copies of 9000 x 28672 37.1 and 33.8).
        auto most_rows = [&](int w) { return ceil_div(ceil_div(M, w * kRows), cus) * w * kRows; };
        const size_t copies = static_cast<size_t>(std::min<int64_t>(4, ceil_div(ceil_div(M, 4 * kRows), cus)));
        const int waves = 4 * most_rows(4) < 3 * most_rows(kW4MaxWaves) && copies * lds <= kW4LdsBytes ? 4 : kW4MaxWaves;
        const int unit = waves * kRows;
        // x in several panels is staged for every round of rows: one round per workgroup then
        const int per_block = panel < N ? unit : static_cast<int>(ceil_div(ceil_div(M, unit), cus * (kW4MaxWaves / waves))) * unit;
        const dim3 grid(static_cast<unsigned>(ceil_div(M, per_block)), static_cast<unsigned>(ceil_div(batch, TB)));
        auto* const fn = &w4_gemv_kernel<T, TB, kRows, kPieces, kZeros>;
        if (lds > 64 * 1024)
            if (int e = enable_lds(reinterpret_cast<const void*>(fn), kW4LdsBytes)) return e;
        fn<<<grid, waves * kWave, lds, stream>>>(
            batch, M, N, group_shift, alpha, q, ldq, static_cast<const T*>(scales), zeros, ldg, static_cast<const T*>(x), ldx, beta,
            static_cast<T*>(y), ldy, per_block, panel);
        return launch_status();
    };
    // Rows per wave and step: as many as leave every CU its sixteen waves.  Three FP32 tokens are bound by reading x from LDS,
    // so there two rows pay earlier: 8000 x 8192 21.4 us, with one row 23.0.
    auto by_rows = [&](auto tb, int two_rows_from) {
        if (M >= 64 * cus) return go(tb, integral_constant<int, 4>{});
        if (M >= two_rows_from * cus) return go(tb, integral_constant<int, 2>{});
        return go(tb, integral_constant<int, 1>{});
    };
    if (batch == 1) return by_rows(integral_constant<int, 1>{}, 32);
    if constexpr (sizeof(T) == 4)
        if (batch > 2) return by_rows(integral_constant<int, 3>{}, 16);
    return by_rows(integral_constant<int, 2>{}, 32);
}

int shift_of(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

}  // namespace
}  // namespace hpcdnn

extern "C" int hpcdnn_w4_gemv(int type, int batch, int M, int N, int group, float alpha, const uint8_t* q, int64_t ldq,
                              const void* scales, const uint8_t* zeros, int64_t ldg, const void* x, int64_t ldx, float beta, void* y,
                              int64_t ldy, void* stream) {
    using namespace hpcdnn;
    const int shift = shift_of(group);
    if (!type_valid(type) || batch < 0 || M < 0 || N < 0 || shift < 0 || N > HPCDNN_W4_MAX_COLS || M > HPCDNN_W4_MAX_ROWS || batch > HPCDNN_W4_MAX_BATCH)
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
    if (!type_valid(type) || M < 0 || N < 0 || shift_of(group) < 0 || N > HPCDNN_W4_MAX_COLS || M > HPCDNN_W4_MAX_ROWS)
        return HPCDNN_ERR_INVALID_VALUE;
    if (M == 0 || N == 0) return HPCDNN_OK;
    if (W == nullptr || !aligned(W, sizeof(float)) || ldw < N || q == nullptr || ldq < (N + 1) / 2 || scales == nullptr ||
        !aligned(scales, type_bytes(type)) || ldg < ceil_div(N, group))
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
