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

namespace hpcdnn {

constexpr int kW4Cols = 32;                      // columns of one lane and load
constexpr int kW4Piece = kW4Cols * kWave;        // columns of a wave and load
constexpr int kW4Waves = 8;                      // waves of a workgroup
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

// One wave takes kRows rows at a time through all columns, kPieces pieces of 2048 columns per row in flight; TB tokens at
// a time.  blockIdx.y counts groups of TB tokens.
template <class T, int TB, int kRows, int kPieces, bool kZeros>
__global__ __launch_bounds__(kW4Waves * kWave) void w4_gemv_kernel(int batch, int M, int N, int group_shift, float alpha,
                                                                   const unsigned char* __restrict__ q, int64_t ldq,
                                                                   const T* __restrict__ scales, const unsigned char* __restrict__ zeros,
                                                                   int64_t ldg, const T* __restrict__ x, int64_t ldx, float beta,
                                                                   T* __restrict__ y, int64_t ldy, int rows_per_block, int panel) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int pieces = panel / kW4Piece;
    float* sums = reinterpret_cast<float*>(lds + static_cast<size_t>(TB) * panel * sizeof(T));
    const int t0 = blockIdx.y * TB, tokens = min(TB, batch - t0);
    x += t0 * ldx;
    y += t0 * ldy;
    const int row_bytes = ((N + 1) / 2 + 3) & ~3;  // whole dwords: the last may hold bytes behind the row, whose x is zero
    const int first = blockIdx.x * rows_per_block;
    bool staged = false;
    for (int r0 = first; r0 < min(M, first + rows_per_block); r0 += kW4Waves * kRows) {
        const int m0 = r0 + wave * kRows;
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
            if (m0 >= M) continue;
            for (int p0 = 0; p0 < pieces; p0 += kPieces) {
                v4u w[kRows][kPieces];
                float s[kRows][kPieces], z[kRows][kPieces];
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const int m = min(m0 + r, M - 1);
                    const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const float*>(q + m * ldq), row_bytes);
#pragma unroll
                    for (int u = 0; u < kPieces; ++u) {
                        const int col = n0 + (p0 + u) * kW4Piece + lane * kW4Cols;
                        const bool in = p0 + u < pieces && col < N;
                        w[r][u] = __builtin_amdgcn_raw_buffer_load_b128(rs, in ? col / 2 : row_bytes, 0, 0);
                        s[r][u] = in ? static_cast<float>(scales[m * ldg + (col >> group_shift)]) : 0.f;
                        if (kZeros) z[r][u] = in ? static_cast<float>(zeros[m * ldg + (col >> group_shift)]) : 0.f;
                        else z[r][u] = 8.f;
                    }
                }
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
                                const v4u wq = nibbles_plus_16<T>(w[r][u][d]);
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
                                const unsigned even = w[r][u][d] & 0x0f0f0f0fu, odd = (w[r][u][d] >> 4) & 0x0f0f0f0fu;
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float wk = static_cast<float>((((k & 1) ? odd : even) >> (8 * (k / 2))) & 0xffu);
#pragma unroll
                                    for (int t = 0; t < TB; ++t) dot[r][t] = __builtin_fmaf(wk, xv[t][k / 4][k & 3], dot[r][t]);
                                }
                            }
                        }
                    }
                    constexpr float kOffset = sizeof(T) == 2 ? 16.f : 0.f;
#pragma unroll
                    for (int t = 0; t < TB; ++t) {
                        const float sx = sums[(t * pieces + p0 + u) * kWave + lane];
#pragma unroll
                        for (int r = 0; r < kRows; ++r)
                            acc[r][t] = __builtin_fmaf(s[r][u], __builtin_fmaf(-(kOffset + z[r][u]), sx, dot[r][t]), acc[r][t]);
                    }
                }
            }
        }
        if (m0 >= M) continue;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const float v = alpha * wave_allsum(acc[r][t]);
                if (lane == r * TB + t && m0 + r < M && t < tokens) {
                    T* dst = y + t * ldy + m0 + r;
                    *dst = static_cast<T>(beta == 0.f ? v : __builtin_fmaf(beta, static_cast<float>(*dst), v));
                }
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
    auto go = [&](auto tb, auto rows, auto pieces) {
        constexpr int TB = decltype(tb)::value, kRows = decltype(rows)::value, kPieces = decltype(pieces)::value;
        const int panel = panel_of(N, TB, sizeof(T));
        const size_t lds = static_cast<size_t>(TB) * panel * sizeof(T) + static_cast<size_t>(TB) * panel / kW4Cols * sizeof(float);
        const int unit = kW4Waves * kRows;
        const int units = static_cast<int>(ceil_div(M, unit));
        const int per_block = static_cast<int>(ceil_div(units, 2 * device_cus())) * unit;
        const dim3 grid(static_cast<unsigned>(ceil_div(M, per_block)), static_cast<unsigned>(ceil_div(batch, TB)));
        w4_gemv_kernel<T, TB, kRows, kPieces, kZeros><<<grid, kW4Waves * kWave, lds, stream>>>(
            batch, M, N, group_shift, alpha, q, ldq, static_cast<const T*>(scales), zeros, ldg, static_cast<const T*>(x), ldx, beta,
            static_cast<T*>(y), ldy, per_block, panel);
    };
    using std::integral_constant;
    if (batch == 1) go(integral_constant<int, 1>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{});
    else go(integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
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
