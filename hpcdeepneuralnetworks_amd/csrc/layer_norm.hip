// Layer normalisation over the rows of a row-major matrix, and its gradient.
//
//   mu = sum_c x / C,  var = sum_c (x - mu)^2 / C,  r = 1 / sqrt(var + eps),  y = (x - mu) r w + b
//   xh = (x - mu) r,   g = dy w,   dx = r (g - sum_c g / C - xh sum_c (g xh) / C),   dw = sum_rows dy xh,   db = sum_rows dy
//
// Both are bound by memory: 2 (forward) and 3 (gradient) values moved per element against about 10 operations.  A row
// is read once and stays in registers between its statistics and its result; all sums are FP32.  Measured: forward of
// 16384 x 4096 BF16 54 us (5.0 TB/s, the rate of a large copy), gradient of 16384 x 6144 BF16 112 us (5.6 TB/s), 4 us of it
// the second launch; one row of 8192 FP16 3.5 us.
#include <algorithm>

#include "layer_types.h"

namespace hpcdnn {

constexpr int kNormRowWaves = 4;     // rows per workgroup where a wave takes a row of its own
constexpr int kNormMaxWaves = 16;

// Parameters of the thread's columns in FP32; `fill` where there are none (and behind the last column).
template <class T, class W, int NV, row_kind kKind>
__device__ __forceinline__ void load_params(const W* p, float fill, const row_values<T, NV, kKind>& s, int cols, float (&out)[NV][kVec<T>]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) out[v][i] = fill;
        if (p == nullptr) continue;
        if constexpr (kKind == kSingleRows) {
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i)
                if (s.own(v, i)) out[v][i] = static_cast<float>(p[s.column(v, i)]);
        } else {
#pragma unroll
            for (int i = 0; i < kVec<T>; i += kVec<W>) {
                if (s.column(v, i) >= cols) continue;
                float f[kVec<W>];
                unpack<W>(load_row(p, s.column(v, i), cols), f);
#pragma unroll
                for (int k = 0; k < kVec<W>; ++k) out[v][i + k] = f[k];
            }
        }
    }
}

// One row per wave (kWaveRow: no exchange between waves) or per workgroup.  The mean and the squared deviations of a
// wave's part of the row are formed in two passes over registers, the parts then joined,
//   mu = mu_0 + sum n_w (mu_w - mu_0) / C,   M2 = sum M2_w + n_w (mu_w - mu)^2,
// so nothing cancels (sum x^2 - C mu^2 would lose the variance of rows with a large mean) and a row costs one barrier.
// A sum of equal FP32 values rounds, and its mean may be some steps beside them; their deviations from it are exact and few
// steps large, so these add up exactly, and the mean is moved by what they leave: a row of equal values has exactly
// that mean, and no spread.  (16-bit values have room in the sum of a wave, and only the join needs its shift by mu_0.)
// The next row is loaded into the registers of the present one as soon as that is unpacked.
template <class T, class W, int NV, bool kWaveRow, row_kind kKind>
__global__ __launch_bounds__(kWaveRow ? kNormRowWaves * kWave : 1024) void layer_norm_kernel(
    int64_t rows, int cols, const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, const W* __restrict__ b, float eps,
    T* __restrict__ y, int64_t ldy, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float part[2][2][kNormMaxWaves];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int waves = blockDim.x / kWave;
    const int64_t step = kWaveRow ? static_cast<int64_t>(gridDim.x) * kNormRowWaves : gridDim.x;
    int64_t r = kWaveRow ? static_cast<int64_t>(blockIdx.x) * kNormRowWaves + wave : blockIdx.x;
    if (r >= rows) return;
    row_values<T, NV, kKind> cur(kWaveRow ? lane : threadIdx.x, kWaveRow ? kWave : blockDim.x, cols);
    cur.load(x, ldx, r, rows);
    loads_start_here();
    float wf[NV][kVec<T>], bf[NV][kVec<T>];
    load_params<T, W, NV, kKind>(w, 1.f, cur, cols, wf);
    load_params<T, W, NV, kKind>(b, 0.f, cur, cols, bf);
    int valid = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) valid += cur.own(v, i);
    const float n_wave = wave_allsum(static_cast<float>(valid));  // at least one
    const float n_cols = static_cast<float>(cols);
    // v / n.  16-bit rows divide: their wave's sum of equal values is exact, and then so is its mean.  FP32 rows multiply, which
    // makes up for the sum that corrects their mean (16384 x 4096 84.0 us with and without it, 85.8 with it and divisions).
    const float inv_wave = 1.f / n_wave, inv_cols = 1.f / n_cols;
    auto over = [](float v, float n, float inv) { return std::is_same_v<T, float> ? v * inv : v / n; };
    // columns of wave (lane & 15): what the join below weighs that wave's mean with
    float n_of_lane = 0.f;
    if (!kWaveRow) {
        if (lane == 0) part[1][0][wave] = n_wave;
        __syncthreads();
        n_of_lane = (lane & 15) < waves ? part[1][0][lane & 15] : 0.f;
    }

    for (int turn = 0; r < rows; r += step, turn ^= 1) {
        float f[NV][kVec<T>], sum = 0.f;
        cur.get(f);
        cur.load(x, ldx, r + step, rows);
        loads_start_here();
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) sum += kKind != kOverlapRows || cur.own(v, i) ? f[v][i] : 0.f;  // (zeros behind the end)
        float mu = over(wave_allsum(sum), n_wave, inv_wave), m2 = 0.f;
        [[maybe_unused]] float left = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) {
                const float d = cur.own(v, i) ? f[v][i] - mu : 0.f;
                m2 = __builtin_fmaf(d, d, m2);
                if constexpr (std::is_same_v<T, float>) left += d;
            }
        m2 = wave_allsum(m2);
        if constexpr (std::is_same_v<T, float>) {
            left = wave_allsum(left);
            const float shift = left * inv_wave;
            if (__builtin_fabsf(left) < __builtin_inff()) {  // (beside an infinity there is nothing to move)
                mu += shift;
                m2 = __builtin_fmaxf(__builtin_fmaf(-left, shift, m2), 0.f);
            }
        }
        if (!kWaveRow) {
            if (lane == 0) {
                part[turn][0][wave] = mu;
                part[turn][1][wave] = m2;
            }
            __syncthreads();
            const bool has = (lane & 15) < waves;
            const float mu_0 = part[turn][0][0];
            const float mu_w = has ? part[turn][0][lane & 15] : 0.f, m2_w = has ? part[turn][1][lane & 15] : 0.f;
            mu = mu_0 + over(row16_allsum(n_of_lane * (mu_w - mu_0)), n_cols, inv_cols);
            if (!(__builtin_fabsf(mu) < __builtin_inff())) mu = row16_allsum(n_of_lane * mu_w) / n_cols;  // the mean of a row with an infinity is one
            m2 = row16_allsum(__builtin_fmaf(n_of_lane * (mu_w - mu), mu_w - mu, m2_w));
        }
        const float rs = 1.f / __builtin_sqrtf(over(m2, n_cols, inv_cols) + eps);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) f[v][i] = __builtin_fmaf((f[v][i] - mu) * rs, wf[v][i], bf[v][i]);
        row_values<T, NV, kKind> out(cur.t, cur.n, cols);
        out.set(f);
        out.store(y, ldy, r, rows);
        if ((kWaveRow ? lane : static_cast<int>(threadIdx.x)) == 0) {
            if (mean != nullptr) mean[r] = mu;
            if (rstd != nullptr) rstd[r] = rs;
        }
    }
}

// Gradient.  A workgroup is several teams of `row_waves` waves, each with a row at a time: rows (workgroup, team), then
// every grid * teams further.  A thread adds dy xh and dy of its columns in registers; the teams' sums are joined in LDS in
// their order at the end, and the workgroup writes one partial row of each, [workgroup][2][cols] in the workspace, added in
// the workgroups' order by layer_norm_params_kernel.  So dw and db do not depend on timing, and with sixteen waves to a
// workgroup the partial rows stay few: they are the only traffic beside x, dy and dx.
template <class T, class W, int NV, bool kWaveRow, row_kind kKind>
__global__ __launch_bounds__(1024) void layer_norm_grad_kernel(
    int64_t rows, int cols, int row_waves, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
    const W* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t lddx,
    float* __restrict__ partial) {
    __shared__ float part[2][2][kNormMaxWaves];
    extern __shared__ float joined[];  // [2][values of a thread][pitch] where there are several teams
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (kWaveRow) row_waves = 1;
    const int teams = (blockDim.x / kWave) / row_waves, team = kWaveRow ? wave : __builtin_amdgcn_readfirstlane(wave / row_waves);
    const int first_wave = team * row_waves;
    const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
    const int64_t block_row = static_cast<int64_t>(blockIdx.x) * teams;
    int64_t r = block_row + team;
    row_values<T, NV, kKind> cx((wave - first_wave) * kWave + lane, row_waves * kWave, cols), cd(cx.t, cx.n, cols);
    const float inv_cols = 1.f / static_cast<float>(cols);
    constexpr bool kKeep = NV * kVec<T> <= 8;  // w in registers; wider rows read it again (from L2), or they would spill (FP32 beyond 8192 columns does, 7 registers)
    float wf[NV][kVec<T>], dw[NV][kVec<T>], db[NV][kVec<T>];
    if (kKeep) load_params<T, W, NV, kKind>(w, 1.f, cx, cols, wf);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < kVec<T>; ++i) dw[v][i] = db[v][i] = 0.f;
    float next_mu, next_rs;
    // The statistics come as vector loads too: a scalar load in flight would be waited for with the LDS accesses of the
    // exchange between the waves, which share its counter.
    auto load = [&](int64_t row) {
        const bool is = row < rows;
        cx.load(x, ldx, row, rows);
        cd.load(dy, lddy, row, rows);
        const int64_t at = is ? row : rows - 1;
        next_mu = buffer_load_f(make_rsrc(mean + at, kKind == kOverlapRows || is ? 4 : 0), 0);
        next_rs = buffer_load_f(make_rsrc(rstd + at, kKind == kOverlapRows || is ? 4 : 0), 0);
        loads_start_here();
    };
    load(r);
    int turn = 0;
    // all teams walk as long as the first has rows: the barrier is the workgroup's
    for (int64_t lead = block_row; lead < rows; lead += step, r += step, turn ^= 1) {
        // into scalar registers, so that the next row's can be on their way in these
        const float mu = wave_first(next_mu), rs = wave_first(next_rs);
        float g_sum = 0.f, gx_sum = 0.f;
        float xh[NV][kVec<T>], g[NV][kVec<T>];
        cx.get(xh);
        cd.get(g);
        if (!kKeep) load_params<T, W, NV, kKind>(w, 1.f, cx, cols, wf);
        load(r + step);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) {
                xh[v][i] = (xh[v][i] - mu) * rs;
                // A team without a row in the last turn must add nothing: it has zeros, or else (kOverlapRows) the last row.
                if (kKind != kOverlapRows || r < rows) {
                    dw[v][i] = __builtin_fmaf(g[v][i], xh[v][i], dw[v][i]);
                    db[v][i] += g[v][i];
                }
                g[v][i] *= wf[v][i];
                const float term = kKind != kOverlapRows || cx.own(v, i) ? g[v][i] : 0.f;
                g_sum += term;
                gx_sum = __builtin_fmaf(term, xh[v][i], gx_sum);
            }
        g_sum = wave_allsum(g_sum);
        gx_sum = wave_allsum(gx_sum);
        if (!kWaveRow) {
            if (lane == 0) {
                part[turn][0][wave] = g_sum;
                part[turn][1][wave] = gx_sum;
            }
            __syncthreads();
            const bool has = (lane & 15) < row_waves;
            g_sum = row16_allsum(has ? part[turn][0][first_wave + (lane & 15)] : 0.f);
            gx_sum = row16_allsum(has ? part[turn][1][first_wave + (lane & 15)] : 0.f);
        }
        const float a = g_sum * inv_cols, c = gx_sum * inv_cols;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) g[v][i] = rs * (g[v][i] - a - xh[v][i] * c);
        row_values<T, NV, kKind> out(cx.t, cx.n, cols);
        out.set(g);
        if (kKind != kOverlapRows || dx != nullptr) out.store(dx, lddx, r, dx != nullptr ? rows : 0);
    }
    if (partial == nullptr) return;
    float* out = partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
    if (teams == 1) {
        // 16 bytes at a time (value by value, 392 x 15808 BF16 took 35.4 us instead of 21.5); what vectors share at the end of
        // a row (kOverlapRows) is stored twice with the same value here too
        const row_buffer<float, true> to_w(out, cols), to_b(out + cols, cols);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < kVec<T>; i += 4) {
                to_w.store16(cx.column(v, i), __builtin_bit_cast(v4u, v4f{dw[v][i], dw[v][i + 1], dw[v][i + 2], dw[v][i + 3]}));
                to_b.store16(cx.column(v, i), __builtin_bit_cast(v4u, v4f{db[v][i], db[v][i + 1], db[v][i + 2], db[v][i + 3]}));
            }
        return;
    }
    // value i of thread t of a team at i * pitch + t, dw and db in turn: neither the threads nor, with a pitch of 8 mod 64,
    // the walk over the columns below meet a bank twice
    const int n = cx.n, pitch = n + 8;
    for (int k = 0; k < teams; ++k) {
        if (k == team) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < kVec<T>; ++i) {
                    float* a = joined + (v * kVec<T> + i) * pitch + cx.t;
                    float* b = a + NV * kVec<T> * pitch;
                    *a = k == 0 ? dw[v][i] : *a + dw[v][i];
                    *b = k == 0 ? db[v][i] : *b + db[v][i];
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
        int value = c / n, thread = c - value * n;
        if (kKind != kSingleRows) {
            const int vec = c / kVec<T>, v = vec / n;
            const int at = kKind == kOverlapRows ? min(vec * kVec<T>, cols - kVec<T>) : vec * kVec<T>;
            value = v * kVec<T> + c - at;
            thread = vec - v * n;
        }
        const float* a = joined + value * pitch + thread;
        out[c] = a[0];
        out[cols + c] = a[NV * kVec<T> * pitch];
    }
}

// dw[c], db[c] = the partial rows added in order: 32 columns by 32 runs of consecutive partial rows per workgroup, the
// runs added in order.  Few enough columns for a handful of workgroups, so the rows are what is spread over the threads.
constexpr int kParamsRuns = 32;
template <class W>
__global__ __launch_bounds__(32 * kParamsRuns) void layer_norm_params_kernel(int parts, int cols, const float* __restrict__ partial,
                                                                             W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float run[kParamsRuns][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x / 32;
    const int per = (parts + kParamsRuns - 1) / kParamsRuns;
    const int first = k * per, last = min(parts, first + per);
    float sum = 0.f;
    if (c < 2 * cols) {
        constexpr int kBatch = 16;
        for (int p = first; p < last; p += kBatch) {
            float t[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) t[u] = p + u < last ? partial[static_cast<int64_t>(p + u) * 2 * cols + c] : 0.f;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) sum += t[u];
        }
    }
    run[k][threadIdx.x & 31] = sum;
    __syncthreads();
    if (k != 0 || c >= 2 * cols) return;
#pragma unroll
    for (int u = 1; u < kParamsRuns; ++u) sum += run[u][threadIdx.x];
    if (c < cols) {
        if (dw != nullptr) dw[c] = static_cast<W>(sum);
    } else if (db != nullptr) {
        db[c - cols] = static_cast<W>(sum);
    }
}

namespace {

// A row's vectors over the lanes: a wave of its own while two vectors per lane hold it, else one workgroup of up to 1024
// threads with one, two or four vectors per thread.
struct norm_shape {
    bool wave_row;
    int nv, threads;
};
norm_shape shape_of(int cols, int vec, int least_nv = 1) {
    const int vecs = static_cast<int>(ceil_div(cols, vec));
    if (vecs <= 2 * kWave) return {true, vecs <= kWave ? 1 : 2, kNormRowWaves * kWave};
    const int nv = std::max(least_nv, vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 4);
    return {false, nv, static_cast<int>(ceil_div(ceil_div(vecs, nv), kWave)) * kWave};
}

// Most workgroups of the gradient, each of which leaves a partial row of dw and db: one per CU, whatever the type.  (Two per
// CU measured 2 % faster for 30000 x 512 BF16, but 5 to 11 % slower from 2048 columns on: the partial rows double.)
int grad_blocks(int rows) { return std::min(rows, device_cus()); }

// f(NV, kWaveRow, kKind) as compile-time constants
template <class T, class F>
void with_shape(const norm_shape& s, row_kind kind, F&& f) {
    using std::integral_constant;
    auto more = [&](auto nv, auto wave_row) {
        if constexpr (sizeof(T) == 2)
            if (kind != kDwordRows) return f(nv, wave_row, integral_constant<row_kind, kOverlapRows>{});
        f(nv, wave_row, integral_constant<row_kind, kDwordRows>{});
    };
    if constexpr (sizeof(T) == 2)
        if (kind == kSingleRows) return f(integral_constant<int, 1>{}, std::true_type{}, integral_constant<row_kind, kSingleRows>{});
    if (s.wave_row) {
        if (s.nv == 1) more(integral_constant<int, 1>{}, std::true_type{});
        else more(integral_constant<int, 2>{}, std::true_type{});
    } else if (s.nv == 1) more(integral_constant<int, 1>{}, std::false_type{});
    else if (s.nv == 2) more(integral_constant<int, 2>{}, std::false_type{});
    else if constexpr (kVec<T> == 4) more(integral_constant<int, 4>{}, std::false_type{});
}

template <class T, class W>
int launch_norm(int rows, int cols, const void* x, int64_t ldx, const void* w, const void* b, float eps, void* y, int64_t ldy,
                float* mean, float* rstd, hipStream_t stream) {
    const norm_shape s = shape_of(cols, kVec<T>);
    const int64_t blocks = s.wave_row ? ceil_div(rows, kNormRowWaves) : rows;
    const int64_t most = static_cast<int64_t>(device_cus()) * (2048 / s.threads);
    const int grid = static_cast<int>(blocks < most ? blocks : most);
    const row_kind kind = kind_of(rows_are_dwords(x, ldx, cols, sizeof(T)) && rows_are_dwords(y, ldy, cols, sizeof(T)), cols);
    with_shape<T>(s, kind, [&](auto nv, auto wave_row, auto rows_kind) {
        layer_norm_kernel<T, W, decltype(nv)::value, decltype(wave_row)::value, decltype(rows_kind)::value><<<grid, s.threads, 0, stream>>>(
            rows, cols, static_cast<const T*>(x), ldx, static_cast<const W*>(w), static_cast<const W*>(b), eps, static_cast<T*>(y), ldy,
            mean, rstd);
    });
    return launch_status();
}

template <class T, class W>
int launch_grad(int rows, int cols, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const float* mean,
                const float* rstd, void* dx, int64_t lddx, void* dw, void* db, float* partial, hipStream_t stream) {
    norm_shape s = shape_of(cols, kVec<T>);
    // Nine or ten waves to a row leave a CU's workgroup at that; with two vectors per thread it is three teams of five.  Only
    // many rows make up for the longer turn: 5000 x 5001 BF16 41 us instead of 49, 16384 x 4160 91 instead of 99, but
    // 1000 x 5000 17.2 instead of 16.3.
    if (!s.wave_row && s.nv == 1 && s.threads > 8 * kWave && s.threads <= 10 * kWave && rows >= 8 * device_cus())
        s = shape_of(cols, kVec<T>, 2);
    const int row_waves = s.wave_row ? 1 : s.threads / kWave;
    const int teams = s.wave_row ? 8 : kNormMaxWaves / row_waves;
    // as many as make the same number of turns: no partial row is written for less (300 x 8192 BF16 13.6 us, with one
    // workgroup per CU 15.7)
    const int64_t per_turn = static_cast<int64_t>(std::max(1, grad_blocks(rows))) * teams;
    const int grid = rows > 0 ? static_cast<int>(ceil_div(rows, ceil_div(rows, per_turn) * teams)) : 0;
    if (grid > 0) {
        const size_t lds = teams > 1 && partial ? 2 * sizeof(float) * s.nv * kVec<T> * (row_waves * kWave + 8) : 0;
        const bool all_dwords = rows_are_dwords(x, ldx, cols, sizeof(T)) && rows_are_dwords(dy, lddy, cols, sizeof(T)) &&
                                (dx == nullptr || rows_are_dwords(dx, lddx, cols, sizeof(T)));
        with_shape<T>(s, kind_of(all_dwords, cols), [&](auto nv, auto wave_row, auto rows_kind) {
            layer_norm_grad_kernel<T, W, decltype(nv)::value, decltype(wave_row)::value, decltype(rows_kind)::value>
                <<<grid, teams * row_waves * kWave, lds, stream>>>(
                    rows, cols, row_waves, static_cast<const T*>(dy), lddy, static_cast<const T*>(x), ldx, static_cast<const W*>(w), mean,
                    rstd, static_cast<T*>(dx), lddx, partial);
        });
        if (int e = launch_status()) return e;
    }
    if (partial != nullptr || (grid == 0 && (dw || db)))
        layer_norm_params_kernel<W><<<static_cast<int>(ceil_div(2 * static_cast<int64_t>(cols), 32)), 32 * kParamsRuns, 0, stream>>>(
            grid, cols, partial, static_cast<W*>(dw), static_cast<W*>(db));
    return launch_status();
}

bool args_valid(int type, int wtype, int rows, int cols) {
    return type_valid(type) && (wtype == HPCDNN_F32 || wtype == type) && rows >= 0 && cols >= 0 && cols <= HPCDNN_LAYER_NORM_MAX_COLS;
}
bool matrix_valid(const void* p, int64_t ld, int cols, int type) { return p != nullptr && ld >= cols && aligned(p, type_bytes(type)); }
bool params_valid(const void* p, int wtype) { return aligned(p, type_bytes(wtype)); }

// f(T*, W*) with the types of the rows and of the parameters
template <class F>
int with_types(int type, int wtype, F&& f) {
    return with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if constexpr (!std::is_same_v<T, float>)
            if (wtype == type) return f(t, t);
        return f(t, static_cast<float*>(nullptr));
    });
}

}  // namespace

size_t layer_norm_grad_workspace_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return static_cast<size_t>(grad_blocks(rows)) * 2 * cols * sizeof(float);
}

}  // namespace hpcdnn

extern "C" int hpcdnn_layer_norm(int type, int wtype, int rows, int cols, const void* x, int64_t ldx, const void* w, const void* b,
                                 float eps, void* y, int64_t ldy, float* mean, float* rstd, void* stream) {
    using namespace hpcdnn;
    if (!args_valid(type, wtype, rows, cols) || !(eps >= 0.f)) return HPCDNN_ERR_INVALID_VALUE;
    if (rows == 0 || cols == 0) return HPCDNN_OK;
    if (!matrix_valid(x, ldx, cols, type) || !matrix_valid(y, ldy, cols, type) || !params_valid(w, wtype) || !params_valid(b, wtype) ||
        !aligned(mean, 4) || !aligned(rstd, 4))
        return HPCDNN_ERR_INVALID_VALUE;
    return with_types(type, wtype, [&](auto* t, auto* p) {
        return launch_norm<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(p)>>(
            rows, cols, x, ldx, w, b, eps, y, ldy, mean, rstd, static_cast<hipStream_t>(stream));
    });
}

extern "C" int hpcdnn_layer_norm_grad(int type, int wtype, int rows, int cols, const void* dy, int64_t lddy, const void* x,
                                      int64_t ldx, const void* w, const float* mean, const float* rstd, void* dx, int64_t lddx, void* dw,
                                      void* db, void* ws, size_t ws_bytes, void* stream) {
    using namespace hpcdnn;
    if (!args_valid(type, wtype, rows, cols)) return HPCDNN_ERR_INVALID_VALUE;
    if (cols == 0 || (dx == nullptr && dw == nullptr && db == nullptr)) return HPCDNN_OK;
    if (!params_valid(w, wtype) || !params_valid(dw, wtype) || !params_valid(db, wtype)) return HPCDNN_ERR_INVALID_VALUE;
    const bool params = dw != nullptr || db != nullptr;
    if (rows > 0) {
        if (!matrix_valid(dy, lddy, cols, type) || !matrix_valid(x, ldx, cols, type) || (dx && !matrix_valid(dx, lddx, cols, type)) ||
            mean == nullptr || rstd == nullptr || !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(ws, 16))
            return HPCDNN_ERR_INVALID_VALUE;
        if (params && (ws == nullptr || ws_bytes < layer_norm_grad_workspace_bytes(rows, cols))) return HPCDNN_ERR_WORKSPACE;
    }
    return with_types(type, wtype, [&](auto* t, auto* p) {
        return launch_grad<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(p)>>(
            rows, cols, dy, lddy, x, ldx, w, mean, rstd, dx, lddx, dw, db, params && rows > 0 ? static_cast<float*>(ws) : nullptr,
            static_cast<hipStream_t>(stream));
    });
}
