// Tokens sorted by the expert they are sent to, their rows copied there and summed back with the router's weights, and
// the gradient of that sum.  With topk choices per token, slot s = t * topk + j is choice j of token t:
//
//   sort     stable by expert: pos[s] = place of slot s (-1: sent nowhere), order[pos[s]] = s, offsets[e] = first place of e
//   gather   out[pos[s]] = x[t]
//   combine  y[t] = sum_j w[s] xs[pos[s]]                      (with w = 1: the gradient of gather)
//   gradient dxs[pos[s]] = w[s] dy[t],  dw[s] = <dy[t], xs[pos[s]]>
//
// Everything goes token by token, so a token's row is read (or written) once and the topk rows once each: bound by memory.
// Measured with 4096 columns in BF16, 16384 tokens of two choices: sort 6 us in two launches, gather 66 us (6.1 TB/s of which
// two thirds are writes); combine of 8191 x 4 rows of 1001 FP32 31 us (5.3 TB/s); its gradient of 8192 x 2 rows of 6144 BF16
// 93 us (5.1 TB/s).  32 tokens of eight choices: sort 3.0 us, gather 3.4 us.
#include <algorithm>

#include "layer_types.h"

namespace hpcdnn {

// ---- sort -----------------------------------------------------------------

constexpr int kSortMaxThreads = 1024;
constexpr int kSortOneBlock = 4096;  // slots up to which one workgroup sorts them in one launch
constexpr int kSortMinSlots = 1024;  // slots of a workgroup beyond that, more where there would be over kSortMaxBlocks
constexpr int kSortMaxBlocks = 128;  // (every one of them reads the counts of all)

// Expert of slot s; slots of a row-contiguous list lie one after the other, and the division is spared.
__device__ __forceinline__ int expert_of(const int* __restrict__ ids, int64_t ldids, unsigned s, unsigned topk) {
    if (ldids == topk) return ids[s];
    const unsigned t = s / topk;
    return ids[t * ldids + (s - t * topk)];
}

// Lanes of the wave that hold the same key as this one, among those with `on`: one ballot per bit of the key.
__device__ __forceinline__ uint64_t same_key(int key, bool on, int bits) {
    uint64_t m = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t one = __ballot((key >> b) & 1);
        m &= ((key >> b) & 1) ? one : ~one;
    }
    return m;
}

// counts[block][e] = slots of the workgroup's chunk that go to expert e
__global__ __launch_bounds__(kSortMaxThreads) void expert_count_kernel(unsigned slots, unsigned per_block, int topk, int experts,
                                                                       const int* __restrict__ ids, int64_t ldids, int* __restrict__ counts) {
    __shared__ int hist[HPCDNN_EXPERTS_MAX];
    for (int e = threadIdx.x; e < experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const unsigned first = blockIdx.x * per_block, last = min(slots, first + per_block);
    for (unsigned s = first + threadIdx.x; s < last; s += blockDim.x) {
        const int id = expert_of(ids, ldids, s, topk);
        if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[blockIdx.x * experts + e] = hist[e];
}

// Places of the workgroup's slots.  Every workgroup adds up the counts of all workgroups by itself (they come from L2), so
// there is no launch for a scan; counts == nullptr: one workgroup has all the slots.  Within the workgroup each wave has a
// run of consecutive slots: it counts them per expert, the counts are scanned over waves, and in a second walk a slot's
// place is the wave's next place for its expert plus the number of earlier lanes with the same expert.  Integer sums only,
// so the order of the LDS additions does not show.  The workgroup has at least as many threads as there are experts.
__global__ __launch_bounds__(kSortMaxThreads) void expert_place_kernel(unsigned slots, unsigned per_block, int topk, int experts, int bits,
                                                                       const int* __restrict__ ids, int64_t ldids,
                                                                       const int* __restrict__ counts, int blocks, int* __restrict__ offsets,
                                                                       int* __restrict__ pos, int* __restrict__ order) {
    extern __shared__ int lds[];
    const int waves = blockDim.x / kWave;
    int* next = lds;                          // [waves][experts] counts, then next places
    int* before = lds + waves * experts;      // [experts] slots of earlier workgroups
    int* total = before + experts;            // [experts] slots of all workgroups
    __shared__ int wave_total[kSortMaxThreads / kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned first = blockIdx.x * per_block, last = min(slots, first + per_block);
    const unsigned per_wave = per_block / waves;  // a multiple of 64
    const unsigned begin = first + wave * per_wave, end = min(last, begin + per_wave);
    // the first 64 slots' experts are on their way while LDS is cleared
    int id0 = begin + lane < end ? expert_of(ids, ldids, begin + lane, topk) : -1;
    for (int i = threadIdx.x; i < (waves + 2) * experts; i += blockDim.x) lds[i] = 0;
    __syncthreads();
    if (id0 >= 0 && id0 < experts) atomicAdd(&next[wave * experts + id0], 1);
    for (unsigned s = begin + kWave + lane; s < end; s += kWave) {
        const int id = expert_of(ids, ldids, s, topk);
        if (id >= 0 && id < experts) atomicAdd(&next[wave * experts + id], 1);
    }
    if (counts != nullptr) {
        // threads (share of the workgroups, expert)
        const int e = threadIdx.x & ((1 << bits) - 1), shares = blockDim.x >> bits, share = threadIdx.x >> bits;
        if (e < experts && share < shares) {
            int all = 0, earlier = 0;
            // eight loads on their way at a time: 83968 choices of 223 experts 8.8 us, one after the other 12.3
            for (int b0 = share; b0 < blocks; b0 += 8 * shares) {
                int c[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) c[u] = b0 + u * shares < blocks ? counts[(b0 + u * shares) * experts + e] : 0;
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    all += c[u];
                    if (b0 + u * shares < static_cast<int>(blockIdx.x)) earlier += c[u];
                }
            }
            atomicAdd(&total[e], all);
            atomicAdd(&before[e], earlier);
        }
    }
    __syncthreads();
    // exclusive scan of the totals over the experts, one per thread, and of the waves' counts
    const int e = threadIdx.x;
    int mine = 0;
    if (e < experts) {
        int sum = 0;
        for (int w = 0; w < waves; ++w) sum += next[w * experts + e];
        mine = counts != nullptr ? total[e] : sum;
    }
    int scan = mine;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int v = __shfl_up(scan, d);
        if (lane >= d) scan += v;
    }
    if (lane == kWave - 1) wave_total[wave] = scan;
    __syncthreads();
    for (int w = 0; w < wave; ++w) scan += wave_total[w];
    if (e < experts) {
        int place = scan - mine + before[e];
        for (int w = 0; w < waves; ++w) {
            const int n = next[w * experts + e];
            next[w * experts + e] = place;
            place += n;
        }
        if (blockIdx.x == 0) {
            offsets[e] = scan - mine;
            if (e == experts - 1) offsets[experts] = scan;
        }
    }
    __syncthreads();
    for (unsigned s0 = begin; s0 < end; s0 += kWave) {
        const unsigned s = s0 + lane;
        const int id = s0 == begin ? id0 : s < end ? expert_of(ids, ldids, s, topk) : -1;
        const bool sent = id >= 0 && id < experts;
        const uint64_t peers = same_key(id, sent, bits);
        const int rank = __popcll(peers & ((1ull << lane) - 1));
        int place = -1;
        if (sent) place = next[wave * experts + id] + rank;
        __builtin_amdgcn_wave_barrier();  // all lanes have read their place before the leaders move it on
        if (sent && rank == 0) next[wave * experts + id] = place + __popcll(peers);
        __builtin_amdgcn_wave_barrier();
        if (s < end) pos[s] = place;
        if (sent && order != nullptr) order[place] = static_cast<int>(s);
    }
}

// ---- rows to their places and back ------------------------------------------

constexpr int kRowWaves = 4;  // waves of a workgroup

// A workgroup is one or more teams of `team_waves` waves, each with a token at a time: narrow rows leave no lanes idle.  A team
// takes a strip of a vector per thread of a row.
struct row_team {
    int lane, wave, waves, first_wave, team, teams, threads, thread;
    __device__ __forceinline__ explicit row_team(int team_waves) {
        lane = threadIdx.x & (kWave - 1);
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        waves = team_waves;
        team = __builtin_amdgcn_readfirstlane(wave / team_waves);
        teams = __builtin_amdgcn_readfirstlane(blockDim.x / kWave / team_waves);
        first_wave = team * team_waves;
        threads = team_waves * kWave;
        thread = (wave - first_wave) * kWave + lane;
    }
};

// A choice's row, or zeros where it has none: through a descriptor without a branch.
template <class T, row_kind kKind>
__device__ __forceinline__ void load_or_clear(row_values<T, 1, kKind>& v, const T* m, int64_t ld, int row, int rows, bool is) {
    if constexpr (kKind == kOverlapRows) {
        if (is) v.load(m, ld, row, rows);
        else v.clear();
    } else {
        v.load(m, ld, is ? row : rows, rows);
    }
}

// First column of a strip.  A strip that is cut short is a row of its own: it may be shorter than a vector, which kOverlapRows
// cannot have, so there the last strip is moved back to end with the row instead.
template <class T, row_kind kKind>
__device__ __forceinline__ int strip_start(int strip, int width, int cols) {
    const int first = strip * width;
    return kKind == kOverlapRows ? max(0, min(first, cols - width)) : first;
}

// out[pos[t][j]] = x[t].
template <class T, row_kind kKind>
__global__ __launch_bounds__(kRowWaves * kWave) void expert_gather_kernel(int tokens, int topk, int rows, int cols, int team_waves,
                                                                          const T* __restrict__ x, int64_t ldx, const int* __restrict__ pos,
                                                                          T* __restrict__ out, int64_t ldout) {
    const row_team m(team_waves);
    const int width = m.threads * kVec<T>, first = strip_start<T, kKind>(blockIdx.y, width, cols), here = min(cols - first, width);
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * m.teams + m.team; t < tokens; t += static_cast<int64_t>(gridDim.x) * m.teams) {
        row_values<T, 1, kKind> v(m.thread, m.threads, here);
        v.load(x + first, ldx, t, tokens);
        for (int j = 0; j < topk; ++j) {
            const int p = pos[t * topk + j];
            if (p >= 0 && p < rows) v.store(out + first, ldout, p, rows);
        }
    }
}

// y[t] = sum_j w[t][j] xs[pos[t][j]], added in FP32 in the order of j.  Four rows are on their way at a time: of one token, or
// of four where each has a single choice, so that a team does not wait for one row after the other.
template <class T, row_kind kKind, int kTokens>
__global__ __launch_bounds__(kRowWaves * kWave) void expert_combine_kernel(int tokens, int topk, int rows, int cols, int team_waves,
                                                                           const T* __restrict__ xs, int64_t ldxs, const int* __restrict__ pos,
                                                                           const float* __restrict__ weights, T* __restrict__ y, int64_t ldy) {
    constexpr int kBatch = 4 / kTokens;
    const row_team m(team_waves);
    const int width = m.threads * kVec<T>, first = strip_start<T, kKind>(blockIdx.y, width, cols), here = min(cols - first, width);
    const int64_t step = static_cast<int64_t>(gridDim.x) * m.teams * kTokens;
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * m.teams + m.team) * kTokens; t0 < tokens; t0 += step) {
        float acc[kTokens][1][kVec<T>];
#pragma unroll
        for (int k = 0; k < kTokens; ++k)
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) acc[k][0][i] = 0.f;
        row_values<T, 1, kKind> sum(m.thread, m.threads, here);
        for (int j0 = 0; j0 < topk; j0 += kBatch) {
            row_values<T, 1, kKind> v[4] = {sum, sum, sum, sum};
            float w[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int64_t t = t0 + b / kBatch;
                const int j = j0 + b % kBatch;
                const int64_t s = min(t, static_cast<int64_t>(tokens) - 1) * topk + min(j, topk - 1);
                const int p = pos[s];
                const bool is = t < tokens && j < topk && p >= 0 && p < rows;  // else zeros, which weigh nothing whatever the weight
                w[b] = !is ? 0.f : weights != nullptr ? weights[s] : 1.f;
                load_or_clear(v[b], xs + first, ldxs, p, rows, is);
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float f[1][kVec<T>];
                v[b].get(f);
#pragma unroll
                for (int i = 0; i < kVec<T>; ++i) acc[b / kBatch][0][i] = __builtin_fmaf(w[b], f[0][i], acc[b / kBatch][0][i]);
            }
        }
#pragma unroll
        for (int k = 0; k < kTokens; ++k) {
            if (t0 + k >= tokens) break;
            sum.set(acc[k]);
            sum.store(y + first, ldy, t0 + k, tokens);
        }
    }
}

// dxs[pos[t][j]] = w[t][j] dy[t],  dw[t][j] = <dy[t], xs[pos[t][j]]>: a choice's dot product is added over the thread's
// columns, the lanes and the waves in that fixed order.  Choices go two at a time; few tokens' choices are spread over
// blockIdx.y.
constexpr int kGradBatch = 2;
template <class T, row_kind kKind>
__global__ __launch_bounds__(kRowWaves * kWave) void expert_combine_grad_kernel(int tokens, int topk, int rows, int cols, int team_waves,
                                                                          const T* __restrict__ dy, int64_t lddy,
                                                                          const T* __restrict__ xs, int64_t ldxs,
                                                                          const int* __restrict__ pos, const float* __restrict__ weights,
                                                                          T* __restrict__ dxs, int64_t lddxs, float* __restrict__ dweights) {
    __shared__ float part[2][kGradBatch][kRowWaves];
    const row_team m(team_waves);
    const int width = m.threads * kVec<T>;
    int turn = 0;
    // all teams walk as long as the first has tokens: the barrier is the workgroup's
    for (int64_t lead = static_cast<int64_t>(blockIdx.x) * m.teams; lead < tokens; lead += static_cast<int64_t>(gridDim.x) * m.teams)
        for (int j0 = kGradBatch * blockIdx.y; j0 < topk; j0 += kGradBatch * gridDim.y, turn ^= 1) {
            const int64_t t = min(lead + m.team, static_cast<int64_t>(tokens) - 1);
            const bool has_token = lead + m.team < tokens;
            int p[kGradBatch];
            float w[kGradBatch], dot[kGradBatch];
            bool is[kGradBatch], any = false;
#pragma unroll
            for (int b = 0; b < kGradBatch; ++b) {
                const int64_t s = t * topk + min(j0 + b, topk - 1);
                p[b] = pos[s];
                is[b] = has_token && j0 + b < topk && p[b] >= 0 && p[b] < rows;
                w[b] = !is[b] ? 0.f : weights != nullptr ? weights[s] : 1.f;
                dot[b] = 0.f;
                any |= is[b];
            }
            if (any)
                for (int strip = 0; strip * width < cols; ++strip) {
                    const int first = strip_start<T, kKind>(strip, width, cols), here = min(cols - first, width);
                    row_values<T, 1, kKind> g(m.thread, m.threads, here), v[kGradBatch] = {g, g};
                    g.load(dy + first, lddy, t, tokens);
#pragma unroll
                    for (int b = 0; b < kGradBatch; ++b) load_or_clear(v[b], xs + first, ldxs, p[b], rows, is[b] && dweights != nullptr);
                    float gf[1][kVec<T>];
                    g.get(gf);
#pragma unroll
                    for (int b = 0; b < kGradBatch; ++b) {
                        float f[1][kVec<T>];
                        v[b].get(f);
#pragma unroll
                        for (int i = 0; i < kVec<T>; ++i) {
                            // columns of its own, and none that an earlier strip had
                            const bool mine = kKind != kOverlapRows || (g.own(0, i) && first + g.column(0, i) >= strip * width);
                            dot[b] = __builtin_fmaf(mine ? gf[0][i] : 0.f, mine ? f[0][i] : 0.f, dot[b]);
                            f[0][i] = gf[0][i] * w[b];
                        }
                        v[b].set(f);
                        if (is[b] && dxs != nullptr) v[b].store(dxs + first, lddxs, p[b], rows);
                    }
                }
            if (dweights != nullptr) {
#pragma unroll
                for (int b = 0; b < kGradBatch; ++b) {
                    dot[b] = wave_allsum(dot[b]);
                    if (m.lane == 0) part[turn][b][m.wave] = dot[b];
                }
                __syncthreads();
                const int b = m.thread;
                if (b < kGradBatch && j0 + b < topk && has_token) {
                    float sum = part[turn][b][m.first_wave];
                    for (int k = 1; k < m.waves; ++k) sum += part[turn][b][m.first_wave + k];
                    dweights[t * topk + j0 + b] = is[b] ? sum : 0.f;
                }
            }
        }
}

namespace {

struct sort_plan {
    int blocks, threads;
    unsigned per_block;  // slots, a multiple of the threads
};
sort_plan plan_sort(int64_t slots, int experts) {
    if (slots <= kSortOneBlock) {
        // a wave per 64 slots up to sixteen, four at least and as many as the scan over the experts needs
        const int threads = static_cast<int>(std::min<int64_t>(kSortMaxThreads, std::max<int64_t>({ceil_div(slots, kWave), ceil_div(experts, kWave), 4}) * kWave));
        return {1, threads, static_cast<unsigned>(std::max<int64_t>(1, ceil_div(slots, threads)) * threads)};
    }
    const int64_t per = std::max<int64_t>(kSortMinSlots, ceil_div(ceil_div(slots, kSortMaxBlocks), kSortMaxThreads) * kSortMaxThreads);
    return {static_cast<int>(ceil_div(slots, per)), kSortMaxThreads, static_cast<unsigned>(per)};
}

bool choices_valid(int tokens, int topk) {
    return tokens >= 0 && topk >= 1 && topk <= HPCDNN_EXPERTS_MAX_TOPK && static_cast<int64_t>(tokens) * topk <= INT32_MAX;
}
bool rows_valid(const void* p, int64_t ld, int cols, int type) { return p != nullptr && ld >= cols && aligned(p, type_bytes(type)); }

// f(T*, kKind) with the type of the rows and how they are read
template <class F>
int with_rows(int type, row_kind kind, F&& f) {
    using std::integral_constant;
    return with_type(type, [&](auto* t) {
        if constexpr (sizeof(*t) == 2) {
            if (kind == kOverlapRows) return f(t, integral_constant<row_kind, kOverlapRows>{});
            if (kind == kSingleRows) return f(t, integral_constant<row_kind, kSingleRows>{});
        }
        return f(t, integral_constant<row_kind, kDwordRows>{});
    });
}

// Waves to a token and the launch: a vector per thread up to four waves, several tokens to a workgroup below that.
struct row_launch {
    int team_waves, threads;
    dim3 grid;
};
row_launch plan_rows(int64_t tokens, int cols, int vec, bool strips) {
    row_launch l;
    l.team_waves = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kRowWaves, ceil_div(cols, vec * kWave))));
    const int teams = kRowWaves / l.team_waves;
    l.threads = teams * l.team_waves * kWave;
    // (a launch holds fewer than 2^32 threads; the teams walk on from there)
    l.grid = dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(tokens, teams), 1 << 20)), strips ? static_cast<unsigned>(ceil_div(cols, vec * l.team_waves * kWave)) : 1u);
    return l;
}

}  // namespace

size_t expert_sort_workspace_bytes(int tokens, int topk, int experts) {
    if (!choices_valid(tokens, topk) || experts < 1 || experts > HPCDNN_EXPERTS_MAX) return 0;
    const sort_plan p = plan_sort(static_cast<int64_t>(tokens) * topk, experts);
    return p.blocks > 1 ? static_cast<size_t>(p.blocks) * experts * sizeof(int) : 0;
}

}  // namespace hpcdnn

extern "C" int hpcdnn_expert_sort(int tokens, int topk, int experts, const int32_t* ids, int64_t ldids, int32_t* offsets, int32_t* pos,
                                  int32_t* order, void* ws, size_t ws_bytes, void* stream_) {
    using namespace hpcdnn;
    if (!choices_valid(tokens, topk) || experts < 1 || experts > HPCDNN_EXPERTS_MAX || offsets == nullptr || !aligned(offsets, 4))
        return HPCDNN_ERR_INVALID_VALUE;
    if (tokens > 0 && (ids == nullptr || ldids < topk || pos == nullptr || !aligned(ids, 4) || !aligned(pos, 4) || !aligned(order, 4)))
        return HPCDNN_ERR_INVALID_VALUE;
    const int64_t slots = static_cast<int64_t>(tokens) * topk;
    const sort_plan p = plan_sort(slots, experts);
    if (p.blocks > 1) {
        if (!aligned(ws, 16)) return HPCDNN_ERR_INVALID_VALUE;
        if (ws == nullptr || ws_bytes < expert_sort_workspace_bytes(tokens, topk, experts)) return HPCDNN_ERR_WORKSPACE;
    }
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    int bits = 0;
    while ((1 << bits) < experts) ++bits;
    const size_t lds = static_cast<size_t>(p.threads / kWave + 2) * experts * sizeof(int);
    int* counts = nullptr;
    if (p.blocks > 1) {
        counts = static_cast<int*>(ws);
        expert_count_kernel<<<p.blocks, p.threads, 0, stream>>>(static_cast<unsigned>(slots), p.per_block, topk, experts, ids, ldids, counts);
    }
    expert_place_kernel<<<p.blocks, p.threads, lds, stream>>>(static_cast<unsigned>(slots), p.per_block, topk, experts, bits, ids, ldids,
                                                              counts, p.blocks, offsets, pos, order);
    return launch_status();
}

extern "C" int hpcdnn_expert_gather(int type, int tokens, int topk, int rows, int cols, const void* x, int64_t ldx, const int32_t* pos,
                                    void* out, int64_t ldout, void* stream) {
    using namespace hpcdnn;
    if (!type_valid(type) || !choices_valid(tokens, topk) || rows < 0 || cols < 0 || cols > HPCDNN_EXPERTS_MAX_COLS) return HPCDNN_ERR_INVALID_VALUE;
    if (tokens == 0 || rows == 0 || cols == 0) return HPCDNN_OK;
    if (!rows_valid(x, ldx, cols, type) || !rows_valid(out, ldout, cols, type) || pos == nullptr || !aligned(pos, 4))
        return HPCDNN_ERR_INVALID_VALUE;
    const size_t e = type_bytes(type);
    return with_rows(type, kind_of(rows_are_dwords(x, ldx, cols, e) && rows_are_dwords(out, ldout, cols, e), cols), [&](auto* t, auto kind) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        const row_launch l = plan_rows(tokens, cols, kVec<T>, true);
        expert_gather_kernel<T, decltype(kind)::value><<<l.grid, l.threads, 0, static_cast<hipStream_t>(stream)>>>(
            tokens, topk, rows, cols, l.team_waves, static_cast<const T*>(x), ldx, pos, static_cast<T*>(out), ldout);
        return launch_status();
    });
}

extern "C" int hpcdnn_expert_combine(int type, int tokens, int topk, int rows, int cols, const void* xs, int64_t ldxs, const int32_t* pos,
                                     const float* weights, void* y, int64_t ldy, void* stream) {
    using namespace hpcdnn;
    if (!type_valid(type) || !choices_valid(tokens, topk) || rows < 0 || cols < 0 || cols > HPCDNN_EXPERTS_MAX_COLS) return HPCDNN_ERR_INVALID_VALUE;
    if (tokens == 0 || cols == 0) return HPCDNN_OK;
    if ((rows > 0 && !rows_valid(xs, ldxs, cols, type)) || !rows_valid(y, ldy, cols, type) || pos == nullptr || !aligned(pos, 4) ||
        !aligned(weights, 4))
        return HPCDNN_ERR_INVALID_VALUE;
    const size_t e = type_bytes(type);
    return with_rows(type, kind_of(rows_are_dwords(xs, ldxs, cols, e) && rows_are_dwords(y, ldy, cols, e), cols), [&](auto* t, auto kind) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        auto go = [&](auto of_tokens) {
            constexpr int kTokens = decltype(of_tokens)::value;
            const row_launch l = plan_rows(ceil_div(tokens, kTokens), cols, kVec<T>, true);
            expert_combine_kernel<T, decltype(kind)::value, kTokens><<<l.grid, l.threads, 0, static_cast<hipStream_t>(stream)>>>(
                tokens, topk, rows, cols, l.team_waves, static_cast<const T*>(xs), ldxs, pos, weights, static_cast<T*>(y), ldy);
            return launch_status();
        };
        // one choice: 6272 x 4544 FP16 20 us, token by token 35; two: 8192 x 6144 BF16 57 us two tokens at a time, 55 one by one
        if (topk == 1) return go(std::integral_constant<int, 4>{});
        return go(std::integral_constant<int, 1>{});
    });
}

extern "C" int hpcdnn_expert_combine_grad(int type, int tokens, int topk, int rows, int cols, const void* dy, int64_t lddy, const void* xs,
                                          int64_t ldxs, const int32_t* pos, const float* weights, void* dxs, int64_t lddxs,
                                          float* dweights, void* stream) {
    using namespace hpcdnn;
    if (!type_valid(type) || !choices_valid(tokens, topk) || rows < 0 || cols < 0 || cols > HPCDNN_EXPERTS_MAX_COLS) return HPCDNN_ERR_INVALID_VALUE;
    if (tokens == 0 || (dxs == nullptr && dweights == nullptr)) return HPCDNN_OK;
    if (pos == nullptr || !aligned(pos, 4) || !aligned(weights, 4) || !aligned(dweights, 4)) return HPCDNN_ERR_INVALID_VALUE;
    if (cols > 0 && (!rows_valid(dy, lddy, cols, type) || (rows > 0 && dweights && !rows_valid(xs, ldxs, cols, type)) ||
                     (rows > 0 && dxs && !rows_valid(dxs, lddxs, cols, type))))
        return HPCDNN_ERR_INVALID_VALUE;
    const size_t e = type_bytes(type);
    const bool all_dwords = rows_are_dwords(dy, lddy, cols, e) && (dweights == nullptr || rows_are_dwords(xs, ldxs, cols, e)) &&
                            (dxs == nullptr || rows_are_dwords(dxs, lddxs, cols, e));
    return with_rows(type, kind_of(all_dwords, cols), [&](auto* t, auto kind) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        row_launch l = plan_rows(tokens, cols, kVec<T>, false);
        // Pairs of choices in workgroups of their own up to sixteen to a CU: 256 x 8 rows of 3586 FP16 8.4 us instead of 13.6,
        // 1800 x 8 of 1792 FP32 43 instead of 48 (44 at eight to a CU); beyond that a token's dy is read once.
        l.grid.y = static_cast<unsigned>(std::min(ceil_div(topk, kGradBatch), ceil_div(16 * static_cast<int64_t>(device_cus()), l.grid.x)));
        expert_combine_grad_kernel<T, decltype(kind)::value><<<l.grid, l.threads, 0, static_cast<hipStream_t>(stream)>>>(
            tokens, topk, rows, cols, l.team_waves, static_cast<const T*>(dy), lddy, static_cast<const T*>(xs), ldxs, pos, weights,
            static_cast<T*>(dxs), lddxs, dweights);
        return launch_status();
    });
}
