// Routing of tokens to experts by scores that are not the logits' own order.  Per token over E logits l, of which those at -infinity are
// not available:
//   s = softmax(l) or sigmoid(l),  c = s + bias (an expert whose bias is -infinity is not available either)
//   the experts in `groups` equal runs: a group's score is the sum of its two largest c; the `kept` best groups take part
//   the k largest c among them (ties of groups and experts: the lowest index) at S;  w = s_S / sum s_S
// with counts, balance and z loss as in route.hip, the balance loss over s / sum s.  The bias steers the choice alone.
//
// What is chosen goes by the order of the c as real numbers, so that it does not depend on how an exponential is rounded.  A row's c are formed in
// fp32, and where two that decide something (neighbours among the k + 1 largest, the last group kept and the
// best one left out) are nearer than what that may be off, the wave does the row again in 64 bits: about 2 rows of a thousand
// with sigmoid scores (8 of 256).  Equal logits with equal biases are a tie, not a near one.
//
// Layout as in route.hip: a row in the registers of L lanes, N elements each, the k largest by 64-bit keys (c above the complement of
// the index).  The c go through LDS for the groups, which may begin anywhere in a lane's elements.
#include "route.h"

namespace muon_amd {

constexpr float RS_UNIT = 0x1p-24f;
constexpr int RS_MAX_GROUPS = 64;

// A double's bits in the order of its value, as `ordered` does for floats.
__device__ __forceinline__ uint64_t ordered_double(double x) {
    const int64_t b = __builtin_bit_cast(int64_t, x == x ? x + 0.0 : __builtin_nan(""));
    return static_cast<uint64_t>(b) ^ (static_cast<uint64_t>(b >> 63) | 0x8000000000000000ull);
}

template <typename T>
__device__ __forceinline__ float logit_of(const T* row, int e) {
    if constexpr (sizeof(T) == 2) return bf2f(row[e]);
    else return row[e];
}

template <typename T>
__device__ __forceinline__ T wave_best(T v) {
    return group_reduce<64>(v, [](T x, T y) { return x > y ? x : y; });
}

// A row once more in 64 bits, by a whole wave: writes the k choices (-1 where there is none).  c: LDS of this wave for E doubles; best: for 64.
template <typename T, bool SIGMOID>
__device__ __noinline__ void choose_again(const T* row, const float* bias, int experts, int k, int groups, int kept, double* c, double* best, int* picks) {
    const int lane = threadIdx.x & 63;
    float most = -__builtin_inff();
    for (int e = lane; e < experts; e += 64) most = fmaxf(most, logit_of(row, e));
    const double top = group_reduce<64>(most, [](float x, float y) { return fmaxf(x, y); });
    double total = 0.0;
    if constexpr (!SIGMOID) {
        for (int e = lane; e < experts; e += 64) total += exp(static_cast<double>(logit_of(row, e)) - top);
        total = group_reduce<64>(total, [](double x, double y) { return x + y; });
    }
    for (int e = lane; e < experts; e += 64) {
        const float x = logit_of(row, e), b = bias ? bias[e] : 0.f;
        const double s = SIGMOID ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - top) / total;
        c[e] = x == -__builtin_inff() ? -__builtin_inf() : s + static_cast<double>(b);
    }
    wave_order();
    if (kept < groups) {
        const int size = experts / groups;
        double first = -__builtin_inf(), second = -__builtin_inf();
        bool none = false;
        if (lane < groups)
            for (int e = lane * size; e < (lane + 1) * size; ++e) {
                const double v = c[e];
                none |= v != v;
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        const double score = none ? __builtin_nan("") : second == -__builtin_inf() ? first : first + second;
        best[lane] = score;
        wave_order();
        int before = 0;
        for (int g = 0; g < groups; ++g) {
            const uint64_t other = ordered_double(best[g]), own = ordered_double(score);
            before += other > own || (other == own && g < lane);
        }
        const uint64_t in = __ballot(lane < groups && before < kept);
        for (int e = lane; e < experts; e += 64)
            if (!(in >> (e / size) & 1)) c[e] = -__builtin_inf();
        wave_order();
    }
    for (int j = 0; j < k; ++j) {
        uint64_t own = 0;
        int at = 0;
        for (int e = lane; e < experts; e += 64) {
            const uint64_t v = ordered_double(c[e]);
            if (v > own) {
                own = v;
                at = e;
            }
        }
        const uint64_t all = wave_best(own);
        const int e = experts - wave_best(own == all ? experts - at : 0);
        const bool there = all > ordered_double(-__builtin_inf());
        if (lane == 0) {
            picks[j] = there ? e : -1;
            c[e < experts ? e : 0] = -__builtin_inf();
        }
        wave_order();
    }
}

template <typename T, int N, int L, bool SIGMOID>
__global__ __launch_bounds__(RT_THREADS) void route_scored_kernel(const MuonRoute a, const float* bias, int groups, int kept) {
    constexpr int ROWS = RT_THREADS / L, WROWS = 64 / L;                      // rows of the workgroup, of a wave
    constexpr int PICKS = N * L < RT_MAX_K + 1 ? N * L : RT_MAX_K + 1, PG = N * L < RS_MAX_GROUPS ? N * L : RS_MAX_GROUPS;
    constexpr int ROWC = N * L + N * L / 32;                                  // a row's c, a place more every 32: groups a power of two apart
    constexpr int CFLOATS = WROWS * ROWC > 2 * N * L ? WROWS * ROWC : 2 * N * L, GFLOATS = 2 * WROWS * PG > 128 ? 2 * WROWS * PG : 128;
    typedef Key<float> K;
    __shared__ float sums[RT_WAVES][N * L];
    __shared__ int tokens[N * L];
    __shared__ float squares[RT_WAVES];
    __shared__ int parts[RT_WAVES];
    __shared__ __align__(8) float by_expert[RT_WAVES][CFLOATS];
    __shared__ __align__(8) float by_group[RT_WAVES][GFLOATS];
    __shared__ int pick_at[RT_WAVES][WROWS][PICKS];
    __shared__ float pick_c[RT_WAVES][WROWS][PICKS];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, base = lane * N, E = a.experts, wave = threadIdx.x >> 6, slot = (threadIdx.x & 63) / L;
    const int size = E / groups, wanted = a.k < E ? a.k + 1 : a.k;           // (one more than is chosen: what the last one is near to)
    float* const row_c = by_expert[wave] + slot * ROWC;
    float* const row_g = by_group[wave] + slot * 2 * PG;                      // scores of the groups, what each may be off by
    int* const row_at = pick_at[wave][slot];
    float* const row_pick = pick_c[wave][slot];
    const auto larger = [](uint64_t u, uint64_t v) { return max(u, v); };
    const auto most_of = [](float u, float v) { return fmaxf(u, v); };
    for (int e = threadIdx.x; e < N * L; e += RT_THREADS) tokens[e] = 0;
    __syncthreads();
    float acc[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        acc[i] = 0.f;
        b[i] = bias && base + i < E ? bias[base + i] : 0.f;
    }
    float square = 0.f;
    int part = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * ROWS + sub; t - sub < a.tokens; t += step) {
        RowPacks<T, N> packs;
        const T* const row = row_of<T>(a, t < a.tokens ? t : a.tokens - 1);
        packs.load(row, base, E);
        const bool in = unmasked(a, t);
        float x[N], s[N];
        packs.get(base, E, in, x);
        // logsumexp, scores
        float top = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, x[i]);
        top = group_reduce<L>(top, most_of);
        if (top == -__builtin_inff()) top = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = x[i] - top;
            s[i] = d == d ? exp_of(d) : d;
            total += s[i];
        }
        total = group_sum<L>(total);
        float per = total != 0.f ? 1.f / total : 0.f, norm = 0.f;
        if constexpr (SIGMOID) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float rest;
                s[i] = sigmoid_of(x[i], rest);
                norm += s[i];
            }
            norm = group_sum<L>(norm);
            norm = norm != 0.f ? 1.f / norm : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] *= per;
            norm = 1.f;
        }
        // What a c may be off by, beside its own rounding: of scores up to 1 or the row's largest probability, or without a bias relative to itself
        // (softmax: that includes the rounding of differences of logits).
        constexpr float OFF = SIGMOID ? 8.f * RS_UNIT : 40.f * RS_UNIT, RELATIVE = SIGMOID ? 8.f * RS_UNIT : 128.f * RS_UNIT;
        const float off = bias ? OFF * (SIGMOID ? 1.f : per) : 0.f, relative = bias ? RS_UNIT : RELATIVE + RS_UNIT;
        bool close = false;
        uint64_t in_groups = ~0ull;
        if (kept < groups) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = base + i;
                row_c[e + e / 32] = x[i] == -__builtin_inff() ? -__builtin_inff() : s[i] + b[i];
            }
            wave_order();
            for (int g = lane; g < groups; g += L) {
                float first = -__builtin_inff(), second = -__builtin_inff();
                bool none = false;
                for (int e = g * size; e < (g + 1) * size; ++e) {
                    const float v = row_c[e + e / 32];
                    none |= v != v;
                    second = fmaxf(second, fminf(first, v));
                    first = fmaxf(first, v);
                }
                const float score = second == -__builtin_inff() ? first : first + second;
                row_g[g] = none ? __builtin_nanf("") : score;
                row_g[PG + g] = 2.f * off + 2.f * relative * (fabsf(first) + (second == -__builtin_inff() ? 0.f : fabsf(second)));
            }
            wave_order();
            // rank of each group; how near the two sides of the border may come
            float low = __builtin_inff(), high = -__builtin_inff();
            uint64_t mine = 0;
            for (int g = lane; g < groups; g += L) {
                const float score = row_g[g];
                const uint32_t own = ordered(score);
                int before = 0;
                for (int o = 0; o < groups; ++o) {
                    const uint32_t other = ordered(row_g[o]);
                    before += other > own || (other == own && o < g);
                }
                if (before < kept) {
                    mine |= 1ull << g;
                    low = fminf(low, score - row_g[PG + g]);
                } else if (score != -__builtin_inff()) {
                    high = fmaxf(high, score + row_g[PG + g]);
                }
            }
            in_groups = group_reduce<L>(mine, [](uint64_t u, uint64_t v) { return u | v; });
            low = -group_reduce<L>(-low, most_of);
            high = group_reduce<L>(high, most_of);
            close = low <= high;
        }
        uint64_t key[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = base + i;
            const bool there = x[i] != -__builtin_inff() && (kept == groups || (in_groups >> (e / size) & 1));
            key[i] = K::of(there ? s[i] + b[i] : -__builtin_inff(), e);
        }
        uint64_t best = 0;
        bool on = false;
        for (int j = 0; j < wanted; ++j) {
            uint64_t m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m = max(m, key[i] - best);
            best += group_reduce<L>(m, larger);
            if (j == 0) on = in && K::available(best);
            if (lane == j % L) {
                row_at[j] = in && K::available(best) ? K::index(best) : -1;
                row_pick[j] = K::value(best);
            }
        }
        wave_order();
        for (int j = lane + 1; j < wanted; j += L) {
            const int at = row_at[j], prev = row_at[j - 1];
            const float c = row_pick[j], before = row_pick[j - 1];
            if (at < 0 || !(before - c <= 2.f * off + 2.f * relative * (fabsf(c) + fabsf(before)))) continue;
            if (!(logit_of(row, at) == logit_of(row, prev) && (!bias || bias[at] == bias[prev]))) close = true;
        }
        const uint64_t again = __ballot(close && on);
        if (again) {
            // a row at a time, each by the whole wave
            for (int q = 0; q < WROWS; ++q) {
                const uint64_t lanes = L == 64 ? ~0ull : ((1ull << (L & 63)) - 1) << (q * L);
                if (!(again & lanes)) continue;
                const int64_t tq = t - slot + q;
                choose_again<T, SIGMOID>(row_of<T>(a, tq), bias, E, a.k, groups, kept, reinterpret_cast<double*>(by_expert[wave]),
                                         reinterpret_cast<double*>(by_group[wave]), pick_at[wave][q]);
            }
            wave_order();
        }
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = on ? fmaf(s[i], norm, acc[i]) : acc[i];
        if (t >= a.tokens) continue;
        // the weights: scores of the choices, formed again from their logits
        const auto score_at = [&](int e) {
            const float l = logit_of(row, e);
            if constexpr (SIGMOID) {
                float rest;
                return sigmoid_of(l, rest);
            } else {
                const float d = l - top;
                return (d == d ? exp_of(d) : d) * per;
            }
        };
        float chosen = 0.f;
        for (int j = lane; j < a.k; j += L) {
            const int e = row_at[j];
            if (e >= 0) chosen += score_at(e);
        }
        chosen = a.normalize ? group_sum<L>(chosen) : 1.f;
        for (int j = lane; j < a.k; j += L) {
            const int e = row_at[j];
            const float score = e >= 0 ? score_at(e) : 0.f;
            a.indices[t * a.k + j] = e;
            a.weights[t * a.k + j] = chosen != 0.f ? score / chosen : 0.f;
            if (e >= 0) atomicAdd(&tokens[e], 1);
        }
        if (lane == 0) {
            const float log_total = logf(total), lse = top + log_total;
            a.lse[t] = on ? lse : -__builtin_inff();
            const float part_of_log = lse - top;                              // what the sum's rounding left out (as in route.hip)
            a.lse_rest[t] = (top - (lse - part_of_log)) + (log_total - part_of_log);
            if (on) square = fmaf(lse, lse, square);
            part += on;
        }
    }
    // join the workgroup's rows: those of a wave, then the waves
#pragma unroll
    for (int i = 0; i < N; ++i) {
        acc[i] = sum_of_groups<L>(acc[i]);
        if ((threadIdx.x & 63) < L) sums[threadIdx.x >> 6][base + i] = acc[i];
    }
    square = group_sum<64>(square);
    part = group_reduce<64>(part, [](int u, int v) { return u + v; });
    if ((threadIdx.x & 63) == 0) {
        squares[threadIdx.x >> 6] = square;
        parts[threadIdx.x >> 6] = part;
    }
    __syncthreads();
    float* const out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * E;
    for (int e = threadIdx.x; e < E; e += RT_THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < RT_WAVES; ++w) sum += sums[w][e];
        out[2 * e] = sum;
        out[2 * e + 1] = __int_as_float(tokens[e]);
    }
    if (threadIdx.x == 0) {
        float* const tail = a.partials + static_cast<int64_t>(gridDim.x) * 2 * E;
        float sum = 0.f;
        int n = 0;
        for (int w = 0; w < RT_WAVES; ++w) {
            sum += squares[w];
            n += parts[w];
        }
        tail[2 * blockIdx.x] = sum;
        tail[2 * blockIdx.x + 1] = __int_as_float(n);
        if (blockIdx.x == 0) tail[2 * gridDim.x] = __int_as_float(0);
    }
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

int muon_amd_route_max_groups(void) { return RS_MAX_GROUPS; }

int muon_amd_route_scored(const MuonRoute* args, int scores, const float* bias, int groups, int groups_kept, void* stream) {
    if (const int rc = check_route(args, "route_scored")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.partials && a.balance && a.z, "route_scored: null workspace or output");
    MUON_REQUIRE(scores == MUON_AMD_SCORES_SOFTMAX || scores == MUON_AMD_SCORES_SIGMOID, "route_scored: scores=%d", scores);
    MUON_REQUIRE(groups > 0 && groups <= RS_MAX_GROUPS && a.experts % groups == 0 && groups_kept > 0 && groups_kept <= groups &&
                     a.k <= groups_kept * (a.experts / groups),
                 "route_scored: %d of %d groups of %d experts for k=%d (at most %d groups)", groups_kept, groups, a.experts, a.k, RS_MAX_GROUPS);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = route_groups(a.tokens, a.experts);
    with_route_type(a.dtype, [&](auto x) {
        with_route_shape(a.experts, [&](auto s) {
            const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(n), dim3(RT_THREADS), 0, st, a, bias, groups, groups_kept); };
            if (scores == MUON_AMD_SCORES_SIGMOID) go(route_scored_kernel<decltype(x), decltype(s)::N, decltype(s)::L, true>);
            else go(route_scored_kernel<decltype(x), decltype(s)::N, decltype(s)::L, false>);
        });
    });
    if (const int rc = check_launch("route_scored")) return rc;
    return launch_route_join(a, n, st);
}

}  // extern "C"
