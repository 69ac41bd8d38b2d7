// Routing of tokens to experts by scores that are not the logits' own order.  Per token over E logits l, of which those at -infinity are
// not available:
//   s = softmax(l) or sigmoid(l),  c = s + bias (an expert whose bias is -infinity is not available either)
//   the experts in `groups` equal runs: a group's score is the sum of its two largest c; the `kept` best groups take part
//   the k largest c among them (ties of groups and experts: the lowest index) at S;  w = s_S / sum s_S
// with counts, balance and z loss as in route.hip, the balance loss over s / sum s.  The bias steers the choice alone.
//
// What is chosen goes by the order of the c as real numbers, so that it does not depend on how an exponential is rounded.  A row's c are formed in
// fp32, and where two that decide something (neighbours among the k + 1 largest, the last of these and what is left out, the last group kept and the
// best one left out) are nearer than what that may be off, the wave does the row again in 64 bits: 5 to 7 rows of 10000 (8 of 256 by
// sigmoid in bf16, 6 of 160 by softmax in fp32, logits of a spread of 1.5).  Where sigmoids saturate and no bias tells them apart, that is every
// row, one after the other in its wave: forward over 65536 x 256 in 4 of 8 groups takes 62 us at a spread of 1.5, 235 (fp32: 262) at 5, 310 from 12 on;
// with random biases 62 to 82.  Equal logits with equal biases are a tie, not a near one; a row of nothing else (a router that starts at zero) is never done again.
//
// Layout as in route.hip: a row in the registers of L lanes, N elements each.  The two largest c of a group come from its lanes, or through LDS where
// groups begin anywhere in a lane's elements.  Instructions bound it (85 for each logit; the vector units issue in 85 % of the cycles in which their CU
// has work): 65536 tokens, 8 of 256 in 4 of 8 groups, sigmoid, bf16 61 us for 38 MB (with 64-bit keys for the choice and the biases in registers
// 116), all logits equal likewise; 30011 tokens, 6 of 160 in 3 of 8, softmax, fp32 41 us.
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

// exp_of that hands on what is no number.
__device__ __forceinline__ float exp_with_nan(float d) { return exp_of_bounded(d < -200.f ? -200.f : d); }

template <typename T>
__device__ __forceinline__ T wave_best(T v) {
    return group_reduce<64>(v, [](T x, T y) { return x > y ? x : y; });
}

// A row once more in 64 bits, by a whole wave: writes the k choices (-1 where there is none).  c: LDS of this wave for E doubles; best: for 64 (which
// the choices may go over).
template <typename T, bool SIGMOID>
__device__ __forceinline__ void choose_again(const T* row, const float* bias, int experts, int k, int groups, int kept, double* c, double* best, int* picks) {
    const int lane = threadIdx.x & 63;
    float most = -__builtin_inff();
#pragma unroll 1
    for (int e = lane; e < experts; e += 64) most = fmaxf(most, logit_of(row, e));
    const double top = group_reduce<64>(most, [](float x, float y) { return fmaxf(x, y); });
    double total = 0.0;
    if constexpr (!SIGMOID) {
#pragma unroll 1
        for (int e = lane; e < experts; e += 64) total += exp(static_cast<double>(logit_of(row, e)) - top);
        total = group_reduce<64>(total, [](double x, double y) { return x + y; });
    }
#pragma unroll 1
    for (int e = lane; e < experts; e += 64) {
        const float x = logit_of(row, e), b = bias ? bias[e] : 0.f;
        const double s = SIGMOID ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - top) / total;
        c[e] = x == -__builtin_inff() ? -__builtin_inf() : s + static_cast<double>(b);
    }
    wave_order();
    if (kept < groups) {
        const int size = experts / groups;
        double first = -__builtin_inf(), second = -__builtin_inf();
        if (lane < groups)
#pragma unroll 1
            for (int e = lane * size; e < (lane + 1) * size; ++e) {
                const double v = c[e] == c[e] ? c[e] : __builtin_inf();
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        const double score = second == -__builtin_inf() ? first : first + second;
        best[lane] = score;
        wave_order();
        int before = 0;
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
            const uint64_t other = ordered_double(best[g]), own = ordered_double(score);
            before += other > own || (other == own && g < lane);
        }
        const uint64_t in = __ballot(lane < groups && before < kept);
#pragma unroll 1
        for (int e = lane; e < experts; e += 64)
            if (!(in >> (e / size) & 1)) c[e] = -__builtin_inf();
        wave_order();
    }
#pragma unroll 1
    for (int j = 0; j < k; ++j) {
        uint64_t own = 0;
        int at = 0;
#pragma unroll 1
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

// The weights and indices of a row by L lanes: scores of the choices, formed again from their logits (softmax: e^(l - top) per).  Weights that add up to
// one go by the ratios of scores, which are there where the scores themselves are below the smallest number: where one of the chosen is so far down, the
// row's scores are formed relative to e^m, m its largest chosen logit (or 0, for a sigmoid above that), e^(l - m) or e^(l - m) / (1 + e^l).
constexpr int LATER = -2;                        // first index of a row that is to be done again
constexpr float FAR_DOWN = 0x1p-116f;            // (2^-126 is the smallest normal number)
template <typename T, int L, bool SIGMOID>
__device__ __forceinline__ void put_choices(const MuonRoute& a, int64_t t, const T* row, float top, float per, const int* picks, int* tokens, int lane) {
    bool relative = false;
    const auto score_at = [&](int e) {
        const float l = logit_of(row, e);
        if constexpr (SIGMOID) {
            if (relative) return exp_with_nan(l - top) * __builtin_amdgcn_rcpf(1.f + exp_of(l));
            float rest;
            return sigmoid_of(l, rest);
        } else {
            const float d = l - top;
            return (d == d ? exp_of(d) : d) * per;
        }
    };
    const int own = lane < a.k ? picks[lane] : -1;
    float first, chosen;
    bool far = false;
    const auto add_up = [&] {
        first = own >= 0 ? score_at(own) : 0.f;
        chosen = first;
        far |= own >= 0 && first < FAR_DOWN;
        for (int j = lane + L; j < a.k; j += L)
            if (const int e = picks[j]; e >= 0) {
                const float s = score_at(e);
                far |= s < FAR_DOWN;
                chosen += s;
            }
    };
    add_up();
    if (a.normalize && __ballot(far)) {
        const auto most_of = [](float u, float v) { return fmaxf(u, v); };
        float most = own >= 0 ? logit_of(row, own) : -__builtin_inff();
        for (int j = lane + L; j < a.k; j += L)
            if (picks[j] >= 0) most = fmaxf(most, logit_of(row, picks[j]));
        most = group_reduce<L>(most, most_of);
        relative = group_reduce<L>(far ? 1.f : 0.f, most_of) != 0.f && (!SIGMOID || most <= 0.f);
        top = relative ? most : top;
        per = relative ? 1.f : per;
        add_up();
    }
    chosen = a.normalize ? group_sum<L>(chosen) : 1.f;
    for (int j = lane; j < a.k; j += L) {
        const int e = picks[j];
        const float score = j == lane ? first : e >= 0 ? score_at(e) : 0.f;
        a.indices[t * a.k + j] = e;
        a.weights[t * a.k + j] = chosen != 0.f ? score / chosen : 0.f;
        if (e >= 0) atomicAdd(&tokens[e], 1);
    }
}

// The sum of v over the lanes before this one in its group of L.
template <int L>
__device__ __forceinline__ int sum_before(int v, int lane) {
    int at = v;
    const auto step = [&](int o, bool there) { at += there ? o : 0; };
    if constexpr (L >= 2) step(moved<0x111>(at), L >= 16 || lane >= 1);          // row_shr:1 (zero at the start of 16 lanes)
    if constexpr (L >= 4) step(moved<0x112>(at), L >= 16 || lane >= 2);
    if constexpr (L >= 8) step(moved<0x114>(at), L >= 16 || lane >= 4);
    if constexpr (L >= 16) step(moved<0x118>(at), true);
    if constexpr (L >= 32) step(__shfl(at, (threadIdx.x & 32) | 15, 64), lane & 16);
    if constexpr (L >= 64) step(__shfl(at, 31, 64), lane & 32);
    return at - v;
}

template <typename T, int N, int L, bool SIGMOID>
__global__ __launch_bounds__(RT_THREADS, 4) void route_scored_kernel(const MuonRoute a, const float* bias, int groups, int kept) {
    constexpr int ROWS = RT_THREADS / L, WROWS = 64 / L;                      // rows of the workgroup, of a wave
    constexpr int PICKS = N * L < RT_MAX_K + 1 ? N * L : RT_MAX_K + 1, PG = N * L < RS_MAX_GROUPS ? N * L : RS_MAX_GROUPS;
    constexpr int LIST = PICKS;                                               // (all `wanted`; the places of more take longer to count than a shorter list)
    constexpr int SPREAD = (N * L + N * L / 32 + 1) / 2 * 2;                  // a row's c, a place more every 32: groups a power of two apart
    constexpr int ROWC = SPREAD > 2 * LIST ? SPREAD : 2 * LIST;               // that, or its list
    constexpr int CFLOATS = WROWS * ROWC > 2 * N * L ? WROWS * ROWC : 2 * N * L;
    constexpr int ROWG = 2 * (PG > PICKS ? PG : PICKS), GFLOATS = WROWS * ROWG > 128 ? WROWS * ROWG : 128;     // a row's groups, then its choices
    __shared__ int tokens[N * L];
    __shared__ __align__(16) float biases[N * L];
    __shared__ float squares[RT_WAVES];
    __shared__ int parts[RT_WAVES];
    __shared__ __align__(8) float by_expert[RT_WAVES][CFLOATS];
    __shared__ __align__(8) float by_group[RT_WAVES][GFLOATS];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, first_of_lane = lane * N, E = a.experts, wave = threadIdx.x >> 6, slot = (threadIdx.x & 63) / L;
    const int size = E / groups, wanted = a.k < E ? a.k + 1 : a.k;           // (one more than is chosen: what the last one is near to)
    float* const row_c = by_expert[wave] + slot * ROWC;
    float* const row_g = by_group[wave] + slot * ROWG;                        // scores of the groups, what each may be off by
    int* const row_at = reinterpret_cast<int*>(row_g);                        // once the groups are known: the choices and their c
    float* const row_pick = row_g + PICKS;
    const auto most_of = [](float u, float v) { return fmaxf(u, v); };
    const auto sum_of = [](int u, int v) { return u + v; };
    for (int e = threadIdx.x; e < N * L; e += RT_THREADS) {
        tokens[e] = 0;
        biases[e] = bias && e < E ? bias[e] : 0.f;
    }
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    // the groups of a lane's elements, a byte each
    uint32_t group_of[N / 4];
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        group_of[q] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) group_of[q] |= static_cast<uint32_t>(min((first_of_lane + 4 * q + i) / size, groups - 1)) << (8 * i);
    }
    float square = 0.f;
    int part = 0;
    bool later = false, biases_none = false, biases_flat = true;             // (flat: one number for all experts)
    for (int e = 0; e < N; ++e) {
        const float b = biases[first_of_lane + e];
        biases_none |= b != b;
        biases_flat &= first_of_lane + e >= E || b == biases[0];
    }
    biases_none = __ballot(biases_none) != 0;
    biases_flat = __ballot(!biases_flat) == 0;
    const bool quarters = 2 * wanted <= 4 * (E * kept / groups) / N;          // maxima of lanes' quarters, where experts are chosen from
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * ROWS + sub; t - sub < a.tokens; t += step) {
        // (opaque copies: what follows from them for each of N elements is formed where it is used, not kept in N registers each)
        int base = first_of_lane;
        asm volatile("" : "+v"(base));
        RowPacks<T, N> packs;
        const T* const row = row_of<T>(a, t < a.tokens ? t : a.tokens - 1);
        packs.load(row, base, E);
        const bool in = unmasked(a, t);
        float x[N], s[N];
        packs.get(base, E, x);
        const int limit = in ? E - base : 0;
        if (__ballot(limit < N)) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = i < limit ? x[i] : -__builtin_inff();
        }
        // logsumexp, scores.  Where the largest logit (of every row of the wave) is not far from zero, a sigmoid's exponential serves both: what
        // is lost of logits far below it is nothing beside its own.
        float top = -__builtin_inff(), low = __builtin_inff(), total = 0.f, norm = 1.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            top = fmaxf(top, x[i]);
            low = fminf(low, x[i]);
        }
        const bool gaps = __ballot(low == -__builtin_inff()) != 0;             // logits that are not available
        if (gaps) {
            low = __builtin_inff();
#pragma unroll
            for (int i = 0; i < N; ++i) low = fminf(low, x[i] == -__builtin_inff() ? __builtin_inff() : x[i]);
        }
        top = group_reduce<L>(top, most_of);
        const bool flat = biases_flat && -group_reduce<L>(-low, most_of) == top;
        if (top == -__builtin_inff()) top = 0.f;
        if (SIGMOID && !__ballot(!(fabsf(top) <= 40.f))) {
            top = 0.f;
            norm = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = exp_with_nan(x[i]);
                s[i] = e * __builtin_amdgcn_rcpf(1.f + e);
                total += e;
                norm += s[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s[i] = exp_with_nan(x[i] - top);
                total += s[i];
            }
            if constexpr (SIGMOID) {
                norm = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float rest;
                    s[i] = sigmoid_of(x[i], rest);
                    norm += s[i];
                }
            }
        }
        total = group_sum<L>(total);
        const float per = total != 0.f ? 1.f / total : 0.f;
        if constexpr (SIGMOID) {
            norm = group_sum<L>(norm);
            norm = norm != 0.f ? 1.f / norm : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] *= per;
        }
        // What a c may be off by, beside its own rounding: of scores up to 1 or the row's largest probability, or without a bias relative to itself
        // (softmax: that includes the rounding of differences of logits) and, where it is below the smallest normal number, by that.
        // The 0.22 |d| units of an exponential (lanes.h) need no room there.  They take every argument d as d (1 - 1.34e-8), which keeps the order of
        // scores; two sums of two that are equal have arguments whose means, weighted by the terms, are within ln 2 of each other (the mean is ln S minus the
        // entropy of the terms' shares), so that the sums move apart by 0.16 units (sigmoids near one: by less); and beside a bias they are 0.22 |d| e^d, at most 0.08.
        constexpr float OFF = SIGMOID ? 8.f * RS_UNIT : 40.f * RS_UNIT, RELATIVE = SIGMOID ? 8.f * RS_UNIT : 128.f * RS_UNIT;
        const float off = bias ? OFF * (SIGMOID ? 1.f : per) : 0x1p-124f, relative = bias ? RS_UNIT : RELATIVE + RS_UNIT;
        // from here on what is chosen by; the token takes part if anything is available
        float c[N], most = -__builtin_inff();
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const f32x4v b = *reinterpret_cast<const f32x4v*>(&biases[base + 4 * q]);
#pragma unroll
            for (int i = 4 * q; i < 4 * q + 4; ++i) {
                c[i] = s[i] + b[i % 4];
            }
        }
        if (gaps) {
#pragma unroll
            for (int i = 0; i < N; ++i) c[i] = x[i] == -__builtin_inff() ? -__builtin_inff() : c[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) most = fmaxf(most, c[i]);
        if (biases_none || __ballot(total != total)) {               // (a maximum passes over what is no number)
#pragma unroll
            for (int i = 0; i < N; ++i) most = c[i] == c[i] ? most : 0.f;
        }
        const bool on = group_reduce<L>(most, most_of) != -__builtin_inff();
        // (shares of sigmoids so small are the probabilities, to 2^-57, and do not vanish with them; such rows have gone the second way above)
        if (const bool small = top < -40.f; SIGMOID && __ballot(small)) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = small ? exp_with_nan(x[i] - top) : s[i];
            norm = small ? per : norm;
        }
        norm = on ? norm : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(s[i], norm, acc[i]);
        // (a row in which anything is no number is done again, where that is the largest value)
        bool again = total != total || biases_none, close = false, lane_in = true;
        uint64_t in_groups = 0;
        if (kept < groups) {
            // the two largest c of each group: of a lane's elements where they are of one group, else through all of them in LDS
            const bool whole = size % N == 0;
            if (whole) {
                float first = c[0], second = -__builtin_inff();
#pragma unroll
                for (int i = 1; i < N; ++i) {
                    second = fmaxf(second, fminf(first, c[i]));
                    first = fmaxf(first, c[i]);
                }
                row_c[2 * lane] = first;
                row_c[2 * lane + 1] = second;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) row_c[base + base / 32 + i] = c[i];      // (a lane's elements lie within 32)
            }
            wave_order();
            bool uneven = false;                                               // (a row of equal logits: not one score for all groups)
            for (int g = lane; g < groups; g += L) {
                float first = -__builtin_inff(), second = -__builtin_inff();
                if (whole) {
                    for (int q = g * (size / N); q < (g + 1) * (size / N); ++q) {
                        const float u = row_c[2 * q], v = row_c[2 * q + 1];
                        second = fmaxf(fmaxf(second, v), fminf(first, u));
                        first = fmaxf(first, u);
                    }
                } else {
                    for (uint32_t e = g * size; e < static_cast<uint32_t>((g + 1) * size); ++e) {
                        const float v = row_c[e + (e >> 5)];
                        second = fmaxf(second, fminf(first, v));
                        first = fmaxf(first, v);
                    }
                }
                const bool one = second == -__builtin_inff();
                uneven |= one && size > 1 && first != -__builtin_inff();
                row_g[g] = one ? first : first + second;
                row_g[PG + g] = 2.f * off + 2.f * relative * (fabsf(first) + (one ? 0.f : fabsf(second)));
            }
            wave_order();
            // rank of each group; how near the two sides of the border may come
            float low = __builtin_inff(), high = -__builtin_inff();
            for (int g = lane; g < groups; g += L) {
                const float score = row_g[g];
                int before = 0;
                for (int o = 0; o < groups; ++o) {
                    const float other = row_g[o];
                    before += other > score || (other == score && o < g);
                }
                if (before < kept) {
                    in_groups |= 1ull << g;
                    low = fminf(low, score - row_g[PG + g]);
                } else if (score != -__builtin_inff()) {
                    high = fmaxf(high, score + row_g[PG + g]);
                }
            }
            in_groups = group_reduce<L>(in_groups, [](uint64_t u, uint64_t v) { return u | v; });
            low = -group_reduce<L>(-low, most_of);
            high = group_reduce<L>(high, most_of);
            close |= low <= high;
            again |= uneven && low <= high;
            if (whole) {
                lane_in = in_groups >> (group_of[0] & 255) & 1;
            } else {
#pragma unroll
                for (int q = 0; q < N / 4; ++q) {
                    uint32_t four = group_of[q];
                    asm volatile("" : "+v"(four));
#pragma unroll
                    for (int i = 0; i < 4; ++i) c[4 * q + i] = in_groups >> (four >> (8 * i) & 255) & 1 ? c[4 * q + i] : -__builtin_inff();
                }
            }
        }
        // The `wanted` largest values, each below the one before (in the order of their bits: as in route.hip, one subtraction and one maximum for
        // each; there is always -infinity to end with), of the maxima of a lane's quarters where these are enough, else of all elements.  Then every
        // element that is as large as the last of them goes into a list, and its place in the order is counted there: equal values are told
        // apart by their index.  (The list is longer by a few for the quarters: at least `wanted` elements, and values, are as large as the last.  65536 x 256:
        // the whole call takes 90.1 us with all elements, 88.0 with the quarters.)
        uint32_t key[N], best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t bits = __float_as_uint(lane_in ? c[i] : -__builtin_inff());
            key[i] = bits ^ (static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u);
        }
        const auto search = [&](const auto& keys) __attribute__((always_inline)) {
            for (int j = 0; j < wanted; ++j) {
                uint32_t m = ORDERED_MINUS_INF - best;
#pragma unroll
                for (const uint32_t v : keys) m = max(m, v - best);
                m = group_reduce<L>(m, [](uint32_t u, uint32_t v) { return max(u, v); });
                best += best == ORDERED_MINUS_INF ? 0u : m;
            }
        };
        if (quarters) {
            uint32_t most_of_quarter[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                most_of_quarter[q] = key[q * (N / 4)];
#pragma unroll
                for (int i = 1; i < N / 4; ++i) most_of_quarter[q] = max(most_of_quarter[q], key[q * (N / 4) + i]);
            }
            search(most_of_quarter);
        } else {
            search(key);
        }
        best = max(best, ORDERED_MINUS_INF + 1);
        int listed = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) listed += key[i] >= best;
        const int at = sum_before<L>(listed, lane);
        listed = group_reduce<L>(listed, sum_of);
        uint64_t* const list = reinterpret_cast<uint64_t*>(row_c);               // value and complement of the index, LIST of them: larger is earlier
        uint64_t* entry = list + at;
        const auto put = [&](int i) { *entry++ = static_cast<uint64_t>(key[i]) << 32 | static_cast<uint32_t>(~base - i); };
        const bool cut = __ballot(listed > LIST) != 0;
        wave_order();
        if (!cut) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (key[i] >= best) put(i);
        } else {
            // A row of the wave has more equal values than the list holds.  The largest value that `wanted` elements reach (all that are
            // available, where these are fewer): those above it are less than `wanted`, and of those that are equal to it the first ones by index go
            // into the list, `wanted` in all at most.
            int above, equal;
            uint32_t value = 0;
            bool found = false;
            for (int j = 0; j < wanted && __ballot(!found); ++j) {
                uint32_t m = ORDERED_MINUS_INF - value;
#pragma unroll
                for (int i = 0; i < N; ++i) m = max(m, key[i] - value);
                m = group_reduce<L>(m, [](uint32_t u, uint32_t v) { return max(u, v); });
                value += found || value == ORDERED_MINUS_INF ? 0u : m;
                int reach = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) reach += key[i] >= value;
                found = group_reduce<L>(reach, sum_of) >= wanted;
            }
            best = max(value, ORDERED_MINUS_INF + 1);
            above = 0, equal = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                above += key[i] > best;
                equal += key[i] == best;
            }
            const int need = wanted - group_reduce<L>(above, sum_of);
            int place = sum_before<L>(equal, lane);
            above += min(max(need - place, 0), equal);
            entry = list + sum_before<L>(above, lane);
            listed = group_reduce<L>(above, sum_of);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (key[i] > best || (key[i] == best && place < need)) put(i);
                place += key[i] == best;
            }
        }
        wave_order();
        for (int q = lane; q < listed; q += L) {
            const uint64_t own = list[q];
            int before = 0;
            for (int o = 0; o < listed; ++o) before += list[o] > own;
            if (before < wanted) {
                row_at[before] = ~static_cast<uint32_t>(own);
                row_pick[before] = value_of(static_cast<uint32_t>(own >> 32));
            }
        }
        for (int j = listed + lane; j < wanted; j += L) row_at[j] = -1;
        wave_order();
        // Whether two scores are nearer than what they may be off, and not a tie: neighbours in the order, and the last one with those that are
        // not in it, where there are ties (as large as it, or the next smaller ones).
        const auto near = [&](float c, int at, float o, int other) {
            if (!(fabsf(o - c) <= 2.f * off + 2.f * relative * (fabsf(c) + fabsf(o)))) return false;
            return !(logit_of(row, at) == logit_of(row, other) && (!bias || bias[at] == bias[other]));
        };
        if (!flat) {
            for (int j = lane + 1; j < wanted; j += L) {
                const int at = row_at[j];
                if (at >= 0) close |= near(row_pick[j], at, row_pick[j - 1], row_at[j - 1]);
            }
            const int last = row_at[wanted - 1];
            const float least = row_pick[wanted - 1];
            if (listed > wanted)
#pragma unroll 1
                for (int q = lane; q < listed; q += L) {
                    const float c = value_of(static_cast<uint32_t>(list[q] >> 32));
                    const int index = static_cast<int>(~static_cast<uint32_t>(list[q]));
                    if (c <= least && index != last) close |= near(c, index, least, last);
                }
            if (cut && last >= 0) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (key[i] <= best && key[i] > ORDERED_MINUS_INF && base + i != last) close |= near(value_of(key[i]), base + i, least, last);
            }
        }
        close = again || (close && !flat);
        close = group_reduce<L>(static_cast<int>(close), [](int u, int v) { return u | v; }) != 0;
        if (t >= a.tokens) continue;
        if (on && close) {                       // (the rows that are done again come after the loop, out of its registers' way)
            if (lane == 0) a.indices[t * a.k] = LATER;
            later = true;
        } else {
            put_choices<T, L, SIGMOID>(a, t, row, top, per, row_at, tokens, lane);
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
    wave_order();                                // (what a lane has left in memory is read by others of its wave)
    if (__ballot(later)) {
        const int whole = threadIdx.x & 63;
        for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS + sub - slot; first < a.tokens; first += step) {
            const int64_t own = first + whole;
            uint64_t again = __ballot(whole < WROWS && own < a.tokens && a.indices[(own < a.tokens ? own : first) * a.k] == LATER);
            for (; again; again &= again - 1) {
                const int64_t t = first + __builtin_ctzll(again);
                const T* const row = row_of<T>(a, t);
                choose_again<T, SIGMOID>(row, bias, E, a.k, groups, kept, reinterpret_cast<double*>(by_expert[wave]),
                                         reinterpret_cast<double*>(by_group[wave]), reinterpret_cast<int*>(by_group[wave]));
                put_choices<T, 64, SIGMOID>(a, t, row, a.lse[t], expf(-a.lse_rest[t]), reinterpret_cast<int*>(by_group[wave]), tokens, whole);
                wave_order();
            }
        }
    }
    // join the workgroup's rows: those of a wave, then the waves
#pragma unroll
    for (int i = 0; i < N; ++i) {
        acc[i] = sum_of_groups<L>(acc[i]);
        if ((threadIdx.x & 63) < L) by_expert[wave][first_of_lane + i] = acc[i];
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
        for (int w = 0; w < RT_WAVES; ++w) sum += by_expert[w][e];
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
