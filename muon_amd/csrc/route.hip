// Routing of tokens to experts with its losses and gradients.  Per token over E logits l, of which those at -infinity
// are not available:
//   p = softmax(l),  lse = log sum exp(l);  the k largest logits (ties: the lowest index) at S;  w = p_S / sum p_S
// and over the N tokens that take part (not masked out, with at least one expert available):
//   counts_e = tokens whose S holds e;   balance = E sum_e (counts_e / (N k)) (sum_t p_te / N);   z = sum_t lse_t^2 / N
// Backward, from the gradients dw, cb and cz (counts is a constant):
//   dl = p (g - sum p g) + 2 cz lse / N p + [at S] w (dw - sum w dw),    g_e = cb E counts_e / (N k) / N
//
// A row stays in the registers of L lanes, N elements each, and rows of one wave do not wait for each other.  What is
// to be found is the k largest: one 32-bit key holds a bf16 logit (in the order of its value) above the complement of
// its index, so that the largest key is the largest logit at the lowest index; for fp32 logits the key has 64 bits.  The
// largest key below the last one found follows from one wrapping subtraction and one maximum per element.
// Instructions bound both passes where there are many experts (65536 tokens, 8 of 256, bf16: 26 us forward for 38 MB, about half
// of it the eight maxima; 21 us backward for 74 MB), launches where there are few (1024 tokens, 2 of 8: 4.4, 3.6 and 4.4 us).
// Sums over tokens: each lane adds the probabilities of its experts over its rows, a workgroup joins its lanes in a
// fixed order, and a second launch joins the workgroups; counts are whole numbers, in any order the same.
#include "route.h"

namespace muon_amd {

// partials: workgroups x experts pairs {sum of p, tokens}, then workgroups x {sum of lse^2, tokens that take part}, then
// what the launch that joins them needs (a counter, which this one clears, and a float for each of its workgroups).
template <typename T, int N, int L>
__global__ __launch_bounds__(RT_THREADS) void route_forward_kernel(const MuonRoute a) {
    constexpr int ROWS = RT_THREADS / L;
    typedef Key<T> K;
    typedef typename K::type key_t;
    __shared__ float sums[RT_WAVES][N * L];
    __shared__ int tokens[N * L];
    __shared__ float squares[RT_WAVES];
    __shared__ int parts[RT_WAVES];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, base = lane * N, E = a.experts;
    const auto larger = [](key_t u, key_t v) { return max(u, v); };
    for (int e = threadIdx.x; e < N * L; e += RT_THREADS) tokens[e] = 0;
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    float square = 0.f;
    int part = 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * ROWS + sub; t - sub < a.tokens; t += step) {
        RowPacks<T, N> row;
        row.load(row_of<T>(a, t < a.tokens ? t : a.tokens - 1), base, E);
        const bool in = unmasked(a, t);
        float x[N];
        row.get(base, E, in, x);
        key_t key[N];
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = K::of(x[i], base + i);
        // The k largest, one after the other (all keys differ and there are at least k, so this never wraps around).  Lane
        // j mod L takes choice j; where there are more choices than lanes, it leaves the earlier ones unscaled.
        key_t best = 0, mine = 0;
        float top = 0.f, chosen = 0.f, my_part = 0.f;
        int my_expert = -1;
        bool on = false;
        for (int j = 0; j < a.k; ++j) {
            key_t m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m = max(m, static_cast<key_t>(key[i] - best));
            best += group_reduce<L>(m, larger);
            if (j == 0) {
                on = in && K::available(best);
                top = on ? K::value(best) : 0.f;
            }
            if (lane == j % L) mine = best;
            if (j % L != L - 1 && j != a.k - 1) continue;
            // the lanes have a choice each, or it is the last
            const bool has = lane <= j % L, there = has && in && K::available(mine);
            my_part = there ? exp_of(K::value(mine) - top) : 0.f;
            my_expert = there ? K::index(mine) : -1;
            chosen += group_sum<L>(my_part);
            if (there) atomicAdd(&tokens[my_expert], 1);
            const int64_t o = t * a.k + (j - j % L) + lane;
            if (has && t < a.tokens) {
                a.indices[o] = my_expert;
                if (j != a.k - 1) a.weights[o] = my_part;
            }
        }
        // softmax over the row (zeros where it takes no part: all of x is -infinity)
        float ex[N], total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            ex[i] = exp_of(x[i] - top);
            total += ex[i];
        }
        total = group_sum<L>(total);
        const float log_total = on ? logf(total) : 0.f, lse = top + log_total, per = on ? 1.f / total : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(ex[i], per, acc[i]);
        if (t >= a.tokens) continue;
        const float scale = on ? (a.normalize ? 1.f / chosen : per) : 0.f;
        for (int j = lane; j < a.k; j += L) {
            const bool last = j + L >= a.k && j / L == (a.k - 1) / L;
            a.weights[t * a.k + j] = (last ? my_part : a.weights[t * a.k + j]) * scale;
        }
        if (lane == 0) {
            a.lse[t] = on ? lse : -__builtin_inff();
            // what the sum's rounding left out, exactly (D. Knuth, "The Art of Computer Programming", volume 2, 4.2.2)
            const float part_of_log = lse - top;
            a.lse_rest[t] = (top - (lse - part_of_log)) + (log_total - part_of_log);
            square = fmaf(lse, lse, square);
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
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < RT_WAVES; ++w) s += sums[w][e];
        out[2 * e] = s;
        out[2 * e + 1] = __int_as_float(tokens[e]);
    }
    if (threadIdx.x == 0) {
        float* const tail = a.partials + static_cast<int64_t>(gridDim.x) * 2 * E;
        float s = 0.f;
        int n = 0;
        for (int w = 0; w < RT_WAVES; ++w) {
            s += squares[w];
            n += parts[w];
        }
        tail[2 * blockIdx.x] = s;
        tail[2 * blockIdx.x + 1] = __int_as_float(n);
        if (blockIdx.x == 0) tail[2 * gridDim.x] = __int_as_float(0);
    }
}

// Joins the partial sums: a workgroup for every RJ_EXPERTS experts, whose threads share the partial sums of each and read
// four of them at a time; the workgroup that is done last adds what the others left, in their order (one workgroup for all
// of 512 partial sums of 256 experts took 18 us, and 36 with one load at a time).
constexpr int RJ_THREADS = 1024, RJ_EXPERTS = 16, RJ_SHARES = RJ_THREADS / RJ_EXPERTS;
__global__ __launch_bounds__(RJ_THREADS) void route_join_kernel(const MuonRoute a, int groups) {
    __shared__ float psum[RJ_SHARES][RJ_EXPERTS];
    __shared__ int csum[RJ_SHARES][RJ_EXPERTS];
    __shared__ bool last;
    __shared__ float squares[RJ_THREADS / 64];
    __shared__ int parts[RJ_THREADS / 64];
    const int E = a.experts, lane = threadIdx.x % RJ_EXPERTS, share = threadIdx.x / RJ_EXPERTS, e = blockIdx.x * RJ_EXPERTS + lane;
    const float* const tail = a.partials + static_cast<int64_t>(groups) * 2 * E;
    int* const counter = reinterpret_cast<int*>(a.partials + static_cast<int64_t>(groups) * 2 * (E + 1));
    float* const dots = reinterpret_cast<float*>(counter) + 1;
    float p = 0.f;
    int c = 0;
    if (e < E) {
        const f32x2_t* const at = reinterpret_cast<const f32x2_t*>(a.partials) + e;
        const auto add = [&](f32x2_t v) {
            p += v[0];
            c += __float_as_int(v[1]);
        };
        int g = share;
        for (; g + 3 * RJ_SHARES < groups; g += 4 * RJ_SHARES) {
            f32x2_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = at[static_cast<int64_t>(g + i * RJ_SHARES) * E];
#pragma unroll
            for (int i = 0; i < 4; ++i) add(v[i]);
        }
        for (; g < groups; g += RJ_SHARES) add(at[static_cast<int64_t>(g) * E]);
    }
    psum[share][lane] = p;
    csum[share][lane] = c;
    __syncthreads();
    for (int half = RJ_SHARES / 2; half > 0; half >>= 1) {
        if (share < half) {
            psum[share][lane] += psum[share + half][lane];
            csum[share][lane] += csum[share + half][lane];
        }
        __syncthreads();
    }
    if (threadIdx.x < 64) {
        float dot = 0.f;
        if (share == 0 && e < E) {
            a.counts[e] = csum[0][lane];
            dot = static_cast<float>(csum[0][lane]) * psum[0][lane];
        }
        dot = group_sum<64>(dot);
        if (threadIdx.x == 0) {
            __hip_atomic_store(&dots[blockIdx.x], dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.x) - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    float s = 0.f;
    int n = 0;
    for (int g = threadIdx.x; g < groups; g += RJ_THREADS) {
        s += tail[2 * g];
        n += __float_as_int(tail[2 * g + 1]);
    }
    s = group_sum<64>(s);
    n = group_reduce<64>(n, [](int u, int v) { return u + v; });
    if ((threadIdx.x & 63) == 0) {
        squares[threadIdx.x >> 6] = s;
        parts[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x > 0) return;
    for (int w = 1; w < RJ_THREADS / 64; ++w) {
        s += squares[w];
        n += parts[w];
    }
    float total = 0.f;
    for (unsigned g = 0; g < gridDim.x; ++g) total += __hip_atomic_load(&dots[g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const float part = static_cast<float>(n > 0 ? n : 1);
    *a.balance = static_cast<float>(E) * (total / (part * static_cast<float>(a.k))) / part;
    *a.z = s / part;
    *a.part = part;
}

constexpr int RB_THREADS = 256;
constexpr int RB_GROUPS = 1024;            // workgroups: four for each CU, each set up once (65536 x 256: 20.8 us; 1536: 20.6, 2048: 22)
// SIGMOID: scores s = sigmoid(l) instead of p, with q = s / sum s in the balance loss (route_scored.hip):
//   dl = s (1 - s) (g - sum q g) / sum s + 2 cz lse / N p + [at S] (1 - s) w (dw - sum w dw)
template <typename T, int N, int L, bool SIGMOID>
__global__ __launch_bounds__(RB_THREADS) void route_backward_kernel(const MuonRoute a) {
    constexpr int ROWS = RB_THREADS / L, G = pack_of<T>;
    // What the weights' gradients add, by expert.  Four experts of a lane lie next to those of the next lane, so that the
    // lanes' reads of 16 bytes fall on all banks.
    __shared__ f32x4v extra[ROWS][N / 4 * L];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, base = lane * N, E = a.experts;
    const auto slot = [&](int e) { return reinterpret_cast<float*>(extra[sub]) + (e / 4 % (N / 4) * L + e / N) * 4 + e % 4; };
    const float n = *a.part;
    const float cb = a.dbalance ? *a.dbalance * static_cast<float>(E) / (n * n * static_cast<float>(a.k)) : 0.f;
    const float cz = a.dz ? *a.dz * 2.f / n : 0.f;
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = static_cast<float>(a.counts[base + i < E ? base + i : E - 1]);       // (all requested together)
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = base + i < E ? cb * g[i] : 0.f;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) extra[sub][q * L + lane] = f32x4v{0.f, 0.f, 0.f, 0.f};
    wave_order();
    const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS, begin = static_cast<int64_t>(blockIdx.x) * ROWS + sub;
    // The next row is on its way while this one is worked on: its logits, and each lane's first choice.
    RowPacks<T, N> next;
    float next_lse, next_rest, next_w = 0.f, next_dw = 0.f;
    int next_e = -1;
    const bool chooses = a.dweights && lane < a.k;
    const auto fetch = [&](int64_t t) {
        const int64_t row = t < a.tokens ? t : a.tokens - 1;
        next.load(row_of<T>(a, row), base, E);
        next_lse = a.lse[row];
        next_rest = a.lse_rest[row];
        if (chooses) {
            next_w = a.weights[row * a.k + lane];
            next_dw = a.dweights[row * a.ld_dweights + lane];
            next_e = a.indices[row * a.k + lane];
        }
    };
    fetch(begin);
    for (int64_t t = begin; t - sub < a.tokens; t += step) {
        RowPacks<T, N> packs = next;
        const bool on = t < a.tokens && next_lse != -__builtin_inff();
        // (what rounding lse left out would go into every probability: all of a row's logits at a value far from zero, as
        // the type's lowest one, lose the logarithm of their number)
        const float lse = on ? next_lse : 0.f, rest = on ? next_rest : 0.f, w = next_w, dw = next_dw;
        const int mine = on ? next_e : -1;
        fetch(t + step);
        // The weights' part; lanes of the row take the k choices in turn.
        if (a.dweights) {
            float dot = mine >= 0 ? w * dw : 0.f;        // (what arrives for a choice that is not there may be no number)
            for (int j = lane + L; j < a.k; j += L)
                if (on && a.indices[t * a.k + j] >= 0) dot = fmaf(a.weights[t * a.k + j], a.dweights[t * a.ld_dweights + j], dot);
            dot = a.normalize ? group_sum<L>(dot) : 0.f;
            if (mine >= 0) *slot(mine) = w * (dw - dot);
            for (int j = lane + L; j < a.k; j += L) {
                const int e = on ? a.indices[t * a.k + j] : -1;
                if (e >= 0) *slot(e) = a.weights[t * a.k + j] * (a.dweights[t * a.ld_dweights + j] - dot);
            }
        }
        wave_order();
        float x[N], p[N], u[N], dot = 0.f;
        [[maybe_unused]] float s[SIGMOID ? N : 1], rest_of[SIGMOID ? N : 1], norm = 0.f;
        packs.get(base, E, x);
        const int limit = on ? E - base : 0;
        if (__ballot(limit < N)) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = i < limit ? x[i] : -__builtin_inff();
        }
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const f32x4v v = extra[sub][q * L + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[4 * q + i] = v[i];
        }
        if (SIGMOID && !__ballot(!(lse >= 0.f && lse <= 33.f))) {
            // One exponential serves both: no logit is too large for it, and where it loses bits for being small, so does p.
            const float whole = exp_of(-lse), per = fmaf(-rest, whole, whole);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float e = exp_of(x[i]);
                rest_of[i] = __builtin_amdgcn_rcpf(1.f + e);
                s[i] = e * rest_of[i];
                p[i] = e * per;
                norm += s[i];
                dot = fmaf(s[i], g[i], dot);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                p[i] = exp_of(x[i] - lse - rest);  // (zero where the token takes no part: x is -infinity)
                if constexpr (SIGMOID) {
                    s[i] = sigmoid_of(x[i], rest_of[i]);
                    if (lse < 0.f) s[i] = p[i] * rest_of[i];       // s / e^lse: the row's norm takes it out, and it does not vanish with s
                    norm += s[i];
                    dot = fmaf(s[i], g[i], dot);
                } else {
                    dot = fmaf(p[i], g[i], dot);
                    if (!a.normalize) dot += u[i]; // p dw: what comes through the probabilities themselves
                }
            }
        }
        dot = group_sum<L>(dot);
        if constexpr (SIGMOID) {
            norm = group_sum<L>(norm);
            norm = norm != 0.f ? 1.f / norm : 0.f;
            dot = dot * norm * norm;
        }
        [[maybe_unused]] const float all = on ? fmaf(cz, lse, -dot) : 0.f, zed = cz * lse;
        wave_order();
        if (a.dweights) {
            if (mine >= 0) *slot(mine) = 0.f;
            for (int j = lane + L; j < a.k; j += L) {
                const int e = on ? a.indices[t * a.k + j] : -1;
                if (e >= 0) *slot(e) = 0.f;
            }
        }
        if (t >= a.tokens) continue;
#pragma unroll
        for (int q = 0; q < N / G; ++q) {
            float d[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int k = G * q + i;
                if constexpr (SIGMOID) d[i] = fmaf(p[k], zed, rest_of[k] * fmaf(s[k], fmaf(g[k], norm, -dot), u[k]));
                else d[i] = fmaf(p[k], g[k] + all, u[k]);
            }
            const Pack<T, G> v = Pack<T, G>::of(d);
            store_pack<T, G, false>(static_cast<T*>(a.dlogits) + t * E, base + G * q, E, !SIGMOID || on ? v : Pack<T, G>::zero());
        }
    }
}

// Forward 16 elements for each lane keep the reductions short (65536 x 256 26 us; 8 elements 29, 32 elements 31); backward, with
// one reduction, 8 leave room for twice the waves (21 us; 16 elements 23, 32 elements 29).
template <typename F>
static void with_route_backward_shape(int experts, F&& f) {
    if (experts <= 64) with_route_shape(experts, f);
    else if (experts <= 128) f(RouteShape<8, 16>{});
    else if (experts <= 256) f(RouteShape<8, 32>{});
    else if (experts <= 512) f(RouteShape<8, 64>{});
    else f(RouteShape<16, 64>{});
}
int launch_route_join(const MuonRoute& a, int groups, hipStream_t stream) {
    hipLaunchKernelGGL(route_join_kernel, dim3((a.experts + RJ_EXPERTS - 1) / RJ_EXPERTS), dim3(RJ_THREADS), 0, stream, a, groups);
    return check_launch("route");
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_route(void) { return sizeof(MuonRoute); }
int muon_amd_route_max_experts(void) { return RT_MAX_EXPERTS; }
int muon_amd_route_max_k(void) { return RT_MAX_K; }

int64_t muon_amd_route_partials(int64_t tokens, int experts) {
    if (tokens <= 0 || experts <= 0 || experts > RT_MAX_EXPERTS) return 0;
    return static_cast<int64_t>(route_groups(tokens, experts)) * 2 * (experts + 1) + 1 + (experts + RJ_EXPERTS - 1) / RJ_EXPERTS;
}

int muon_amd_route(const MuonRoute* args, void* stream) {
    if (const int rc = check_route(args, "route")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.partials && a.balance && a.z, "route: null workspace or output");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = route_groups(a.tokens, a.experts);
    with_route_type(a.dtype, [&](auto x) {
        with_route_shape(a.experts, [&](auto s) {
            hipLaunchKernelGGL((route_forward_kernel<decltype(x), decltype(s)::N, decltype(s)::L>), dim3(n), dim3(RT_THREADS), 0, st, a);
        });
    });
    if (const int rc = check_launch("route")) return rc;
    return launch_route_join(a, n, st);
}

int muon_amd_route_backward(const MuonRoute* args, void* stream) { return muon_amd_route_scored_backward(args, MUON_AMD_SCORES_SOFTMAX, stream); }

int muon_amd_route_scored_backward(const MuonRoute* args, int scores, void* stream) {
    if (const int rc = check_route(args, "route_backward")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.dlogits, "route_backward: null output");
    MUON_REQUIRE(scores == MUON_AMD_SCORES_SOFTMAX || scores == MUON_AMD_SCORES_SIGMOID, "route_backward: scores=%d", scores);
    with_route_type(a.dtype, [&](auto x) {
        with_route_backward_shape(a.experts, [&](auto s) {
            constexpr int ROWS = RB_THREADS / decltype(s)::L;
            const int64_t n = (a.tokens + ROWS - 1) / ROWS;
            const auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(n < RB_GROUPS ? n : RB_GROUPS), dim3(RB_THREADS), 0, static_cast<hipStream_t>(stream), a);
            };
            if (scores == MUON_AMD_SCORES_SIGMOID) go(route_backward_kernel<decltype(x), decltype(s)::N, decltype(s)::L, true>);
            else go(route_backward_kernel<decltype(x), decltype(s)::N, decltype(s)::L, false>);
        });
    });
    return check_launch("route_backward");
}

}  // extern "C"
