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
#include <type_traits>

#include "vector.h"

namespace muon_amd {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_K = 32;
constexpr int RT_THREADS = 512;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int RT_GROUPS = 512;             // workgroups at most: their partial sums are joined by one launch

// Another lane's value, by one of the moves that vector instructions make on the way (data through LDS has ten times
// the latency, and the choices of a row are a chain of such moves).
template <int CTRL, typename T>
__device__ __forceinline__ T moved(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, static_cast<uint64_t>(moved<CTRL>(static_cast<uint32_t>(b >> 32))) << 32 | moved<CTRL>(static_cast<uint32_t>(b)));
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
    }
}
// Both 16-lane rows of each 32 lanes (ROWS) or both halves of the wave, each in every lane of the two, joined by f.
template <bool ROWS, typename T, typename F>
__device__ __forceinline__ T joined(T v, F&& f) {
    const auto swap = [](uint32_t w) {
        const auto r = ROWS ? __builtin_amdgcn_permlane16_swap(w, w, false, false) : __builtin_amdgcn_permlane32_swap(w, w, false, false);
        return u32x2v{r[0], r[1]};
    };
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const u32x2v hi = swap(static_cast<uint32_t>(b >> 32)), lo = swap(static_cast<uint32_t>(b));
        return f(__builtin_bit_cast(T, static_cast<uint64_t>(hi[0]) << 32 | lo[0]), __builtin_bit_cast(T, static_cast<uint64_t>(hi[1]) << 32 | lo[1]));
    } else {
        const u32x2v r = swap(__builtin_bit_cast(uint32_t, v));
        return f(__builtin_bit_cast(T, static_cast<uint32_t>(r[0])), __builtin_bit_cast(T, static_cast<uint32_t>(r[1])));
    }
}
// f over L lanes next to each other, in every one of them.
template <int L, typename T, typename F>
__device__ __forceinline__ T group_reduce(T v, F&& f) {
    if constexpr (L >= 2) v = f(v, moved<0xB1>(v));              // quad_perm 1,0,3,2
    if constexpr (L >= 4) v = f(v, moved<0x4E>(v));              // quad_perm 2,3,0,1
    if constexpr (L >= 8) v = f(v, moved<0x141>(v));             // row_half_mirror
    if constexpr (L >= 16) v = f(v, moved<0x140>(v));            // row_mirror
    if constexpr (L >= 32) v = joined<true>(v, f);
    if constexpr (L >= 64) v = joined<false>(v, f);
    return v;
}
// The sum over the lanes of a wave that have the same place in groups of L lanes, in every one of them.
template <int L>
__device__ __forceinline__ float sum_of_groups(float v) {
    if constexpr (L <= 1) v += moved<0xB1>(v);
    if constexpr (L <= 2) v += moved<0x4E>(v);
    if constexpr (L <= 4) v += moved<0x124>(v);                  // row_ror:4
    if constexpr (L <= 8) v += moved<0x128>(v);                  // row_ror:8
    const auto sum = [](float a, float b) { return a + b; };
    if constexpr (L <= 16) v = joined<true>(v, sum);
    if constexpr (L <= 32) v = joined<false>(v, sum);
    return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<L>(v, [](float a, float b) { return a + b; });
}

// e^d for d at most 0: 2^(d log2 e) by the target's instruction, with what the product lost put back, so
// about two units off over the whole range.  Not a number gives zero like -infinity: what a row with such a logit, or with
// +infinity, returns then follows from its sum of zero (1 / 0 times 0) or from its lse, neither of which is a number.
__device__ __forceinline__ float exp_of(float d) {
    constexpr float L = 1.44269504088896341f, LN2 = 0.69314718055994531f;
    d = fmaxf(d, -200.f);                                        // (e^-200 is zero; -infinity would leave no number in `lost`)
    const float t = d * L, lost = fmaf(d, L, -t), e = __builtin_amdgcn_exp2f(t);
    return fmaf(e * LN2, lost, e);
}

// A logit's bits in the order of its value: negative numbers below positive ones, both zeros equal, NaN above all.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x == x ? x + 0.f : __builtin_nanf(""));
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t ORDERED_MINUS_INF = 0x007fffffu;          // of -infinity

template <typename T>
struct Key;
template <>
struct Key<uint16_t> {
    typedef uint32_t type;
    static __device__ __forceinline__ type of(float x, int e) { return (ordered(x) & 0xffff0000u) | (0xffffu - static_cast<uint32_t>(e)); }
    static __device__ __forceinline__ int index(type k) { return static_cast<int>(0xffffu - (k & 0xffffu)); }
    // (-infinity and what is beyond the row: 0x007f in the upper half and below)
    static __device__ __forceinline__ bool available(type k) { return (k >> 16) > (ORDERED_MINUS_INF >> 16); }
    static __device__ __forceinline__ float value(type k) { return __uint_as_float(__float_as_uint(value_of(k)) & 0xffff0000u); }
};
template <>
struct Key<float> {
    typedef uint64_t type;
    static __device__ __forceinline__ type of(float x, int e) {
        return (static_cast<uint64_t>(ordered(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(e));
    }
    static __device__ __forceinline__ int index(type k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
    static __device__ __forceinline__ bool available(type k) { return static_cast<uint32_t>(k >> 32) > ORDERED_MINUS_INF; }
    static __device__ __forceinline__ float value(type k) { return value_of(static_cast<uint32_t>(k >> 32)); }
};

// Where a token's row of logits is, and whether it takes part.
template <typename T>
__device__ __forceinline__ const T* row_of(const MuonRoute& a, int64_t t) {
    return static_cast<const T*>(a.logits) + t * a.ld_logits;
}
__device__ __forceinline__ bool unmasked(const MuonRoute& a, int64_t t) { return t < a.tokens && (!a.mask || a.mask[t]); }

// A row's packs as they are requested, and its logits in fp32 once they are there: -infinity beyond the row and where the
// token takes no part.
template <typename T, int N>
struct RowPacks {
    static constexpr int G = pack_of<T>;
    Pack<T, G> v[N / G];
    __device__ __forceinline__ void load(const T* row, int base, int experts) {
#pragma unroll
        for (int g = 0; g < N / G; ++g) v[g] = request<T, G, false>(row, base + G * g, experts);
    }
    __device__ __forceinline__ void get(int base, int experts, bool in, float (&x)[N]) {
#pragma unroll
        for (int g = 0; g < N / G; ++g) {
            settle<T, G>(v[g], base + G * g, experts);
#pragma unroll
            for (int i = 0; i < G; ++i) x[G * g + i] = in && base + G * g + i < experts ? v[g][i] : -__builtin_inff();
        }
    }
};

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

// What lanes of a wave left in LDS is there for its other lanes (whose accesses are in order), for the compiler too.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr int RB_THREADS = 256;
constexpr int RB_GROUPS = 1024;            // workgroups: four for each CU, each set up once (65536 x 256: 20.8 us; 1536: 20.6, 2048: 22)
template <typename T, int N, int L>
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
        packs.get(base, E, on, x);
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            const f32x4v v = extra[sub][q * L + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[4 * q + i] = v[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = exp_of(x[i] - lse - rest);      // (zero where the token takes no part: x is -infinity)
            dot = fmaf(p[i], g[i], dot);
            if (!a.normalize) dot += u[i];         // p dw: what comes through the probabilities themselves
        }
        dot = group_sum<L>(dot);
        const float all = on ? fmaf(cz, lse, -dot) : 0.f;
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
            for (int i = 0; i < G; ++i) d[i] = fmaf(p[G * q + i], g[G * q + i] + all, u[G * q + i]);
            store_pack<T, G, false>(static_cast<T*>(a.dlogits) + t * E, base + G * q, E, Pack<T, G>::of(d));
        }
    }
}

template <int A, int B>
struct RouteShape {
    static constexpr int N = A, L = B;
};
template <typename F>
static void with_route_shape(int experts, F&& f) {
    if (experts <= 8) f(RouteShape<8, 1>{});
    else if (experts <= 16) f(RouteShape<8, 2>{});
    else if (experts <= 32) f(RouteShape<8, 4>{});
    else if (experts <= 64) f(RouteShape<8, 8>{});
    else if (experts <= 128) f(RouteShape<16, 8>{});
    else if (experts <= 256) f(RouteShape<16, 16>{});
    else if (experts <= 512) f(RouteShape<16, 32>{});
    else f(RouteShape<16, 64>{});
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
static int route_groups(int64_t tokens, int experts) {
    int rows = 1;
    with_route_shape(experts, [&](auto s) { rows = RT_THREADS / decltype(s)::L; });
    const int64_t n = (tokens + rows - 1) / rows;
    return static_cast<int>(n < RT_GROUPS ? n : RT_GROUPS);
}

static int check_route(const MuonRoute* a, const char* what) {
    MUON_REQUIRE(a, "%s: null arguments", what);
    MUON_REQUIRE(a->tokens > 0 && a->experts > 0 && a->experts <= RT_MAX_EXPERTS, "%s: tokens=%lld experts=%d (at most %d)", what,
                 static_cast<long long>(a->tokens), a->experts, RT_MAX_EXPERTS);
    MUON_REQUIRE(a->k > 0 && a->k <= a->experts && a->k <= RT_MAX_K, "%s: k=%d of %d experts (at most %d)", what, a->k, a->experts, RT_MAX_K);
    MUON_REQUIRE(a->logits && a->weights && a->indices && a->counts && a->part && a->lse && a->lse_rest, "%s: null pointer", what);
    MUON_REQUIRE(a->dtype == MUON_AMD_SRC_F32 || a->dtype == MUON_AMD_SRC_BF16, "%s: dtype=%d", what, a->dtype);
    return MUON_AMD_OK;
}


template <typename F>
static void with_route_type(int dtype, F&& f) {
    if (dtype == MUON_AMD_SRC_BF16) f(uint16_t{});
    else f(float{});
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
    hipLaunchKernelGGL(route_join_kernel, dim3((a.experts + RJ_EXPERTS - 1) / RJ_EXPERTS), dim3(RJ_THREADS), 0, st, a, n);
    return check_launch("route");
}

int muon_amd_route_backward(const MuonRoute* args, void* stream) {
    if (const int rc = check_route(args, "route_backward")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.dlogits, "route_backward: null output");
    with_route_type(a.dtype, [&](auto x) {
        with_route_backward_shape(a.experts, [&](auto s) {
            constexpr int ROWS = RB_THREADS / decltype(s)::L;
            const int64_t n = (a.tokens + ROWS - 1) / ROWS;
            hipLaunchKernelGGL((route_backward_kernel<decltype(x), decltype(s)::N, decltype(s)::L>), dim3(n < RB_GROUPS ? n : RB_GROUPS),
                               dim3(RB_THREADS), 0, static_cast<hipStream_t>(stream), a);
        });
    });
    return check_launch("route_backward");
}

}  // extern "C"
