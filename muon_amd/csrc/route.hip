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
// Sums over tokens: each lane adds the probabilities of its experts over its rows, a workgroup joins its lanes in a
// fixed order, and a second launch joins the workgroups; counts are whole numbers, in any order the same.
#include <type_traits>

#include "vector.h"

namespace muon_amd {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_K = 32;
constexpr int RT_THREADS = 256;
constexpr int RT_GROUPS = 512;             // workgroups at most: their partial sums are joined by one launch

// The value of `v` in the lane a power of two away, within groups of L lanes.
template <typename T>
__device__ __forceinline__ T lane_xor(T v, int mask) {
    return __shfl_xor(v, mask, 64);
}
template <int L, typename T, typename F>
__device__ __forceinline__ T group_reduce(T v, F&& f) {
#pragma unroll
    for (int m = 1; m < L; m <<= 1) v = f(v, lane_xor(v, m));
    return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    return group_reduce<L>(v, [](float a, float b) { return a + b; });
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

template <typename T, int N, int L>
__device__ __forceinline__ void load_row(const T* row, int base, int experts, bool in, float (&x)[N]) {
    constexpr int G = pack_of<T>;
#pragma unroll
    for (int g = 0; g < N / G; ++g) {
        const Pack<T, G> v = load_pack<T, G, false>(row, base + G * g, in ? experts : 0);
#pragma unroll
        for (int i = 0; i < G; ++i) x[G * g + i] = in && base + G * g + i < experts ? v[i] : -__builtin_inff();
    }
}

// partials: workgroups x experts pairs {sum of p, tokens}, then workgroups x {sum of lse^2, tokens that take part}.
template <typename T, int N, int L>
__global__ __launch_bounds__(RT_THREADS) void route_forward_kernel(const MuonRoute a) {
    constexpr int ROWS = RT_THREADS / L;
    typedef Key<T> K;
    __shared__ float sums[ROWS][N * L + 1];
    __shared__ int tokens[N * L];
    __shared__ float squares[RT_THREADS / 64];
    __shared__ int parts[RT_THREADS / 64];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, base = lane * N, E = a.experts;
    for (int e = threadIdx.x; e < N * L; e += RT_THREADS) tokens[e] = 0;
    __syncthreads();
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    float square = 0.f;
    int part = 0;
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.tokens; first += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t t = first + sub;
        const bool in = unmasked(a, t);
        float x[N];
        load_row<T, N, L>(row_of<T>(a, t), base, E, in, x);
        typename K::type key[N];
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = K::of(x[i], base + i);
        // The k largest, one after the other (all keys differ and there are at least k, so this never wraps around).  Lane
        // j mod L takes choice j; where there are more choices than lanes, it leaves the earlier ones unscaled.
        typename K::type best = 0;
        float top = 0.f, chosen = 0.f, my_part = 0.f;
        int my_expert = -1;
        bool on = false;
        for (int j = 0; j < a.k; ++j) {
            typename K::type m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m = max(m, static_cast<typename K::type>(key[i] - best));
            m = group_reduce<L>(m, [](typename K::type u, typename K::type v) { return max(u, v); });
            best += m;
            const bool there = in && K::available(best);
            if (j == 0) {
                on = there;
                top = K::value(best);
            }
            const float ex = there ? expf(K::value(best) - top) : 0.f;
            chosen += ex;
            if (lane == j % L) {
                my_part = ex;
                my_expert = there ? K::index(best) : -1;
                if (there) atomicAdd(&tokens[my_expert], 1);
                if (j + L < a.k && t < a.tokens) {
                    a.weights[t * a.k + j] = my_part;
                    a.indices[t * a.k + j] = my_expert;
                }
            }
        }
        // softmax over the row
        float ex[N], total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            ex[i] = on ? expf(x[i] - top) : 0.f;
            total += ex[i];
        }
        total = group_sum<L>(total);
        const float lse = on ? top + logf(total) : 0.f, per = on ? 1.f / total : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(ex[i], per, acc[i]);
        if (t >= a.tokens) continue;
        const float scale = on ? (a.normalize ? 1.f / chosen : per) : 0.f;
        for (int j = lane; j < a.k; j += L) {
            const bool last = j + L >= a.k;
            a.weights[t * a.k + j] = (last ? my_part : a.weights[t * a.k + j]) * scale;
            if (last) a.indices[t * a.k + j] = my_expert;
        }
        if (lane == 0) {
            a.lse[t] = on ? lse : -__builtin_inff();
            square = fmaf(lse, lse, square);
            part += on;
        }
    }
    // join the workgroup's rows
#pragma unroll
    for (int i = 0; i < N; ++i) sums[sub][base + i] = acc[i];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        square += lane_xor(square, m);
        part += lane_xor(part, m);
    }
    if ((threadIdx.x & 63) == 0) {
        squares[threadIdx.x >> 6] = square;
        parts[threadIdx.x >> 6] = part;
    }
    __syncthreads();
    float* const out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * E;
    for (int e = threadIdx.x; e < E; e += RT_THREADS) {
        float s = 0.f;
        for (int r = 0; r < ROWS; ++r) s += sums[r][e];
        out[2 * e] = s;
        out[2 * e + 1] = __int_as_float(tokens[e]);
    }
    if (threadIdx.x == 0) {
        float* const tail = a.partials + static_cast<int64_t>(gridDim.x) * 2 * E + 2 * blockIdx.x;
        tail[0] = (squares[0] + squares[1]) + (squares[2] + squares[3]);
        tail[1] = __int_as_float((parts[0] + parts[1]) + (parts[2] + parts[3]));
    }
}

// One workgroup joins the partial sums: counts, both losses, and the number of tokens that take part.
constexpr int RJ_THREADS = 1024;
__global__ __launch_bounds__(RJ_THREADS) void route_join_kernel(const MuonRoute a, int groups) {
    __shared__ float psum[RJ_THREADS];
    __shared__ int csum[RJ_THREADS];
    __shared__ float red[RJ_THREADS / 64];
    __shared__ float shared_square;
    __shared__ int shared_part;
    const int E = a.experts;
    // shares of the workgroups for each expert: a power of two that fills the launch
    int width = 64;
    while (width < E) width <<= 1;
    const int shares = RJ_THREADS / width, e = threadIdx.x % width, share = threadIdx.x / width;
    float p = 0.f;
    int c = 0;
    if (e < E) {
        const f32x2_t* const at = reinterpret_cast<const f32x2_t*>(a.partials) + e;
        int g = share;
        for (; g + 7 * shares < groups; g += 8 * shares) {       // (eight loads on their way at once: one at a time took 36 us)
            f32x2_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at[static_cast<int64_t>(g + i * shares) * E];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p += v[i][0];
                c += __float_as_int(v[i][1]);
            }
        }
        for (; g < groups; g += shares) {
            const f32x2_t v = at[static_cast<int64_t>(g) * E];
            p += v[0];
            c += __float_as_int(v[1]);
        }
    }
    psum[threadIdx.x] = p;
    csum[threadIdx.x] = c;
    if (threadIdx.x < 64) {
        const float* const tail = a.partials + static_cast<int64_t>(groups) * 2 * E;
        float s = 0.f;
        int n = 0;
        for (int g = threadIdx.x; g < groups; g += 64) {
            s += tail[2 * g];
            n += __float_as_int(tail[2 * g + 1]);
        }
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
            s += lane_xor(s, m);
            n += lane_xor(n, m);
        }
        if (threadIdx.x == 0) {
            shared_square = s;
            shared_part = n;
        }
    }
    __syncthreads();
    float dot = 0.f;
    if (share == 0 && e < E) {
        for (int o = 1; o < shares; ++o) {
            p += psum[o * width + e];
            c += csum[o * width + e];
        }
        a.counts[e] = c;
        dot = static_cast<float>(c) * p;
    }
    dot = wave_sum(dot);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        float total = 0.f;
        for (int w = 0; w < RJ_THREADS / 64; ++w) total += red[w];
        const float n = static_cast<float>(shared_part > 0 ? shared_part : 1);
        *a.balance = static_cast<float>(E) * (total / (n * static_cast<float>(a.k))) / n;
        *a.z = shared_square / n;
        *a.part = n;
    }
}

// What lanes of a wave left in LDS is there for its other lanes (whose accesses are in order), for the compiler too.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T, int N, int L>
__global__ __launch_bounds__(RT_THREADS) void route_backward_kernel(const MuonRoute a) {
    constexpr int ROWS = RT_THREADS / L, G = pack_of<T>;
    __shared__ float extra[ROWS][N * L + 4];          // what the weights' gradients add, by expert
    const int lane = threadIdx.x % L, sub = threadIdx.x / L, base = lane * N, E = a.experts;
    const float n = *a.part;
    const float cb = a.dbalance ? *a.dbalance * static_cast<float>(E) / (n * n * static_cast<float>(a.k)) : 0.f;
    const float cz = a.dz ? *a.dz * 2.f / n : 0.f;
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        g[i] = base + i < E ? cb * static_cast<float>(a.counts[base + i]) : 0.f;
        extra[sub][base + i] = 0.f;
    }
    wave_order();
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.tokens; first += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t t = first + sub;
        const float lse = t < a.tokens ? a.lse[t] : -__builtin_inff();
        const bool on = lse != -__builtin_inff();
        float x[N];
        load_row<T, N, L>(row_of<T>(a, t), base, E, on, x);
        // the weights' part: lanes of the row take the k choices in turn
        if (a.dweights && on) {
            float dot = 0.f;
            for (int j = lane; j < a.k; j += L) dot = fmaf(a.weights[t * a.k + j], a.dweights[t * a.ld_dweights + j], dot);
            dot = a.normalize ? group_sum<L>(dot) : 0.f;
            for (int j = lane; j < a.k; j += L) {
                const int e = a.indices[t * a.k + j];
                if (e >= 0) extra[sub][e] = a.weights[t * a.k + j] * (a.dweights[t * a.ld_dweights + j] - dot);
            }
        }
        wave_order();
        float p[N], u[N], dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            p[i] = on ? expf(x[i] - lse) : 0.f;
            u[i] = extra[sub][base + i];
            dot = fmaf(p[i], g[i], dot);
            if (!a.normalize) dot += u[i];         // p dw: what comes through the probabilities themselves
        }
        dot = group_sum<L>(dot);
        const float all = on ? fmaf(cz, lse, -dot) : 0.f;
        wave_order();
        if (a.dweights && on)
            for (int j = lane; j < a.k; j += L) {
                const int e = a.indices[t * a.k + j];
                if (e >= 0) extra[sub][e] = 0.f;
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
    MUON_REQUIRE(a->logits && a->weights && a->indices && a->counts && a->part && a->lse, "%s: null pointer", what);
    MUON_REQUIRE(a->dtype == MUON_AMD_SRC_F32 || a->dtype == MUON_AMD_SRC_BF16, "%s: dtype=%d", what, a->dtype);
    return MUON_AMD_OK;
}


template <typename F>
static void with_route(const MuonRoute& a, F&& f) {
    with_route_shape(a.experts, [&](auto s) {
        if (a.dtype == MUON_AMD_SRC_BF16) f(uint16_t{}, s);
        else f(float{}, s);
    });
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_route(void) { return sizeof(MuonRoute); }
int muon_amd_route_max_experts(void) { return RT_MAX_EXPERTS; }
int muon_amd_route_max_k(void) { return RT_MAX_K; }

int64_t muon_amd_route_partials(int64_t tokens, int experts) {
    if (tokens <= 0 || experts <= 0 || experts > RT_MAX_EXPERTS) return 0;
    return static_cast<int64_t>(route_groups(tokens, experts)) * 2 * (experts + 1);
}

int muon_amd_route(const MuonRoute* args, void* stream) {
    if (const int rc = check_route(args, "route")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.partials && a.balance && a.z, "route: null workspace or output");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = route_groups(a.tokens, a.experts);
    with_route(a, [&](auto x, auto s) {
        hipLaunchKernelGGL((route_forward_kernel<decltype(x), decltype(s)::N, decltype(s)::L>), dim3(n), dim3(RT_THREADS), 0, st, a);
    });
    if (const int rc = check_launch("route")) return rc;
    hipLaunchKernelGGL(route_join_kernel, dim3(1), dim3(RJ_THREADS), 0, st, a, n);
    return check_launch("route");
}

int muon_amd_route_backward(const MuonRoute* args, void* stream) {
    if (const int rc = check_route(args, "route_backward")) return rc;
    const MuonRoute a = *args;
    MUON_REQUIRE(a.dlogits, "route_backward: null output");
    with_route(a, [&](auto x, auto s) {
        constexpr int ROWS = RT_THREADS / decltype(s)::L;
        const int64_t n = (a.tokens + ROWS - 1) / ROWS;
        hipLaunchKernelGGL((route_backward_kernel<decltype(x), decltype(s)::N, decltype(s)::L>), dim3(n < 2048 ? n : 2048), dim3(RT_THREADS),
                           0, static_cast<hipStream_t>(stream), a);
    });
    return check_launch("route_backward");
}

}  // extern "C"
