// What the routing kernels share: keys that order logits, rows in registers, the shapes of launches.
#pragma once

#include <type_traits>

#include "lanes.h"

namespace muon_amd {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_K = 32;
constexpr int RT_THREADS = 512;
constexpr int RT_WAVES = RT_THREADS / 64;
constexpr int RT_GROUPS = 512;             // workgroups at most: their partial sums are joined by one launch

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
    // (zeros beyond the row)
    __device__ __forceinline__ void get(int base, int experts, float (&x)[N]) {
#pragma unroll
        for (int g = 0; g < N / G; ++g) {
            settle<T, G>(v[g], base + G * g, experts);
#pragma unroll
            for (int i = 0; i < G; ++i) x[G * g + i] = v[g][i];
        }
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

// Joins what `groups` workgroups of a forward launch left (route.hip).
int launch_route_join(const MuonRoute& a, int groups, hipStream_t stream);

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
