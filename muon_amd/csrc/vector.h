// Groups of eight elements in their storage type (fp32, or bf16 as uint16_t) at any element address, as the streaming
// kernels move them: 16 bytes of bf16, twice 16 bytes of fp32.  The target's vector accesses take any address.
#pragma once

#include "common.h"

namespace muon_amd {

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef float f32x4v_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4v_any __attribute__((ext_vector_type(4), aligned(2)));

#define MUON_GLOBAL __attribute__((address_space(1)))

// NT: the non-temporal hint, for what this launch touches once and nothing reads soon.
template <bool NT, typename V, typename P>
__device__ __forceinline__ V load_as(const P* p) {
    const MUON_GLOBAL V* const q = (const MUON_GLOBAL V*)(p);
    return NT ? __builtin_nontemporal_load(q) : *q;
}
template <bool NT, typename V, typename P>
__device__ __forceinline__ void store_as(P* p, V v) {
    MUON_GLOBAL V* const q = (MUON_GLOBAL V*)(p);
    if (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
}

template <typename T>
struct Group8;

template <>
struct Group8<float> {
    f32x4v a, b;
    __device__ __forceinline__ float operator[](int k) const { return k < 4 ? a[k] : b[k - 4]; }
    __device__ __forceinline__ void set(int k, float v) {
        if (k < 4) a[k] = v;
        else b[k - 4] = v;
    }
    static __device__ __forceinline__ Group8 zero() { return {f32x4v{0.f, 0.f, 0.f, 0.f}, f32x4v{0.f, 0.f, 0.f, 0.f}}; }
    template <bool NT>
    static __device__ __forceinline__ Group8 load(const float* p) {
        return {load_as<NT, f32x4v_any>(p), load_as<NT, f32x4v_any>(p + 4)};
    }
    // the first n of the eight (the others zero)
    static __device__ __forceinline__ Group8 load_first(const float* p, int n) {
        Group8 g = zero();
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (k < n) g.set(k, p[k]);
        return g;
    }
    template <bool NT>
    __device__ __forceinline__ void store(float* p) const {
        store_as<NT, f32x4v_any>(p, a);
        store_as<NT, f32x4v_any>(p + 4, b);
    }
    __device__ __forceinline__ void store_first(float* p, int n) const {
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (k < n) p[k] = (*this)[k];
    }
    // eight values in this storage type
    static __device__ __forceinline__ Group8 of(const float (&v)[8]) {
        return {f32x4v{v[0], v[1], v[2], v[3]}, f32x4v{v[4], v[5], v[6], v[7]}};
    }
};

template <>
struct Group8<uint16_t> {
    u32x4v v;
    __device__ __forceinline__ float operator[](int k) const { return k & 1 ? bf_hi(v[k >> 1]) : bf_lo(v[k >> 1]); }
    static __device__ __forceinline__ Group8 zero() { return {u32x4v{0u, 0u, 0u, 0u}}; }
    template <bool NT>
    static __device__ __forceinline__ Group8 load(const uint16_t* p) {
        return {load_as<NT, u32x4v_any>(p)};
    }
    static __device__ __forceinline__ Group8 load_first(const uint16_t* p, int n) {
        Group8 g = zero();
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (k < n) g.v[k >> 1] |= static_cast<uint32_t>(p[k]) << (16 * (k & 1));
        return g;
    }
    template <bool NT>
    __device__ __forceinline__ void store(uint16_t* p) const {
        store_as<NT, u32x4v_any>(p, v);
    }
    __device__ __forceinline__ void store_first(uint16_t* p, int n) const {
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (k < n) p[k] = static_cast<uint16_t>(v[k >> 1] >> (16 * (k & 1)));
    }
    static __device__ __forceinline__ Group8 of(const float (&x)[8]) {
        return {u32x4v{pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(x[4], x[5]), pack2bf(x[6], x[7])}};
    }
};

// The group at element e of a row (tensor) of n elements: whole, its first n - e elements, or nothing.
template <typename T, bool NT>
__device__ __forceinline__ Group8<T> load_group(const T* p, int64_t e, int64_t n) {
    if (e + 8 <= n) return Group8<T>::template load<NT>(p + e);
    return Group8<T>::load_first(p + e, e < n ? static_cast<int>(n - e) : 0);
}
template <typename T, bool NT>
__device__ __forceinline__ void store_group(T* p, int64_t e, int64_t n, const Group8<T>& g) {
    if (e + 8 <= n) g.template store<NT>(p + e);
    else if (e < n) g.store_first(p + e, static_cast<int>(n - e));
}

}  // namespace muon_amd
