// Packs of four or eight elements in their storage type (fp32, or bf16 as uint16_t) at any element address, as the
// streaming kernels move them.  The target's vector accesses take any address.
//
// A pack is 16 bytes or less (eight fp32 elements are two packs of four): lanes then lie next to each other in every
// access.  Eight fp32 elements per lane as two accesses 32 bytes apart touch each line twice, with the non-temporal hint
// once too early: AdamW with 32-bit states over 32000 x 2048 bf16 took 341 us that way.
#pragma once

#include "common.h"

namespace muon_amd {

typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));
typedef float f32x4v_any __attribute__((ext_vector_type(4), aligned(4)));

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

// G elements of T.
template <typename T, int G>
struct Pack;

template <>
struct Pack<float, 4> {
    f32x4v v;
    __device__ __forceinline__ float operator[](int k) const { return v[k]; }
    static __device__ __forceinline__ Pack zero() { return {f32x4v{0.f, 0.f, 0.f, 0.f}}; }
    template <bool NT>
    static __device__ __forceinline__ Pack load(const float* p) {
        return {load_as<NT, f32x4v_any>(p)};
    }
    template <bool NT>
    __device__ __forceinline__ void store(float* p) const {
        store_as<NT, f32x4v_any>(p, v);
    }
    __device__ __forceinline__ void put(int k, float x) { v[k] = x; }         // an element in storage, as it is loaded
    __device__ __forceinline__ float get(int k) const { return v[k]; }
    static __device__ __forceinline__ Pack of(const float (&x)[4]) { return {f32x4v{x[0], x[1], x[2], x[3]}}; }
};

template <int G>
struct Pack<uint16_t, G> {
    typedef uint32_t words __attribute__((ext_vector_type(G / 2)));
    typedef uint32_t words_any __attribute__((ext_vector_type(G / 2), aligned(2)));
    words v;
    __device__ __forceinline__ float operator[](int k) const { return k & 1 ? bf_hi(v[k >> 1]) : bf_lo(v[k >> 1]); }
    static __device__ __forceinline__ Pack zero() { return {words(0u)}; }
    template <bool NT>
    static __device__ __forceinline__ Pack load(const uint16_t* p) {
        return {load_as<NT, words_any>(p)};
    }
    template <bool NT>
    __device__ __forceinline__ void store(uint16_t* p) const {
        store_as<NT, words_any>(p, v);
    }
    __device__ __forceinline__ void put(int k, uint16_t x) { v[k >> 1] |= static_cast<uint32_t>(x) << (16 * (k & 1)); }
    __device__ __forceinline__ uint16_t get(int k) const { return static_cast<uint16_t>(v[k >> 1] >> (16 * (k & 1))); }
    static __device__ __forceinline__ Pack of(const float (&x)[G]) {
        Pack p;
#pragma unroll
        for (int k = 0; k < G / 2; ++k) p.v[k] = pack2bf(x[2 * k], x[2 * k + 1]);
        return p;
    }
};

// The pack at element e of a row (tensor) of n elements: whole, its first n - e elements and zeros, or zeros.
template <typename T, int G, bool NT, typename I>
__device__ __forceinline__ Pack<T, G> load_pack(const T* p, I e, I n) {
    if (e + G <= n) return Pack<T, G>::template load<NT>(p + e);
    Pack<T, G> g = Pack<T, G>::zero();
    if (e < n)                      // (lanes beyond the row do not walk through the elements)
#pragma unroll
        for (int k = 0; k < G - 1; ++k)
            if (e + k < n) g.put(k, p[e + k]);
    return g;
}
template <typename T, int G, bool NT, typename I>
__device__ __forceinline__ void store_pack(T* p, I e, I n, const Pack<T, G>& g) {
    if (e + G <= n) {
        g.template store<NT>(p + e);
        return;
    }
    if (e < n)
#pragma unroll
        for (int k = 0; k < G - 1; ++k)
            if (e + k < n) p[e + k] = g.get(k);
}

// The pack at element c of a row of `width`.  It is requested whole and without a branch, from where it lies in the row
// (the last one of a row that ends within it: from its last G elements), so that all loads of a row go out
// together; settle() then moves what a lane at the end of the row got to its place, with zeros beyond the row.  (With a
// branch at each load residual_norm over 5003 x 1600 took 46 us backward, and 38 without.)
template <typename T, int G, bool NT>
__device__ __forceinline__ Pack<T, G> request(const T* row, int c, int width) {
    if (width < G) return load_pack<T, G, NT>(row, c, width);
    return Pack<T, G>::template load<NT>(row + min(c, width - G));
}
template <typename T, int G>
__device__ __forceinline__ void settle(Pack<T, G>& v, int c, int width) {
    if (width < G || c + G <= width) return;
    const int shift = min(c - (width - G), G);
#pragma unroll
    for (int by = 1; by <= G; by <<= 1) {
        Pack<T, G> moved = Pack<T, G>::zero();
#pragma unroll
        for (int k = 0; k + by < G; ++k) moved.put(k, v.get(k + by));
        if (shift & by) v = moved;
    }
}

// Elements of a pack where T decides alone: 16 bytes.
template <typename T>
constexpr int pack_of = 16 / sizeof(T);

}  // namespace muon_amd
