// Values moved and joined between the lanes of a wave, and the exponential that the softmax kernels share.
#pragma once

#include "vector.h"

namespace muon_amd {

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

// What lanes of a wave left in LDS is there for its other lanes (whose accesses are in order), for the compiler too.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// e^d for d at most 0: 2^(d log2 e) by the target's instruction, with what the product's rounding lost put back.  What the constant's
// rounding lost is not (log2 e is 1.93e-8 larger than L): e^(d (1 - 1.34e-8)), larger than e^d by 0.22 |d| units of 2^-24 beside about three
// of the other roundings: 25 at the smallest normal number.  The order of two exponentials is that of their arguments all the same.  Not a number gives zero like -infinity: what a row with such a logit, or with
// +infinity, returns then follows from its sum of zero (1 / 0 times 0) or from its lse, neither of which is a number.
__device__ __forceinline__ float exp_of_bounded(float d) {       // (from -200 on)
    constexpr float L = 1.44269504088896341f, LN2 = 0.69314718055994531f;
    const float t = d * L, lost = fmaf(d, L, -t), e = __builtin_amdgcn_exp2f(t);
    return fmaf(e * LN2, lost, e);
}

// (e^-200 is zero; -infinity would leave no number in `lost`)
__device__ __forceinline__ float exp_of(float d) { return exp_of_bounded(fmaxf(d, -200.f)); }

// 1 / (1 + e^-x) and, with it, 1 / (1 + e^x): about five units off, relative to themselves, and the smaller one 0.22 |x| more, as e^-|x| is.  Not a
// number gives what is none.
__device__ __forceinline__ float sigmoid_of(float x, float& rest) {
    const float t = exp_of(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + t), small = t * r;
    rest = x >= 0.f ? small : r;
    return x != x ? x : x >= 0.f ? r : small;
}

}  // namespace muon_amd
