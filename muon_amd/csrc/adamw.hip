// AdamW over many tensors in one launch, with states in 32 or in 8 bits, and the values that 8-bit states stand for.
//
//   g' = c g;  m <- m + w1 (g' - m);  v <- v + w2 (g'^2 - v);  p <- p wd_factor - (lr / bias1) m / (sqrt(v / bias2) + eps)
//
// with c read from device memory (the coefficient of a clipped gradient) or 1.  Arithmetic is fp32 whatever p is stored
// in; p rounds once.
//
// States of 8 bits.  128 consecutive elements of a tensor (a block) share a power of two 2^(E - 127), E one byte, for
// each moment; an element keeps three bits of mantissa and its exponent below the shared one:
//   m: sign, four bits of exponent, 2^(E - 127) (1 + f/8) 2^(e - 15): the codes of OCP's e4m3, whose largest is 1.75 x 2^8
//   v: five bits of exponent, 2^(E - 127) (1 + f/8) 2^(e - 31), no sign
// (e = 0: f/8 of the lowest power, as in IEEE 754).  A power of two as the shared factor makes scaling exact, and E the
// exponent field of the largest magnitude of the block, one more where that element itself could round past the
// largest code.  E = 255 says that the block holds a value that is not finite: all of it reads as NaN, so an overflow
// shows in the next step as it would in 32 bits.
// Rounding to three bits is dithered: to the 20 bits that are dropped, 20 bits are added that go by the element's place
// in its tensor and by the step, as good as independent from step to step and between the moments, so that a moment is
// right on average.  To nearest, one that moves by less than half a step of its code (6 % of it; a step moves v by at
// most 1 - beta2 of itself) would never move; and a sequence that fills the unit interval evenly over the steps (multiples
// of an irrational number) leaves moments 2 % off, since what is rounded goes by the steps before.
// v above zero never rounds to the code zero, whose update would divide by eps alone.
#include <type_traits>

#include "vector.h"

namespace muon_amd {

constexpr int AW_THREADS = 256;
constexpr int AW_BLOCK_ELEMS = 8192;                            // elements of a block of the table
// Elements per thread, whose loads all go out first: 16, and two workgroups for each block, or 32 where codes go with fp32
// parameters.  (16 and 32: 32-bit states over 32000 x 2048 bf16 217 and 226 us, 8-bit states over 50257 x 768 bf16 67.6
// and 69.5, their values 40 and 43; 8-bit states over 128256 x 4096 fp32 1444 and 1391.)
constexpr int AW_EACH = 16, AW8_EACH_F32 = 32;
constexpr int workgroups_per_block(int each) { return AW_BLOCK_ELEMS / (AW_THREADS * each); }
constexpr int AW_SHARED = 128;                                  // elements that share an exponent

struct AdamWArgs {
    float neg_lr;        // -lr / bias1
    float wd_factor, w1, w2, eps;
    float rsqrt_bias2;   // 1 / sqrt(bias2)
    uint32_t dither;     // of the step
};

// The dither of element i at step t: h = i D + mix(t) mod 2^32, x the low 24 bits of h ^ (h >> 15), and of the products
// of x with a constant for each moment (24-bit factors: the target's fast integer product) bits 12 to 31.
constexpr uint32_t DITHER_I = 0x9E3779B9u, DITHER_M = 0xC13FA9u, DITHER_V = 0x91E10Du;
__host__ __device__ __forceinline__ uint32_t mix_step(uint32_t t) {
    uint32_t x = t * 0x9E3779B9u;
    x = (x ^ (x >> 16)) * 0xC13FA9A9u;
    x = (x ^ (x >> 15)) * 0x91E10DA5u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ AdamWArgs read_args(AdamWArgs a, const float* sc) {
    if (sc) {   // {lr, wd_factor, w1, w2, eps, bias1, bias2, step} read at run time instead of the arguments
        a.neg_lr = -sc[0] / sc[5];
        a.wd_factor = sc[1];
        a.w1 = sc[2];
        a.w2 = sc[3];
        a.eps = sc[4];
        a.rsqrt_bias2 = 1.f / sqrtf(sc[6]);
        a.dither = mix_step(static_cast<uint32_t>(sc[7]));
    }
    return a;
}

// The two moments; the square is rounded before it is subtracted from, as for tensors of fp32.  A weight of a half and
// more is taken from the other end, new + (w - 1)(new - old), which is `new` itself for w = 1.  ORDINARY: neither weight is
// (the two selections for each element are then left out).
template <bool ORDINARY>
__device__ __forceinline__ float lerp_from(float old, float now, float w) {
    const bool far = !ORDINARY && fabsf(w) >= 0.5f;
    return fmaf(far ? w - 1.f : w, now - old, far ? now : old);
}
template <bool ORDINARY>
__device__ __forceinline__ void moments(float& m, float& v, float g, const AdamWArgs& a) {
#pragma clang fp contract(off)
    const float gg = g * g;
    m = lerp_from<ORDINARY>(m, g, a.w1);
    v = lerp_from<ORDINARY>(v, gg, a.w2);
}
// Whether the arguments are those of an ordinary run, for which 8-bit states have a kernel path of their own: small weights, and
// an eps beside which the root of a subnormal v (below 2^-63) is lost, so that the path may take it for zero.  (131 M fp32
// elements: 347 us that way, 367 the other; 39 M in bf16: 68 both ways.)
__device__ __forceinline__ bool ordinary(const AdamWArgs& a) {
    return fabsf(a.w1) < 0.5f && fabsf(a.w2) < 0.5f && a.eps >= 0x1p-39f * a.rsqrt_bias2;
}

// ---- states in 32 bits -------------------------------------------------------------------------------------
// Memory bounds it: 22 bytes an element with bf16 parameters, 28 with fp32 (32000 x 2048 bf16: 218 us, 6.6 TB/s).  Lists of small
// tensors are one launch's latency (49 of 768: 3.9 us).
template <typename T>
__device__ __forceinline__ void adamw32_pack(Pack<T, 4>& p, const Pack<T, 4>& g, Pack<float, 4>& m, Pack<float, 4>& v, float c,
                                             const AdamWArgs& a) {
    float pn[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float mk = m[k], vk = v[k];
        moments<false>(mk, vk, g[k] * c, a);
        m.v[k] = mk;
        v.v[k] = vk;
        pn[k] = fmaf(a.neg_lr, mk / fmaf(sqrtf(vk), a.rsqrt_bias2, a.eps), p[k] * a.wd_factor);
    }
    p = Pack<T, 4>::of(pn);
}

template <typename T>
__device__ __forceinline__ void adamw32_block(const MuonAdamWDesc& d, int64_t base, float c, const AdamWArgs& a) {
    constexpr int PACKS = AW_EACH / 4, ELEMS = AW_THREADS * AW_EACH;
    const int64_t numel = d.numel;
    T* __restrict__ const p = static_cast<T*>(d.param);
    const T* __restrict__ const g = static_cast<const T*>(d.grad);
    float* __restrict__ const m = static_cast<float*>(d.exp_avg);
    float* __restrict__ const v = static_cast<float*>(d.exp_avg_sq);
    if (base + ELEMS <= numel) {
        Pack<T, 4> pv[PACKS], gv[PACKS];
        Pack<float, 4> mv[PACKS], vv[PACKS];
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int64_t e = base + (i * AW_THREADS + threadIdx.x) * 4;
            gv[i] = Pack<T, 4>::template load<true>(g + e);
            mv[i] = Pack<float, 4>::load<true>(m + e);
            vv[i] = Pack<float, 4>::load<true>(v + e);
            pv[i] = Pack<T, 4>::template load<true>(p + e);
        }
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int64_t e = base + (i * AW_THREADS + threadIdx.x) * 4;
            adamw32_pack<T>(pv[i], gv[i], mv[i], vv[i], c, a);
            mv[i].store<true>(m + e);
            vv[i].store<true>(v + e);
            pv[i].template store<true>(p + e);
        }
        return;
    }
#pragma unroll 1
    for (int64_t e = base + threadIdx.x * 4; e < numel && e < base + ELEMS; e += AW_THREADS * 4) {
        Pack<T, 4> pv = load_pack<T, 4, true>(p, e, numel);
        const Pack<T, 4> gv = load_pack<T, 4, true>(g, e, numel);
        Pack<float, 4> mv = load_pack<float, 4, true>(m, e, numel), vv = load_pack<float, 4, true>(v, e, numel);
        adamw32_pack<T>(pv, gv, mv, vv, c, a);
        store_pack<float, 4, true>(m, e, numel, mv);
        store_pack<float, 4, true>(v, e, numel, vv);
        store_pack<T, 4, true>(p, e, numel, pv);
    }
}

// DTYPE: the type of every parameter of the launch, or AW_MIXED.  A kernel for both types takes the registers of the
// larger half (fp32 in packs of four), and 8-bit states over 50257 x 768 bf16 took 80 us in it, 69 in one of their own.
constexpr int AW_MIXED = -1;
template <int DTYPE, typename F>
__device__ __forceinline__ void with_type(const MuonAdamWDesc& d, F&& f) {
    if (DTYPE == MUON_AMD_SRC_BF16 || (DTYPE == AW_MIXED && d.dtype == MUON_AMD_SRC_BF16)) f(uint16_t{});
    else f(float{});
}

template <int DTYPE>
__global__ __launch_bounds__(AW_THREADS) void adamw32_kernel(const MuonAdamWDesc* __restrict__ descs,
                                                            const int32_t* __restrict__ prefix, int ntensors, AdamWArgs args,
                                                            const float* __restrict__ grad_scale, const float* __restrict__ sc) {
    const AdamWArgs a = read_args(args, sc);
    const float c = grad_scale ? *grad_scale : 1.f;
    constexpr int PARTS = workgroups_per_block(AW_EACH);
    const int b = blockIdx.x / PARTS, ti = find_segment_wave(prefix, ntensors, b);
    const MuonAdamWDesc d = descs[ti];
    const int64_t base = static_cast<int64_t>(b - prefix[ti]) * AW_BLOCK_ELEMS + blockIdx.x % PARTS * (AW_THREADS * AW_EACH);
    with_type<DTYPE>(d, [&](auto t) { adamw32_block<decltype(t)>(d, base, c, a); });
}

// ---- states in 8 bits --------------------------------------------------------------------------------------
// 10 bytes an element with bf16 parameters and 16 with fp32, in one pass: 50257 x 768 bf16 68 us (5.7 TB/s), where arithmetic
// and memory take about as long as each other, and 128256 x 4096 fp32 1405 us (6.0 TB/s).  Codes are read and written with
// the non-temporal hint (without: 1536 against 1424 us at that time).
// The larger of two pairs of 16-bit numbers over LANES (16 or 32) lanes next to each other, in every lane.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max2(uint32_t x) {
    const auto larger = [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
    };
    x = larger(x, __builtin_amdgcn_mov_dpp(x, 0xB1, 0xf, 0xf, true));       // quad_perm 1,0,3,2
    x = larger(x, __builtin_amdgcn_mov_dpp(x, 0x4E, 0xf, 0xf, true));       // quad_perm 2,3,0,1
    x = larger(x, __builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true));      // row_half_mirror
    x = larger(x, __builtin_amdgcn_mov_dpp(x, 0x140, 0xf, 0xf, true));      // row_mirror
    if constexpr (LANES == 32) {
        const auto rows = __builtin_amdgcn_permlane16_swap(x, x, false, false);       // even rows twice, odd rows twice
        x = larger(rows[0], rows[1]);
    }
    return x;
}

// G codes of one byte each, as words.
template <int G>
struct Codes {
    typedef uint32_t words __attribute__((ext_vector_type(G / 4)));
    typedef uint32_t words_any __attribute__((ext_vector_type(G / 4), aligned(1)));
    words w;
    static __device__ __forceinline__ Codes load(const uint8_t* p) { return {load_as<true, words_any>(p)}; }
    __device__ __forceinline__ void store(uint8_t* p) const { store_as<true, words_any>(p, w); }
    static __device__ __forceinline__ Codes load(const uint8_t* p, int64_t e, int64_t n) {
        if (e + G <= n) return load(p + e);
        Codes c{words(0u)};
#pragma unroll
        for (int k = 0; k < G - 1; ++k)
            if (e + k < n) c.w[k >> 2] |= static_cast<uint32_t>(p[e + k]) << (8 * (k & 3));
        return c;
    }
    __device__ __forceinline__ void store(uint8_t* p, int64_t e, int64_t n) const {
        if (e + G <= n) {
            store(p + e);
            return;
        }
#pragma unroll
        for (int k = 0; k < G - 1; ++k)
            if (e + k < n) p[e + k] = static_cast<uint8_t>(w[k >> 2] >> (8 * (k & 3)));
    }
};

// The values of codes, as they are held (m) or (v), whose block has the shared exponent E.
template <int G>
__device__ __forceinline__ void decode_m(const Codes<G>& c, int E, float (&m)[G]) {
#pragma unroll
    for (int h = 0; h < G / 4; ++h) {
        const uint32_t w = c.w[h];
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        m[4 * h] = ldexpf(lo[0], E - 135);            // (e4m3 itself: 2^(e - 7))
        m[4 * h + 1] = ldexpf(lo[1], E - 135);
        m[4 * h + 2] = ldexpf(hi[0], E - 135);
        m[4 * h + 3] = ldexpf(hi[1], E - 135);
    }
}
template <int G>
__device__ __forceinline__ void decode_v(const Codes<G>& c, int E, float (&v)[G]) {
#pragma unroll
    for (int k = 0; k < G; ++k) v[k] = ldexpf(__uint_as_float(((c.w[k >> 2] >> (8 * (k & 3))) & 0xffu) << 20), E - 31);
}

// The top bytes of four words, in their order.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&w)[4]) {
    return __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0703u) | __builtin_amdgcn_perm(w[3], w[2], 0x07030c0cu);
}

// The root of v by the target's instruction, which is a unit off and takes subnormal numbers for zero; they are scaled up
// unless ORDINARY allows that.  (A unit each of the root and of the reciprocal below is a relative 2^-22 of an update that
// goes by codes of three bits; the correctly rounded ones of the 32-bit states are about 20 instructions longer.)
template <bool ORDINARY>
__device__ __forceinline__ float root(float v) {
    if (ORDINARY) return __builtin_amdgcn_sqrtf(v);
    const bool low = v < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(low ? v * 0x1p32f : v) * (low ? 0x1p-16f : 1.f);
}

// One pack: parameters and moments after the step, the new codes, and the new shared exponents of its block, which is
// that of 128 / G lanes (every lane of the wave calls this; what is beyond the tensor is zero).
// Its arithmetic (about 40 instructions an element) takes nearly as long as bf16 parameters take to move: so codes are rounded where they end up in the top
// byte of a word (the magnitude's bits and the dither's, both four bits higher than the code's own place), four of
// which two byte permutations collect, and zeros among the codes of v are looked for four at a time.
template <typename T, int G, bool ORDINARY>
__device__ __forceinline__ void adamw8_pack(Pack<T, G>& p, const Pack<T, G>& g, Codes<G>& mc, Codes<G>& vc, int& Em, int& Ev,
                                            uint32_t i0, float c, const AdamWArgs& a) {
    float m[G], v[G], pn[G];
    decode_m<G>(mc, Em, m);
    decode_v<G>(vc, Ev, v);
    const float poison = max(Em, Ev) == 255 ? __builtin_nanf("") : 0.f;
    float most_m = 0.f;
    uint32_t most_v = 0;
#pragma unroll
    for (int k = 0; k < G; ++k) {
        const float gk = fmaf(g[k], c, poison);
        moments<ORDINARY>(m[k], v[k], gk, a);
        most_m = fmaxf(most_m, fabsf(m[k]));
        most_v = max(most_v, __float_as_uint(v[k]));         // (the bits, so that NaN counts; m is not finite only where v is not)
        const float denominator = fmaf(root<ORDINARY>(v[k]), a.rsqrt_bias2, a.eps);
        pn[k] = fmaf(a.neg_lr, m[k] * __builtin_amdgcn_rcpf(denominator), p[k] * a.wd_factor);
    }
    p = Pack<T, G>::of(pn);
    most_v = min(most_v, 0x7fffffffu);                       // (a NaN's sign and the carry would wrap around to a small exponent)
    // exponent fields, one more where three bits of mantissa are not enough below the next power (m: 1.75 is the last)
    const uint32_t both = lanes_max2<AW_SHARED / G>(((__float_as_uint(most_m) + 0x1fffffu) >> 23) | ((most_v + 0xfffffu) >> 23 << 16));
    Em = static_cast<int>(both & 0xffffu);
    Ev = static_cast<int>(both >> 16);
    if (max(Em, Ev) >= 255) Em = Ev = 255;
    uint32_t h32 = i0 * DITHER_I + a.dither;
#pragma unroll
    for (int h = 0; h < G / 4; ++h) {
        uint32_t sm[4], sv[4], signs[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float mk = m[4 * h + k], vk = v[4 * h + k];
            const uint32_t x = (h32 ^ (h32 >> 15)) & 0xffffffu;
            // (the bits of a product below the dither's 20 change no code: they end below the magnitude's lowest)
            sm[k] = (__float_as_uint(ldexpf(fabsf(mk), 15 - Em)) << 4) + (x * DITHER_M >> 8);
            sv[k] = (__float_as_uint(ldexpf(vk, 31 - Ev)) << 4) + (x * DITHER_V >> 8);
            signs[k] = __float_as_uint(mk);
            h32 += DITHER_I;
        }
        mc.w[h] = top_bytes(sm) | (top_bytes(signs) & 0x80808080u);
        uint32_t cv = top_bytes(sv);
        if ((cv - 0x01010101u) & ~cv & 0x80808080u)           // a code is zero: the least one unless v is zero itself
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (!(cv >> (8 * k) & 0xffu) && v[4 * h + k] != 0.f) cv |= 1u << (8 * k);
        vc.w[h] = cv;
    }
}

template <typename T, int EACH, bool ORDINARY>
__device__ __forceinline__ void adamw8_block(const MuonAdamWDesc& d, int64_t base, float c, const AdamWArgs& a) {
    constexpr int G = pack_of<T>, PACKS = EACH / G, LANES = AW_SHARED / G, ELEMS = AW_THREADS * EACH;
    const int64_t numel = d.numel;
    T* __restrict__ const p = static_cast<T*>(d.param);
    const T* __restrict__ const g = static_cast<const T*>(d.grad);
    uint8_t* __restrict__ const m = static_cast<uint8_t*>(d.exp_avg);
    uint8_t* __restrict__ const v = static_cast<uint8_t*>(d.exp_avg_sq);
    uint8_t* __restrict__ const me = d.exp_avg_exponent;
    uint8_t* __restrict__ const ve = d.exp_avg_sq_exponent;
    if (base + ELEMS <= numel) {
        Pack<T, G> pv[PACKS], gv[PACKS];
        Codes<G> mv[PACKS], vv[PACKS];
        int Em[PACKS], Ev[PACKS];
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int64_t e = base + (i * AW_THREADS + threadIdx.x) * G;
            Em[i] = load_as<false, uint8_t>(me + e / AW_SHARED);
            Ev[i] = load_as<false, uint8_t>(ve + e / AW_SHARED);
            mv[i] = Codes<G>::load(m + e);
            vv[i] = Codes<G>::load(v + e);
            gv[i] = Pack<T, G>::template load<true>(g + e);
            pv[i] = Pack<T, G>::template load<true>(p + e);
        }
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int64_t e = base + (i * AW_THREADS + threadIdx.x) * G;
            adamw8_pack<T, G, ORDINARY>(pv[i], gv[i], mv[i], vv[i], Em[i], Ev[i], static_cast<uint32_t>(e), c, a);
            mv[i].store(m + e);
            vv[i].store(v + e);
            pv[i].template store<true>(p + e);
            if ((threadIdx.x & (LANES - 1)) == 0) {
                store_as<false, uint8_t>(me + e / AW_SHARED, static_cast<uint8_t>(Em[i]));
                store_as<false, uint8_t>(ve + e / AW_SHARED, static_cast<uint8_t>(Ev[i]));
            }
        }
        return;
    }
#pragma unroll 1
    for (int64_t at = base; at < numel && at < base + ELEMS; at += AW_THREADS * G) {      // (the wave stays whole: its lanes exchange maxima)
        const int64_t e = at + threadIdx.x * G;
        const bool any = e < numel;
        int Em = any ? me[e / AW_SHARED] : 0, Ev = any ? ve[e / AW_SHARED] : 0;
        Codes<G> mv = Codes<G>::load(m, e, numel), vv = Codes<G>::load(v, e, numel);
        Pack<T, G> pv = load_pack<T, G, true>(p, e, numel);
        const Pack<T, G> gv = load_pack<T, G, true>(g, e, numel);
        adamw8_pack<T, G, ORDINARY>(pv, gv, mv, vv, Em, Ev, static_cast<uint32_t>(e), c, a);
        mv.store(m, e, numel);
        vv.store(v, e, numel);
        store_pack<T, G, true>(p, e, numel, pv);
        if (any && (threadIdx.x & (LANES - 1)) == 0) {
            me[e / AW_SHARED] = static_cast<uint8_t>(Em);
            ve[e / AW_SHARED] = static_cast<uint8_t>(Ev);
        }
    }
}

constexpr int adamw8_each(int dtype) { return dtype == MUON_AMD_SRC_BF16 ? AW_EACH : AW8_EACH_F32; }
template <int DTYPE>
__global__ __launch_bounds__(AW_THREADS) void adamw8_kernel(const MuonAdamWDesc* __restrict__ descs,
                                                           const int32_t* __restrict__ prefix, int ntensors, AdamWArgs args,
                                                           const float* __restrict__ grad_scale, const float* __restrict__ sc) {
    const AdamWArgs a = read_args(args, sc);
    const float c = grad_scale ? *grad_scale : 1.f;
    constexpr int EACH = adamw8_each(DTYPE), PARTS = workgroups_per_block(EACH);
    const int b = blockIdx.x / PARTS, ti = find_segment_wave(prefix, ntensors, b);
    const MuonAdamWDesc d = descs[ti];
    const int64_t base = static_cast<int64_t>(b - prefix[ti]) * AW_BLOCK_ELEMS + blockIdx.x % PARTS * (AW_THREADS * EACH);
    with_type<DTYPE>(d, [&](auto t) {
        if (ordinary(a)) adamw8_block<decltype(t), EACH, true>(d, base, c, a);
        else adamw8_block<decltype(t), EACH, false>(d, base, c, a);
    });
}

// The values of 8-bit states in bf16, which holds each of them exactly down to the least one that it has (three bits of
// mantissa; only blocks below 2^-100 reach bf16's own subnormal numbers).  Memory bounds it, 2 bytes in and 4 out (50257 x 768 40 us,
// 128256 x 4096 555 us: 5.7 TB/s); all loads ahead of the stores, 32 elements a thread or the non-temporal hint change nothing.
__global__ __launch_bounds__(AW_THREADS) void adamw_values_kernel(const MuonAdamWValuesDesc* __restrict__ descs,
                                                                 const int32_t* __restrict__ prefix, int ntensors) {
    constexpr int PARTS = workgroups_per_block(AW_EACH);
    const int b = blockIdx.x / PARTS, ti = find_segment_wave(prefix, ntensors, b);
    const MuonAdamWValuesDesc d = descs[ti];
    const int64_t base = static_cast<int64_t>(b - prefix[ti]) * AW_BLOCK_ELEMS + blockIdx.x % PARTS * (AW_THREADS * AW_EACH), numel = d.numel;
#pragma unroll
    for (int i = 0; i < AW_EACH / 8; ++i) {
        const int64_t e = base + (i * AW_THREADS + threadIdx.x) * 8;
        if (e >= numel) return;
        const int Em = load_as<false, uint8_t>(d.exp_avg_exponent + e / AW_SHARED), Ev = load_as<false, uint8_t>(d.exp_avg_sq_exponent + e / AW_SHARED);
        float m[8], v[8];
        decode_m<8>(Codes<8>::load(d.exp_avg, e, numel), Em, m);
        decode_v<8>(Codes<8>::load(d.exp_avg_sq, e, numel), Ev, v);
        if (Em == 255)
            for (float& x : m) x = __builtin_nanf("");
        if (Ev == 255)
            for (float& x : v) x = __builtin_nanf("");
        store_pack<uint16_t, 8, false>(d.exp_avg_out, e, numel, Pack<uint16_t, 8>::of(m));
        store_pack<uint16_t, 8, false>(d.exp_avg_sq_out, e, numel, Pack<uint16_t, 8>::of(v));
    }
}

// Checks a table's block prefix against its tensors' sizes.
template <typename D>
static int check_prefix(const char* what, const D* descs, int n, const int32_t* prefix) {
    MUON_REQUIRE(descs && prefix, "%s: null table", what);
    MUON_REQUIRE(n > 0, "%s: ntensors=%d", what, n);
    MUON_REQUIRE(prefix[0] == 0, "%s: prefix must start at 0", what);
    for (int i = 0; i < n; ++i) {
        MUON_REQUIRE(descs[i].numel > 0, "%s: tensor %d: numel=%lld", what, i, static_cast<long long>(descs[i].numel));
        const int64_t nblk = (descs[i].numel + AW_BLOCK_ELEMS - 1) / AW_BLOCK_ELEMS;
        MUON_REQUIRE(static_cast<int64_t>(prefix[i + 1]) - prefix[i] == nblk, "%s: tensor %d: prefix gives %d blocks, need %lld", what,
                     i, prefix[i + 1] - prefix[i], static_cast<long long>(nblk));
    }
    return MUON_AMD_OK;
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_adamw_desc(void) { return sizeof(MuonAdamWDesc); }
size_t muon_amd_sizeof_adamw_values_desc(void) { return sizeof(MuonAdamWValuesDesc); }
int muon_amd_adamw_shared_elems(void) { return AW_SHARED; }

int muon_amd_validate_adamw(const MuonAdamWDesc* descs, int ntensors, const int32_t* prefix, int state_bits) {
    MUON_REQUIRE(state_bits == 8 || state_bits == 32, "validate_adamw: state_bits=%d", state_bits);
    if (const int rc = check_prefix("validate_adamw", descs, ntensors, prefix)) return rc;
    for (int i = 0; i < ntensors; ++i) {
        const MuonAdamWDesc& d = descs[i];
        MUON_REQUIRE(d.param && d.grad && d.exp_avg && d.exp_avg_sq, "validate_adamw: tensor %d: null pointer", i);
        MUON_REQUIRE(state_bits == 32 || (d.exp_avg_exponent && d.exp_avg_sq_exponent),
                     "validate_adamw: tensor %d: states in 8 bits need their exponents", i);
        MUON_REQUIRE(d.dtype == MUON_AMD_SRC_F32 || d.dtype == MUON_AMD_SRC_BF16, "validate_adamw: tensor %d: dtype=%d", i, d.dtype);
        const uintptr_t elem = d.dtype == MUON_AMD_SRC_BF16 ? 2 : 4;
        MUON_REQUIRE(reinterpret_cast<uintptr_t>(d.param) % elem == 0 && reinterpret_cast<uintptr_t>(d.grad) % elem == 0 &&
                         (state_bits == 8 || (reinterpret_cast<uintptr_t>(d.exp_avg) % 4 == 0 &&
                                              reinterpret_cast<uintptr_t>(d.exp_avg_sq) % 4 == 0)),
                     "validate_adamw: tensor %d: address not a multiple of the element's size", i);
    }
    return MUON_AMD_OK;
}

int muon_amd_validate_adamw_values(const MuonAdamWValuesDesc* descs, int ntensors, const int32_t* prefix) {
    if (const int rc = check_prefix("validate_adamw_values", descs, ntensors, prefix)) return rc;
    for (int i = 0; i < ntensors; ++i) {
        const MuonAdamWValuesDesc& d = descs[i];
        MUON_REQUIRE(d.exp_avg && d.exp_avg_sq && d.exp_avg_exponent && d.exp_avg_sq_exponent && d.exp_avg_out && d.exp_avg_sq_out,
                     "validate_adamw_values: tensor %d: null pointer", i);
        MUON_REQUIRE(reinterpret_cast<uintptr_t>(d.exp_avg_out) % 2 == 0 && reinterpret_cast<uintptr_t>(d.exp_avg_sq_out) % 2 == 0,
                     "validate_adamw_values: tensor %d: address not a multiple of the element's size", i);
    }
    return MUON_AMD_OK;
}

int muon_amd_adamw(const MuonAdamWDesc* descs_dev, const int32_t* block_prefix_dev, int ntensors, int nblocks, int dtype, int state_bits,
                   float lr, float wd_factor, float w1, float w2, float eps, float bias1, float bias2, uint32_t step,
                   const float* grad_scale_dev, const float* scalars_dev, void* stream) {
    MUON_REQUIRE(descs_dev && block_prefix_dev, "adamw: null table");
    MUON_REQUIRE(ntensors > 0 && nblocks > 0, "adamw: ntensors=%d nblocks=%d", ntensors, nblocks);
    MUON_REQUIRE(state_bits == 8 || state_bits == 32, "adamw: state_bits=%d", state_bits);
    MUON_REQUIRE(dtype == MUON_AMD_SRC_F32 || dtype == MUON_AMD_SRC_BF16 || dtype == AW_MIXED, "adamw: dtype=%d", dtype);
    MUON_REQUIRE(scalars_dev || (bias1 != 0.f && bias2 > 0.f), "adamw: zero bias correction");
    const AdamWArgs a{-lr / bias1, wd_factor, w1, w2, eps, 1.f / sqrtf(bias2), mix_step(step)};
    const auto pick = [&](auto f32, auto bf16, auto mixed) { return dtype == MUON_AMD_SRC_F32 ? f32 : dtype == MUON_AMD_SRC_BF16 ? bf16 : mixed; };
    const auto kernel = state_bits == 8
                            ? pick(adamw8_kernel<MUON_AMD_SRC_F32>, adamw8_kernel<MUON_AMD_SRC_BF16>, adamw8_kernel<AW_MIXED>)
                            : pick(adamw32_kernel<MUON_AMD_SRC_F32>, adamw32_kernel<MUON_AMD_SRC_BF16>, adamw32_kernel<AW_MIXED>);
    const int parts = workgroups_per_block(state_bits == 8 ? adamw8_each(dtype) : AW_EACH);
    MUON_REQUIRE(nblocks <= INT32_MAX / parts, "adamw: nblocks=%d", nblocks);
    hipLaunchKernelGGL(kernel, dim3(nblocks * parts), dim3(AW_THREADS), 0, static_cast<hipStream_t>(stream), descs_dev, block_prefix_dev,
                       ntensors, a, grad_scale_dev, scalars_dev);
    return check_launch("adamw");
}

int muon_amd_adamw_values(const MuonAdamWValuesDesc* descs_dev, const int32_t* block_prefix_dev, int ntensors, int nblocks,
                          void* stream) {
    MUON_REQUIRE(descs_dev && block_prefix_dev, "adamw_values: null table");
    MUON_REQUIRE(ntensors > 0 && nblocks > 0, "adamw_values: ntensors=%d nblocks=%d", ntensors, nblocks);
    MUON_REQUIRE(nblocks <= INT32_MAX / workgroups_per_block(AW_EACH), "adamw_values: nblocks=%d", nblocks);
    hipLaunchKernelGGL(adamw_values_kernel, dim3(nblocks * workgroups_per_block(AW_EACH)), dim3(AW_THREADS), 0, static_cast<hipStream_t>(stream), descs_dev,
                       block_prefix_dev, ntensors);
    return check_launch("adamw_values");
}

}  // extern "C"
