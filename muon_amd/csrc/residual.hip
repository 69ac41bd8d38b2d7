// The step between two blocks of a transformer, with its gradients: the norm after a block, its gate and residual
// scale, the addition to the residual stream, and the norm before the next block.  Per row (token) of D channels:
//   nb = b rb,  rb = (mean(b^2) + eps)^-1/2;   h = x + s sig(z) nb wpost
//   nh = h rh,  rh = (mean(h^2) + eps)^-1/2;   y = nh wpre
// and backward, from the gradients dh and dy of both results, with k = s wpost:
//   e  = dh + rh dy wpre,  c1 = mean(dy wpre nh),  dx = e - rh c1 nh
//   c2 = mean(dx k sig nb),  db = rb (dx k sig - c2 nb),  dz = dx k nb sig (1 - sig)
//   q  = sum over rows of dx sig nb:  dwpost = s q,  ds = wpost q;   dwpre = sum over rows of dy nh
// All sums are fp32 whatever the tensors are stored in; h enters the second norm and the gradients unrounded (the
// backward pass forms it again from x and b, which costs what reading it would), so that the gradients of the vectors are
// as exact as the inputs.  c2 follows from sums that do not wait for c1 (dx is linear in it):
//   D c2 = sum(e k sig nb) - rh c1 sum(nh k sig nb)
// so that a row takes one reduction; the gradient of a gate for the whole row is (1 - sig) D c2.
//
// Memory bounds both passes (16384 x 4096 bf16 with a gate per element: forward 119 us, 5.6 TB/s; backward 195 us, 5.5 TB/s; their
// bytes at 6.5 TB/s: 103 and 165).  Backward is at the registers' limit: the next row ahead of time spills, fewer registers
// recompute; and from 5121 channels on (a workgroup of 768 threads and more, 128 registers each) some kernels spill as they are, 1
// to 10 registers of a lane, above 8192 (16 channels a thread) all of them, 49 to 98.  A row stays in the registers of TPR threads (one wave up to 1024 channels forward, 512
// backward: no barrier), 16 bytes of the residual stream per access; a workgroup takes row after row with the weights of
// its channels in LDS and, backward, their sums in registers; the workgroups' sums are joined in a fixed order by a second launch (7 us).
#include <type_traits>

#include "vector.h"

namespace muon_amd {

enum { GATE_NONE = MUON_AMD_GATE_NONE, GATE_TOKEN = MUON_AMD_GATE_TOKEN, GATE_CHANNEL = MUON_AMD_GATE_CHANNEL };
constexpr int RN_MAX_WIDTH = 16384;
constexpr int RN_THREADS = 256;            // of a workgroup, more where a row needs them

// The sum over the 64 lanes, in every lane.
__device__ __forceinline__ float lanes_sum(float v) {
    const auto other = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    v += other(v, std::integral_constant<int, 0xB1>{});      // quad_perm 1,0,3,2
    v += other(v, std::integral_constant<int, 0x4E>{});      // quad_perm 2,3,0,1
    v += other(v, std::integral_constant<int, 0x141>{});     // row_half_mirror
    v += other(v, std::integral_constant<int, 0x140>{});     // row_mirror
    const auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
    return (row(0) + row(16)) + (row(32) + row(48));
}

// Sums over the threads of a row.  Rows of one wave need no barrier; else every wave leaves its sums in one of two sets of
// slots, which the caller alternates between (one barrier a sum: who writes a set again has passed the barrier after
// which the others read it).
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float (*slots)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = lanes_sum(s[k]);
    if constexpr (TPR > 64) {
        constexpr int WAVES = TPR / 64;                  // (a power of two where rows share a workgroup)
        const int wave = threadIdx.x >> 6, first = TPR < RN_THREADS ? wave & ~(WAVES - 1) : 0;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) slots[wave][k] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) t += slots[first + w][k];
            s[k] = t;
        }
    }
}

// The gate of logits stored as B.  exp(-z) by the target's power of two alone is off by 2^-24 |z| relative to itself (60 units at
// -80): 2^-15 of what a bf16 logit's own rounding makes of it, but more than an fp32 result should be, so
// fp32 logits take the exact one (8192 x 2048 all in fp32: 59 us forward and 100 backward both ways; for bf16 logits beside an
// fp32 stream it would cost 2 to 7 %).  Below -87.3, where the gate is no normal number, it is zero.  1 - sigmoid, which the
// gate's gradient takes, has the rounding of one: 2^-24 absolute.
template <typename B>
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + (sizeof(B) == 4 ? expf(-z) : __expf(-z)));
}

// A pack's elements of a vector of weights in fp32 (zero beyond the row).
template <int G>
__device__ __forceinline__ void load_weights(const void* p, int dtype, int c, int width, float (&w)[G]) {
    if (dtype == MUON_AMD_SRC_BF16) {
        const Pack<uint16_t, G> g = load_pack<uint16_t, G, false>(static_cast<const uint16_t*>(p), c, width);
#pragma unroll
        for (int k = 0; k < G; ++k) w[k] = g[k];
    } else {
        #pragma unroll
        for (int h = 0; h < G; h += 4) {
            const Pack<float, 4> g = load_pack<float, 4, false>(static_cast<const float*>(p), c + h, width);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[h + k] = g[k];
        }
    }
}
__device__ __forceinline__ float load_one(const void* p, int dtype, int64_t i) {
    return dtype == MUON_AMD_SRC_BF16 ? bf2f(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_one(void* p, int dtype, int64_t i, float v) {
    if (dtype == MUON_AMD_SRC_BF16) static_cast<uint16_t*>(p)[i] = f2bf(v);
    else static_cast<float*>(p)[i] = v;
}
// The scale of a pack's channels: one per channel, one for all, or none.
template <int G>
__device__ __forceinline__ void load_scale(const MuonResidualNorm& a, int c, float (&s)[G]) {
    if (a.scale && !a.scale_is_one) {
        load_weights(a.scale, a.weight_dtype, c, a.width, s);
        return;
    }
    const float one = a.scale ? load_one(a.scale, a.weight_dtype, 0) : 1.f;
#pragma unroll
    for (int k = 0; k < G; ++k) s[k] = one;
}

// The weights of a workgroup's channels, which it uses for row after row: k = scale * post_weight, and pre_weight.  They
// wait in LDS (128 KB for the widest row; 32 bytes of reads per 8 elements and row, far below what LDS gives;
// conflict-free: four channels of a thread next to those of the next), which leaves room for more waves in the registers:
// with the weights there 8192 x 8192 bf16 took 254 us backward instead of 205.
template <int TPR, int V, int G>
struct Weights {
    static constexpr int QUADS = V * G / 4;
    f32x4v* shared;                        // [2][QUADS][TPR]

    __device__ __forceinline__ void load(const MuonResidualNorm& a, f32x4v* space) {
        shared = space;
        const int t = threadIdx.x % TPR;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            float s[G], post[G], pre[G];
            load_scale<G>(a, c, s);
            load_weights<G>(a.post_weight, a.weight_dtype, c, a.width, post);
            load_weights<G>(a.pre_weight, a.weight_dtype, c, a.width, pre);
#pragma unroll
            for (int i = 0; i < G; ++i) post[i] *= s[i];
            if (threadIdx.x < TPR)
#pragma unroll
                for (int h = 0; h < G / 4; ++h) {
                    shared[(j * (G / 4) + h) * TPR + t] = f32x4v{post[4 * h], post[4 * h + 1], post[4 * h + 2], post[4 * h + 3]};
                    shared[(QUADS + j * (G / 4) + h) * TPR + t] = f32x4v{pre[4 * h], pre[4 * h + 1], pre[4 * h + 2], pre[4 * h + 3]};
                }
        }
        __syncthreads();
    }
    template <int WHICH>
    __device__ __forceinline__ void get(int j, float (&out)[G]) const {
#pragma unroll
        for (int h = 0; h < G / 4; ++h) {
            const f32x4v v = shared[(WHICH * QUADS + j * (G / 4) + h) * TPR + threadIdx.x % TPR];
#pragma unroll
            for (int i = 0; i < 4; ++i) out[4 * h + i] = v[i];
        }
    }
};

// A result that is larger than what the memory-side cache keeps of a launch goes out with the non-temporal hint, so that it
// does not push out what is still to be read: 16384 x 4096 bf16 6 % longer without the hint forward and 4 % backward; with everything
// in the cache the hint costs (8192 x 2048: 26.2 -> 28.6 and 39.9 -> 42.5 us).
constexpr int64_t RN_CACHE = 256ll << 20;
template <typename T, int G>
__device__ __forceinline__ void store_row(T* p, int c, int n, const Pack<T, G>& g, bool nt) {
    if (nt) store_pack<T, G, true>(p, c, n, g);
    else store_pack<T, G, false>(p, c, n, g);
}

template <typename X, typename B, int GATE, int TPR, int V, int G>
__global__ __launch_bounds__(TPR > RN_THREADS ? TPR : RN_THREADS) void residual_forward_kernel(const MuonResidualNorm a, const bool nt) {
    constexpr int THREADS = TPR > RN_THREADS ? TPR : RN_THREADS, ROWS = THREADS / TPR;
    __shared__ float slots[2][THREADS / 64][1];
    const int t = threadIdx.x % TPR, width = a.width;
    typedef Weights<TPR, V, G> W;
    __shared__ f32x4v weights[2 * W::QUADS * TPR];
    W w;
    w.load(a, weights);
    const float per = 1.f / static_cast<float>(width);
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.rows; first += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t place = first + (ROWS > 1 ? threadIdx.x / TPR : 0);
        const bool in = ROWS == 1 || place < a.rows;              // (rows of several waves meet at barriers)
        const int64_t row = in ? place : a.rows - 1;
        const int n = in ? width : 0;
        const X* const x = static_cast<const X*>(a.x) + row * a.ld_x;
        const B* const b = static_cast<const B*>(a.b) + row * a.ld_b;
        const B* const z = static_cast<const B*>(a.gate) + row * a.ld_gate;
        Pack<X, G> xv[V];
        Pack<B, G> bv[V], zv[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            bv[j] = request<B, G, true>(b, c, width);
            xv[j] = request<X, G, true>(x, c, width);
            if constexpr (GATE == GATE_CHANNEL) zv[j] = request<B, G, true>(z, c, width);
        }
        float whole = 1.f;
        if constexpr (GATE == GATE_TOKEN) whole = sigmoid<B>(load_one(a.gate, a.block_dtype, row * a.ld_gate));
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            settle<B, G>(bv[j], c, width);
            settle<X, G>(xv[j], c, width);
            if constexpr (GATE == GATE_CHANNEL) settle<B, G>(zv[j], c, width);
        }
        float sum[1] = {0.f};
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < G; ++i) sum[0] = fmaf(bv[j][i], bv[j][i], sum[0]);
        row_sums<TPR, 1>(sum, slots[0]);
        const float rb = 1.f / sqrtf(fmaf(sum[0], per, a.eps));
        float h[V][G];
        sum[0] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            float k[G];
            w.template get<0>(j, k);
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const float sig = GATE == GATE_CHANNEL ? sigmoid<B>(zv[j][i]) : whole;
                h[j][i] = fmaf(bv[j][i] * rb, k[i] * sig, xv[j][i]);
                if (c + i < width) sum[0] = fmaf(h[j][i], h[j][i], sum[0]);
            }
            store_row<X, G>(static_cast<X*>(a.h) + row * width, c, n, Pack<X, G>::of(h[j]), nt);
        }
        row_sums<TPR, 1>(sum, slots[1]);
        const float rh = 1.f / sqrtf(fmaf(sum[0], per, a.eps));
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            float y[G], wpre[G];
            w.template get<1>(j, wpre);
#pragma unroll
            for (int i = 0; i < G; ++i) y[i] = h[j][i] * rh * wpre[i];
            store_row<B, G>(static_cast<B*>(a.y) + row * width, c, n, Pack<B, G>::of(y), nt);
        }
        if (in && t == 0 && a.rstd) {
            a.rstd[2 * row] = rb;
            a.rstd[2 * row + 1] = rh;
        }
    }
}

// (Four waves per SIMD where a workgroup's size allows them: 5003 x 1600 with an fp32 stream 66 -> 47 us.)
template <typename X, typename B, int GATE, int TPR, int V, int G>
__global__ __launch_bounds__(TPR > RN_THREADS ? TPR : RN_THREADS, 4) void residual_backward_kernel(const MuonResidualNorm a, const bool nt) {
    constexpr int THREADS = TPR > RN_THREADS ? TPR : RN_THREADS, ROWS = THREADS / TPR;
    __shared__ float slots[2][THREADS / 64][3];
    const int t = threadIdx.x % TPR, width = a.width;
    typedef Weights<TPR, V, G> W;
    __shared__ f32x4v weights[2 * W::QUADS * TPR];
    W w;
    w.load(a, weights);
    float q[V][G], r[V][G];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < G; ++i) q[j][i] = r[j][i] = 0.f;
    const float per = 1.f / static_cast<float>(width);
    int set = 0;
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * ROWS; first < a.rows; first += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t place = first + (ROWS > 1 ? threadIdx.x / TPR : 0);
        const bool in = ROWS == 1 || place < a.rows;
        const int64_t row = in ? place : a.rows - 1;
        const int n = in ? width : 0;
        const X* const x = static_cast<const X*>(a.x) + row * a.ld_x;
        const B* const b = static_cast<const B*>(a.b) + row * a.ld_b;
        const B* const z = static_cast<const B*>(a.gate) + row * a.ld_gate;
        Pack<X, G> xv[V], dhv[V];
        Pack<B, G> bv[V], zv[V], dyv[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            bv[j] = request<B, G, true>(b, c, width);
            xv[j] = request<X, G, true>(x, c, width);
            if constexpr (GATE == GATE_CHANNEL) zv[j] = request<B, G, true>(z, c, width);
            // (without the gradient of one result any row stands in for it, and is then taken for zeros)
            dyv[j] = request<B, G, true>(a.dy ? static_cast<const B*>(a.dy) + row * a.ld_dy : b, c, width);
            dhv[j] = request<X, G, true>(a.dh ? static_cast<const X*>(a.dh) + row * a.ld_dh : x, c, width);
        }
        const float rb = a.rstd[2 * row], rh = a.rstd[2 * row + 1];
        float whole = 1.f;
        if constexpr (GATE == GATE_TOKEN) whole = sigmoid<B>(load_one(a.gate, a.block_dtype, row * a.ld_gate));
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            settle<B, G>(bv[j], c, width);
            settle<X, G>(xv[j], c, width);
            if constexpr (GATE == GATE_CHANNEL) settle<B, G>(zv[j], c, width);
            settle<B, G>(dyv[j], c, width);
            settle<X, G>(dhv[j], c, width);
            if (!a.dy) dyv[j] = Pack<B, G>::zero();
            if (!a.dh) dhv[j] = Pack<X, G>::zero();
        }
        float sums[3] = {0.f, 0.f, 0.f};
        float nh[V][G], e[V][G], sig[V][G];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float k[G], wpre[G];
            w.template get<0>(j, k);
            w.template get<1>(j, wpre);
#pragma unroll
            for (int i = 0; i < G; ++i) {
                sig[j][i] = GATE == GATE_CHANNEL ? sigmoid<B>(zv[j][i]) : whole;
                const float kk = k[i] * sig[j][i], nb = bv[j][i] * rb;
                nh[j][i] = fmaf(nb, kk, xv[j][i]) * rh;
                const float dn = dyv[j][i] * wpre[i];
                e[j][i] = fmaf(rh, dn, dhv[j][i]);
                sums[0] = fmaf(dn, nh[j][i], sums[0]);
                sums[1] = fmaf(e[j][i] * kk, nb, sums[1]);
                sums[2] = fmaf(nh[j][i] * kk, nb, sums[2]);
                if (in) r[j][i] = fmaf(dyv[j][i], nh[j][i], r[j][i]);      // (a row that stands in for one beyond the last adds nothing)
            }
        }
        row_sums<TPR, 3>(sums, slots[set]);
        set ^= 1;
        const float c1 = sums[0] * per * rh, dc2 = fmaf(-c1, sums[2], sums[1]), c2 = dc2 * per;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * TPR + t) * G;
            float dx[G], db[G], dz[G], k[G];
            w.template get<0>(j, k);
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const float nb = bv[j][i] * rb, kk = k[i] * sig[j][i];
                dx[i] = fmaf(-c1, nh[j][i], e[j][i]);
                db[i] = rb * fmaf(dx[i], kk, -c2 * nb);
                const float g = dx[i] * nb;
                if (in) q[j][i] = fmaf(g, sig[j][i], q[j][i]);
                dz[i] = g * kk * (1.f - sig[j][i]);
            }
            if (a.dx) store_row<X, G>(static_cast<X*>(a.dx) + row * width, c, n, Pack<X, G>::of(dx), nt);
            if (a.db) store_row<B, G>(static_cast<B*>(a.db) + row * width, c, n, Pack<B, G>::of(db), nt);
            if constexpr (GATE == GATE_CHANNEL)
                if (a.dgate) store_row<B, G>(static_cast<B*>(a.dgate) + row * width, c, n, Pack<B, G>::of(dz), nt);
        }
        if constexpr (GATE == GATE_TOKEN)
            if (in && t == 0 && a.dgate) store_one(a.dgate, a.block_dtype, row, (1.f - whole) * dc2);
    }
    // sums of this workgroup: its rows' threads one after the other, through LDS where there is more than one
    if (!a.partials) return;
    float* const out = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * width;
    if constexpr (ROWS > 1) {
        __shared__ float joined[ROWS - 1][2][V][G][TPR];
        const int sub = threadIdx.x / TPR;
        if (sub > 0)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    joined[sub - 1][0][j][i][t] = q[j][i];
                    joined[sub - 1][1][j][i][t] = r[j][i];
                }
        __syncthreads();
        if (sub > 0) return;
        for (int o = 0; o < ROWS - 1; ++o)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    q[j][i] += joined[o][0][j][i][t];
                    r[j][i] += joined[o][1][j][i][t];
                }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (j * TPR + t) * G;
#pragma unroll
        for (int h = 0; h < G; h += 4) {
            store_pack<float, 4, false>(out, c + h, width, Pack<float, 4>{f32x4v{q[j][h], q[j][h + 1], q[j][h + 2], q[j][h + 3]}});
            store_pack<float, 4, false>(out + width, c + h, width, Pack<float, 4>{f32x4v{r[j][h], r[j][h + 1], r[j][h + 2], r[j][h + 3]}});
        }
    }
}

// The sums over the workgroups: RS_COLUMNS columns of q or r per workgroup, RS_SHARES shares of the partial rows, each
// of which reads four rows at a time, joined in order.  What bounds it is latency: 64 columns and 16 shares (few
// workgroups with long shares) took 18 us for 1024 partial rows of 2048.
constexpr int RS_COLUMNS = 16, RS_SHARES = 64;
__global__ __launch_bounds__(RS_COLUMNS * RS_SHARES) void residual_columns_kernel(const MuonResidualNorm a, int npartials,
                                                                                  float* __restrict__ one) {
    __shared__ float part[RS_SHARES][RS_COLUMNS];
    const int lane = threadIdx.x % RS_COLUMNS, share = threadIdx.x / RS_COLUMNS, width = a.width;
    const int c = blockIdx.x * RS_COLUMNS + lane, which = blockIdx.y;            // 0: q, 1: r
    float s = 0.f;
    if (c < width) {
        const float* const from = a.partials + static_cast<int64_t>(which) * width + c;
        const int64_t step = 2 * static_cast<int64_t>(width);
        int g = share;
        for (; g + 3 * RS_SHARES < npartials; g += 4 * RS_SHARES) {
            const float p0 = from[g * step], p1 = from[(g + RS_SHARES) * step], p2 = from[(g + 2 * RS_SHARES) * step],
                        p3 = from[(g + 3 * RS_SHARES) * step];
            s += (p0 + p1) + (p2 + p3);
        }
        for (; g < npartials; g += RS_SHARES) s += from[g * step];
    }
    part[share][lane] = s;
    __syncthreads();
    for (int half = RS_SHARES / 2; half >= 64 / RS_COLUMNS; half >>= 1) {
        if (share < half) part[share][lane] += part[share + half][lane];
        __syncthreads();
    }
    if (share > 0 || c >= width) return;
    s = part[0][lane];
    for (int o = 1; o < 64 / RS_COLUMNS; ++o) s += part[o][lane];
    if (which) {
        if (a.dpre_weight) store_one(a.dpre_weight, a.weight_dtype, c, s);
        return;
    }
    if (a.dpost_weight)
        store_one(a.dpost_weight, a.weight_dtype, c, a.scale ? s * load_one(a.scale, a.weight_dtype, a.scale_is_one ? 0 : c) : s);
    const float ds = s * load_one(a.post_weight, a.weight_dtype, c);
    if (one) one[c] = ds;
    else if (a.dscale) store_one(a.dscale, a.weight_dtype, c, ds);
}

// The gradient of a scale that all channels share.
__global__ __launch_bounds__(256) void residual_scale_kernel(const float* __restrict__ one, int width, void* dscale, int dtype) {
    __shared__ float part[4];
    float s = 0.f;
    for (int c = threadIdx.x; c < width; c += 256) s += one[c];
    s = lanes_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) store_one(dscale, dtype, 0, (part[0] + part[1]) + (part[2] + part[3]));
}

// How a width is shared among threads: threads per row and times eight elements per thread.
template <int T, int E>
struct Shape {
    static constexpr int TPR = T, EIGHTS = E;
};
// Backward, where the waves of a row take most of the registers, about as few whole waves as hold it: 5120 channels in the
// threads of 8192 took 158 us over 8192 rows, in their own 137.  Forward that gains nothing (87 and 90 us).
template <typename F>
static void with_forward_shape(int width, F&& f) {
    if (width <= 512) f(Shape<64, 1>{});
    else if (width <= 1024) f(Shape<64, 2>{});
    else if (width <= 2048) f(Shape<128, 2>{});
    else if (width <= 4096) f(Shape<256, 2>{});
    else if (width <= 8192) f(Shape<512, 2>{});
    else f(Shape<1024, 2>{});
}
template <typename F>
static void with_backward_shape(int width, F&& f) {
    if (width <= 512) f(Shape<64, 1>{});
    else if (width <= 1024) f(Shape<128, 1>{});
    else if (width <= 2048) f(Shape<256, 1>{});
    else if (width <= 3072) f(Shape<384, 1>{});
    else if (width <= 4096) f(Shape<512, 1>{});
    else if (width <= 5120) f(Shape<640, 1>{});
    else if (width <= 6144) f(Shape<768, 1>{});
    else if (width <= 7168) f(Shape<896, 1>{});
    else if (width <= 8192) f(Shape<1024, 1>{});
    else f(Shape<1024, 2>{});
}
template <typename F>
static void with_types(const MuonResidualNorm& a, F&& f) {
    const auto gates = [&](auto x, auto b) {
        if (!a.gate) f(x, b, std::integral_constant<int, GATE_NONE>{});
        else if (a.gate_is_token) f(x, b, std::integral_constant<int, GATE_TOKEN>{});
        else f(x, b, std::integral_constant<int, GATE_CHANNEL>{});
    };
    if (a.stream_dtype == MUON_AMD_SRC_BF16) gates(uint16_t{}, uint16_t{});
    else if (a.block_dtype == MUON_AMD_SRC_BF16) gates(float{}, uint16_t{});
    else gates(float{}, float{});
}

static int elem_size(int dtype) { return dtype == MUON_AMD_SRC_BF16 ? 2 : 4; }

// Workgroups of a launch over `rows` rows: all of them, up to `per_cu` for each of the 256 CUs.
static int workgroups(int64_t rows, int rows_each, int per_cu) {
    const int64_t n = (rows + rows_each - 1) / rows_each;
    return static_cast<int>(n < 256 * per_cu ? n : 256 * per_cu);
}
// Forward: 2048 threads a CU, and up to four times that where each still takes four rows for
// each row's threads, to be worth the weights that it loads: 32768 x 4096 bf16 243 -> 231 us, 32768 x 2048 126 -> 119, 16384 x 4096
// 122 -> 119.  (Up to 512 channels 1792 to 2048 threads fit a CU at once; the registers of wider rows leave 1024 to 1536 there, and
// the rest of the launch follows as workgroups end.)  Rows of more than 256 threads, whose weights are many: 16384 x 5120 166 -> 173, so not there.
static int forward_workgroups(int64_t rows, int threads, int tpr) {
    const int each = threads / tpr, per_cu = 2048 / threads;
    const int once = workgroups(rows, each, per_cu), most = tpr > RN_THREADS ? 0 : workgroups(rows, 4 * each, 4 * per_cu);
    return once > most ? once : most;
}
static int backward_workgroups(int64_t rows, int width) {
    int n = 0;
    with_backward_shape(width, [&](auto s) {
        constexpr int TPR = decltype(s)::TPR, THREADS = TPR > RN_THREADS ? TPR : RN_THREADS;
        n = workgroups(rows, THREADS / TPR, 1024 / THREADS);
    });
    return n;
}

static int check_residual(const MuonResidualNorm* a, const char* what) {
    MUON_REQUIRE(a, "%s: null arguments", what);
    MUON_REQUIRE(a->rows > 0 && a->width > 0 && a->width <= RN_MAX_WIDTH, "%s: rows=%lld width=%d (at most %d)", what,
                 static_cast<long long>(a->rows), a->width, RN_MAX_WIDTH);
    MUON_REQUIRE(a->x && a->b && a->post_weight && a->pre_weight, "%s: null input", what);
    for (const int32_t t : {a->stream_dtype, a->block_dtype, a->weight_dtype})
        MUON_REQUIRE(t == MUON_AMD_SRC_F32 || t == MUON_AMD_SRC_BF16, "%s: dtype=%d", what, t);
    MUON_REQUIRE(a->stream_dtype == MUON_AMD_SRC_F32 || a->block_dtype == MUON_AMD_SRC_BF16,
                 "%s: a bf16 residual stream takes a bf16 block", what);
    MUON_REQUIRE(a->eps >= 0.f, "%s: eps=%g", what, a->eps);
    return MUON_AMD_OK;
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_residual_norm(void) { return sizeof(MuonResidualNorm); }
int muon_amd_residual_norm_max_width(void) { return RN_MAX_WIDTH; }

int64_t muon_amd_residual_norm_partials(int64_t rows, int width) {
    if (rows <= 0 || width <= 0 || width > RN_MAX_WIDTH) return 0;
    return (static_cast<int64_t>(backward_workgroups(rows, width)) * 2 + 1) * width;
}

int muon_amd_residual_norm(const MuonResidualNorm* args, void* stream) {
    if (const int rc = check_residual(args, "residual_norm")) return rc;
    MUON_REQUIRE(args->h && args->y, "residual_norm: null output");
    const MuonResidualNorm a = *args;
    const bool nt = a.rows * a.width * (2 * elem_size(a.stream_dtype) + (a.gate && !a.gate_is_token ? 3 : 2) * elem_size(a.block_dtype)) > RN_CACHE;
    with_types(a, [&](auto x, auto b, auto gate) {
        with_forward_shape(a.width, [&](auto s) {
            constexpr int TPR = decltype(s)::TPR, G = pack_of<decltype(x)>, V = 8 / G * decltype(s)::EIGHTS, THREADS = TPR > RN_THREADS ? TPR : RN_THREADS;
            hipLaunchKernelGGL((residual_forward_kernel<decltype(x), decltype(b), decltype(gate)::value, TPR, V, G>),
                               dim3(forward_workgroups(a.rows, THREADS, TPR)), dim3(THREADS), 0, static_cast<hipStream_t>(stream), a, nt);
        });
    });
    return check_launch("residual_norm");
}

int muon_amd_residual_norm_backward(const MuonResidualNorm* args, void* stream) {
    if (const int rc = check_residual(args, "residual_norm_backward")) return rc;
    const MuonResidualNorm a = *args;
    MUON_REQUIRE(a.rstd && (a.dy || a.dh), "residual_norm_backward: null input");
    const bool columns = a.dpost_weight || a.dpre_weight || a.dscale;
    MUON_REQUIRE(!columns || a.partials, "residual_norm_backward: null workspace");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int n = backward_workgroups(a.rows, a.width);
    const bool nt = a.rows * a.width * (3 * elem_size(a.stream_dtype) + (a.gate && !a.gate_is_token ? 5 : 3) * elem_size(a.block_dtype)) > RN_CACHE;
    MuonResidualNorm b = a;
    if (!columns) b.partials = nullptr;
    with_types(a, [&](auto x, auto y, auto gate) {
        with_backward_shape(a.width, [&](auto s) {
            constexpr int TPR = decltype(s)::TPR, G = pack_of<decltype(x)>, V = 8 / G * decltype(s)::EIGHTS, THREADS = TPR > RN_THREADS ? TPR : RN_THREADS;
            hipLaunchKernelGGL((residual_backward_kernel<decltype(x), decltype(y), decltype(gate)::value, TPR, V, G>), dim3(n), dim3(THREADS),
                               0, st, b, nt);
        });
    });
    if (const int rc = check_launch("residual_norm_backward")) return rc;
    if (!columns) return MUON_AMD_OK;
    float* const one = a.dscale && a.scale_is_one ? a.partials + static_cast<int64_t>(n) * 2 * a.width : nullptr;
    hipLaunchKernelGGL(residual_columns_kernel, dim3((a.width + RS_COLUMNS - 1) / RS_COLUMNS, 2), dim3(RS_COLUMNS * RS_SHARES), 0, st, a, n, one);
    if (const int rc = check_launch("residual_norm_backward")) return rc;
    if (one) hipLaunchKernelGGL(residual_scale_kernel, dim3(1), dim3(256), 0, st, one, a.width, a.dscale, a.weight_dtype);
    return check_launch("residual_norm_backward");
}

}  // extern "C"
