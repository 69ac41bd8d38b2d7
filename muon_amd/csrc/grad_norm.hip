// The 2-norm of many gradients together, the coefficient that clips it, and the gradients scaled in place:
//   norm = sqrt(sum_i g_i^2),  coefficient = min(1, max_norm / (norm + 1e-6))
// Squares and sums are formed in 64 bits (the target adds and multiplies them as fast as 32), so no gradient that is
// finite in its own type overflows and none is lost below the sum.  The order of the sum is fixed: a workgroup strides
// over the blocks of the table, its threads' sums join in a tree, and the workgroups' sums are added by index.
// Memory bounds both passes: over 531 M bf16 gradients the squares take 157 us (6.8 TB/s) and the scaling 326 (6.5 TB/s).
#include "vector.h"

namespace muon_amd {

constexpr int GN_THREADS = 256;
constexpr int GN_EACH = 32;                                     // elements per thread and block
constexpr int GN_BLOCK_ELEMS = GN_THREADS * GN_EACH;            // as the blocks of the optimizer's launches
constexpr int GN_PARTIALS = 4096;                               // workgroups (2048: 164 instead of 156 us over 531 M bf16 gradients)

template <int THREADS>
__device__ __forceinline__ double block_sum(double v, double (&waves)[THREADS / 64]) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) s += waves[w];
    return s;
}

// Calls f(tensor, first element there) for a workgroup's share of the table's blocks, every gridDim.x-th: workgroups that
// run together then read next to each other (a contiguous share for each took 10 % longer over 531 M bf16 gradients).
// The tensor is looked up once and followed from there.
template <typename F>
__device__ __forceinline__ void for_blocks(const MuonGradDesc* __restrict__ descs, const int32_t* __restrict__ prefix, int ntensors,
                                           int nblocks, F&& f) {
    const int step = static_cast<int>(gridDim.x);
    int b = static_cast<int>(blockIdx.x);
    if (b >= nblocks) return;
    int ti = find_segment(prefix, ntensors, b);
    int begins = prefix[ti], ends = prefix[ti + 1];
    MuonGradDesc d = descs[ti];
    for (; b < nblocks; b += step) {
        if (b >= ends) {
            do {
                begins = ends;
                ends = prefix[++ti + 1];
            } while (b >= ends);
            d = descs[ti];
        }
        f(d, static_cast<int64_t>(b - begins) * GN_BLOCK_ELEMS);
    }
}

// Gradients that the memory-side cache holds are left in it for the pass that comes next (AdamW over 65 M bf16 gradients
// then takes 225 us instead of 242); more than that are read with the non-temporal hint (531 M: 177 -> 156 us).
constexpr int64_t GN_CACHED = 1ll << 27;

template <typename T, bool NT>
__device__ __forceinline__ double squares_of_block(const MuonGradDesc& d, int64_t base) {
    const T* __restrict__ const g = static_cast<const T*>(d.grad);
    constexpr int G = pack_of<T>, PACKS = GN_EACH / G;
    Pack<T, G> gv[PACKS];
#pragma unroll
    for (int i = 0; i < PACKS; ++i) gv[i] = load_pack<T, G, NT>(g, base + (i * GN_THREADS + threadIdx.x) * G, d.numel);
    double s[2] = {0., 0.};
#pragma unroll
    for (int i = 0; i < PACKS; ++i)
#pragma unroll
        for (int k = 0; k < G; ++k) {
            const double x = gv[i][k];
            s[k & 1] = fma(x, x, s[k & 1]);
        }
    return s[0] + s[1];
}

template <bool NT>
__global__ __launch_bounds__(GN_THREADS) void grad_squares_kernel(const MuonGradDesc* __restrict__ descs,
                                                                 const int32_t* __restrict__ prefix, int ntensors, int nblocks,
                                                                 double* __restrict__ partials) {
    __shared__ double red[4];
    double s = 0.;
    for_blocks(descs, prefix, ntensors, nblocks, [&](const MuonGradDesc& d, int64_t base) {
        s += d.dtype == MUON_AMD_SRC_BF16 ? squares_of_block<uint16_t, NT>(d, base) : squares_of_block<float, NT>(d, base);
    });
    const double total = block_sum<GN_THREADS>(s, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// The norm from the partial sums, in every thread.
template <int THREADS>
__device__ __forceinline__ float norm_of(const double* __restrict__ partials, int n) {
    __shared__ double red[THREADS / 64];
    double s = 0.;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += THREADS) s += partials[i];
    return static_cast<float>(sqrt(block_sum<THREADS>(s, red)));
}
// A norm that is not a number gives a coefficient that is not one either.
__device__ __forceinline__ float coefficient_of(float norm, float max_norm) {
    const float c = max_norm / (norm + 1e-6f);
    return c > 1.f ? 1.f : c;
}

constexpr int GN_JOIN = 1024;
__global__ __launch_bounds__(GN_JOIN) void grad_norm_kernel(const double* __restrict__ partials, int n, float max_norm,
                                                           float* __restrict__ out) {
    const float norm = norm_of<GN_JOIN>(partials, n);
    if (threadIdx.x == 0) {
        out[0] = norm;
        out[1] = coefficient_of(norm, max_norm);
    }
}

// A workgroup scales a part of a block, whose loads all go out first (531 M bf16 gradients: 326 us; whole blocks 336, quarters 391,
// and 4096 workgroups that stride over the blocks 358).
constexpr int GN_PARTS = 2, GN_PART_ELEMS = GN_BLOCK_ELEMS / GN_PARTS;
template <typename T>
__device__ __forceinline__ void scale_part(const MuonGradDesc& d, int64_t base, float c) {
    T* __restrict__ const g = static_cast<T*>(d.grad);
    constexpr int G = pack_of<T>, PACKS = GN_PART_ELEMS / GN_THREADS / G;
    const auto scaled = [&](const Pack<T, G>& v) {
        float x[G];
#pragma unroll
        for (int k = 0; k < G; ++k) x[k] = v[k] * c;
        return Pack<T, G>::of(x);
    };
    if (base + GN_PART_ELEMS <= d.numel) {
        Pack<T, G> v[PACKS];
#pragma unroll
        for (int i = 0; i < PACKS; ++i) v[i] = Pack<T, G>::template load<true>(g + base + (i * GN_THREADS + threadIdx.x) * G);
#pragma unroll
        for (int i = 0; i < PACKS; ++i) scaled(v[i]).template store<true>(g + base + (i * GN_THREADS + threadIdx.x) * G);
        return;
    }
#pragma unroll 1
    for (int64_t e = base + threadIdx.x * G; e < d.numel && e < base + GN_PART_ELEMS; e += GN_THREADS * G)
        store_pack<T, G, true>(g, e, d.numel, scaled(load_pack<T, G, true>(g, e, d.numel)));
}

// JOIN: every workgroup forms the coefficient from the partial sums (8 bytes for each block, from the L2) instead of
// a launch between the two passes.  Up to 8 M gradients that is faster whether they are then scaled or not (bf16, scaled: 1 M 8.2 ->
// 6.7 us, 8 M 16.7 -> 15.5, 64 M 65 -> 72; fp32, not scaled: 1 M 6.6 -> 5.3, 8 M 9.5 -> 8.6, 16 M 17.7 -> 18.9, 64 M 54 -> 76).
constexpr int GN_JOINED = 1024;            // blocks
template <bool JOIN>
__global__ __launch_bounds__(GN_THREADS) void grad_scale_kernel(const MuonGradDesc* __restrict__ descs,
                                                               const int32_t* __restrict__ prefix, int ntensors,
                                                               const double* __restrict__ partials, int n, float max_norm,
                                                               float* __restrict__ out) {
    float c;
    if constexpr (JOIN) {
        const float norm = norm_of<GN_THREADS>(partials, n);
        c = coefficient_of(norm, max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            out[0] = norm;
            out[1] = c;
        }
    } else {
        c = out[1];
    }
    if (c == 1.f) return;                 // (a coefficient that is not a number goes on)
    const int b = blockIdx.x / GN_PARTS, ti = find_segment_wave(prefix, ntensors, b);
    const MuonGradDesc d = descs[ti];
    const int64_t base = static_cast<int64_t>(b - prefix[ti]) * GN_BLOCK_ELEMS + blockIdx.x % GN_PARTS * GN_PART_ELEMS;
    if (d.dtype == MUON_AMD_SRC_BF16) scale_part<uint16_t>(d, base, c);
    else scale_part<float>(d, base, c);
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_grad_desc(void) { return sizeof(MuonGradDesc); }
int muon_amd_grad_norm_partials(void) { return GN_PARTIALS; }

int muon_amd_validate_grads(const MuonGradDesc* descs, int ntensors, const int32_t* prefix) {
    MUON_REQUIRE(descs && prefix, "validate_grads: null table");
    MUON_REQUIRE(ntensors > 0, "validate_grads: ntensors=%d", ntensors);
    MUON_REQUIRE(prefix[0] == 0, "validate_grads: prefix must start at 0");
    for (int i = 0; i < ntensors; ++i) {
        const MuonGradDesc& d = descs[i];
        MUON_REQUIRE(d.grad && d.numel > 0, "validate_grads: tensor %d: null pointer or numel=%lld", i, static_cast<long long>(d.numel));
        MUON_REQUIRE(d.dtype == MUON_AMD_SRC_F32 || d.dtype == MUON_AMD_SRC_BF16, "validate_grads: tensor %d: dtype=%d", i, d.dtype);
        MUON_REQUIRE(reinterpret_cast<uintptr_t>(d.grad) % (d.dtype == MUON_AMD_SRC_BF16 ? 2 : 4) == 0,
                     "validate_grads: tensor %d: address not a multiple of the element's size", i);
        const int64_t nblk = (d.numel + GN_BLOCK_ELEMS - 1) / GN_BLOCK_ELEMS;
        MUON_REQUIRE(static_cast<int64_t>(prefix[i + 1]) - prefix[i] == nblk, "validate_grads: tensor %d: prefix gives %d blocks, need %lld",
                     i, prefix[i + 1] - prefix[i], static_cast<long long>(nblk));
    }
    return MUON_AMD_OK;
}

static int grad_squares(const MuonGradDesc* descs_dev, const int32_t* prefix_dev, int ntensors, int nblocks, double* partials_dev,
                        float max_norm, const float* out_dev, hipStream_t stream) {
    MUON_REQUIRE(descs_dev && prefix_dev && partials_dev && out_dev, "grad_norm: null table, workspace or output");
    MUON_REQUIRE(ntensors > 0 && nblocks > 0, "grad_norm: ntensors=%d nblocks=%d", ntensors, nblocks);
    MUON_REQUIRE(nblocks <= INT32_MAX / GN_PARTS, "grad_norm: nblocks=%d", nblocks);
    MUON_REQUIRE(max_norm >= 0.f, "grad_norm: max_norm=%g", max_norm);
    const auto kernel = static_cast<int64_t>(nblocks) * GN_BLOCK_ELEMS > GN_CACHED ? grad_squares_kernel<true> : grad_squares_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(nblocks < GN_PARTIALS ? nblocks : GN_PARTIALS), dim3(GN_THREADS), 0, stream,
                       descs_dev, prefix_dev, ntensors, nblocks, partials_dev);
    return check_launch("grad_norm");
}

int muon_amd_grad_norm(const MuonGradDesc* descs_dev, const int32_t* block_prefix_dev, int ntensors, int nblocks, double* partials_dev,
                       float max_norm, float* out_dev, void* stream) {
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (const int rc = grad_squares(descs_dev, block_prefix_dev, ntensors, nblocks, partials_dev, max_norm, out_dev, s)) return rc;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(GN_JOIN), 0, s, partials_dev, nblocks < GN_PARTIALS ? nblocks : GN_PARTIALS,
                       max_norm, out_dev);
    return check_launch("grad_norm");
}

int muon_amd_grad_clip(const MuonGradDesc* descs_dev, const int32_t* block_prefix_dev, int ntensors, int nblocks, double* partials_dev,
                       float max_norm, float* out_dev, void* stream) {
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (const int rc = grad_squares(descs_dev, block_prefix_dev, ntensors, nblocks, partials_dev, max_norm, out_dev, s)) return rc;
    const int n = nblocks < GN_PARTIALS ? nblocks : GN_PARTIALS;
    const bool join = nblocks <= GN_JOINED;
    if (!join) {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(GN_JOIN), 0, s, partials_dev, n, max_norm, out_dev);
        if (const int rc = check_launch("grad_norm")) return rc;
    }
    hipLaunchKernelGGL(join ? grad_scale_kernel<true> : grad_scale_kernel<false>, dim3(nblocks * GN_PARTS), dim3(GN_THREADS), 0, s, descs_dev,
                       block_prefix_dev, ntensors, partials_dev, n, max_norm, out_dev);
    return check_launch("grad_clip");
}

}  // extern "C"
