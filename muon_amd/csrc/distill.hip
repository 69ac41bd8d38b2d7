// Distillation from a teacher's top logits.  Per token over V logits x of the student, and a list of the teacher's logits t
// at indices i, at a temperature T:
//   p = softmax(x / T) over the vocabulary,  q = softmax(t / T) over the list
//   loss = T^2 sum_k q_k (log q_k - log p_{i_k})
// Backward, from the gradient g of the token's loss:  dx = g T (p - sum_k q_k [i_k = v])
// (mean: g is the scalar's divided by the N tokens that take part).  An entry whose index is outside of the vocabulary is not
// there; neither is one whose logit is -infinity.  A token whose list has no entry, or that is masked out, takes no part: loss and gradient are zero,
// whatever its logits hold.
//
// Memory bounds both passes: forward reads the logits once (a running maximum and sum in every thread), backward reads
// them and writes the gradient.  Arithmetic is in base 2: with c = log2(e) / T a thread keeps m, its largest logit, and
// s = sum 2^((x - m) c); m and log2(s) are kept apart for backward, so that probabilities go by differences of logits
// however far from zero these are (with x c - m c in one instruction, a row at 1e30 is lost in the rounding of m c).  Rows are shared by several workgroups where
// there are few of them, and joined in the order of their parts.  Loads and stores of the rows carry the non-temporal hint: nothing is read again
// while it is in a cache, but for what fits the last one (8192 x 128256 bf16, both passes: 1140 -> 1021 us, 6.2 TB/s of the
// 6.3 GB).  Backward has them for every size, though logits about as large as the last cache come faster by plain loads where nothing has pushed them out
// since forward read them (4096 x 32000, 262 MB, repeated: 147 us and 140; 8192 x 128256: 1007 and 1067): what runs between the two passes of a training
// step decides that, and is not known here.  Of 8192 x 128256 forward takes 317 us (6.6 TB/s), the losses' sum 5, backward 689 (6.1 TB/s).
#include "lanes.h"

namespace muon_amd {

constexpr int DT_MAX_TOP = 1024;
constexpr int DT_THREADS = 256, DT_WAVES = DT_THREADS / 64;
constexpr int DT_UNROLL = 4;                               // packs that a thread has in flight
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

// A running maximum and the sum of 2^((x - m) c) below it.
struct RunningSum {
    float m = -__builtin_inff(), s = 0.f;
    // (a reference of -infinity, where nothing but that has been seen, would leave no number)
    static __device__ __forceinline__ float reference(float m) { return m == -__builtin_inff() ? 0.f : m; }
    static __device__ __forceinline__ float power(float x, float ref, float c) { return __builtin_amdgcn_exp2f((x - ref) * c); }
    __device__ __forceinline__ void join(float m2, float s2, float c) {
        const float top = fmaxf(m, m2), ref = reference(top);
        s = s * power(m, ref, c) + s2 * power(m2, ref, c);
        m = top;
    }
};

template <typename T>
__device__ __forceinline__ float element(const void* p, int64_t i) {
    if constexpr (sizeof(T) == 2) return bf2f(static_cast<const T*>(p)[i]);
    else return static_cast<const T*>(p)[i];
}
__device__ __forceinline__ float teacher_of(const MuonDistill& a, int64_t i) {
    return a.teacher_dtype == MUON_AMD_SRC_BF16 ? element<uint16_t>(a.teacher, i) : element<float>(a.teacher, i);
}
// The index of entry k of token t, or -1 where it is not there.
__device__ __forceinline__ int index_of(const MuonDistill& a, int64_t t, int k) {
    const int64_t i = a.index_bits == 64 ? static_cast<const int64_t*>(a.indices)[t * a.ld_indices + k]
                                         : static_cast<const int32_t*>(a.indices)[t * a.ld_indices + k];
    return i >= 0 && i < a.vocab ? static_cast<int>(i) : -1;
}

// A token's list, by a wave.  What a lane has of it in the first place (an entry and the student's logit there; more than 64 are read again
// below) is requested when it is made, and used in finish().
struct TokenList {
    float v0 = 0.f, x0 = 0.f;
    bool open = false;
    __device__ __forceinline__ TokenList() {}
    __device__ __forceinline__ void entry(const MuonDistill& a, int64_t t, int k, float& v, float& x) const {
        const int i = open && k < a.top ? index_of(a, t, k) : -1;
        v = k < a.top ? teacher_of(a, t * a.ld_teacher + k) : -__builtin_inff();
        const int64_t at = t * a.ld_logits + (i >= 0 ? i : 0);
        x = i < 0 ? 0.f : a.dtype == MUON_AMD_SRC_BF16 ? element<uint16_t>(a.logits, at) : element<float>(a.logits, at);
        if (i < 0) v = -__builtin_inff();
    }
    __device__ __forceinline__ TokenList(const MuonDistill& a, int64_t t) : open(!a.mask || a.mask[t]) { entry(a, t, threadIdx.x & 63, v0, x0); }
    // The token's loss and statistics, with the maximum and sum of its logits in `r` (of each lane: joined here).  Whether it takes part.
    __device__ __forceinline__ bool finish(const MuonDistill& a, int64_t t, float c, const RunningSum& r, float& loss) const {
        const auto larger = [](float x, float y) { return fmaxf(x, y); };
        const int lane = threadIdx.x & 63;
        // the list: whether anything is there, its maximum and sum
        bool some = v0 != -__builtin_inff();
        float most = fmaxf(v0, -__builtin_inff());
        for (int k = lane + 64; k < a.top; k += 64) {
            float v, x;
            entry(a, t, k, v, x);
            some |= v != -__builtin_inff();
            most = fmaxf(most, v);
        }
        const bool on = __ballot(some) != 0;
        float tm = -__builtin_inff(), tl = 0.f, m = 0.f, l = 0.f;
        loss = 0.f;
        if (on) {
            tm = RunningSum::reference(group_reduce<64>(most, larger));     // (a list of nothing but NaN has a number here all the same)
            float s = RunningSum::power(v0, tm, c);
            for (int k = lane + 64; k < a.top; k += 64) {
                float v, x;
                entry(a, t, k, v, x);
                s += RunningSum::power(v, tm, c);
            }
            tl = __log2f(group_sum<64>(s));
            m = group_reduce<64>(r.m, larger);
            l = __log2f(group_sum<64>(r.s * RunningSum::power(r.m, RunningSum::reference(m), c)));
            m = RunningSum::reference(m);
            const auto term = [&](float v, float x) {
                const float y = (v - tm) * c - tl, q = __builtin_amdgcn_exp2f(y);             // log2 q, q
                if (v != -__builtin_inff() && q != 0.f) loss = fmaf(q, y - ((x - m) * c - l), loss);
            };
            term(v0, x0);
            for (int k = lane + 64; k < a.top; k += 64) {
                float v, x;
                entry(a, t, k, v, x);
                term(v, x);
            }
            loss = group_sum<64>(loss) * (LN2 * a.temperature * a.temperature);
        }
        if (lane == 0) {
            a.losses[t] = loss;
            reinterpret_cast<f32x4v*>(a.stats)[t] = f32x4v{m, l, tm, tl};
        }
        return on;
    }
};

// Part `blockIdx.x % parts` of a token's logits: its maximum and sum.  The only part of a token has its list too (a launch for the lists
// took 13 us for 4096 x 64; the whole call 154.5 -> 148.4 us, requested ahead of the row 146.9).
template <typename T>
__global__ __launch_bounds__(DT_THREADS) void distill_stats_kernel(const MuonDistill a, int parts, int length) {
    constexpr int G = pack_of<T>;
    __shared__ float top[DT_WAVES], sum[DT_WAVES];
    const float c = LOG2E / a.temperature;
    const int64_t t = blockIdx.x / parts;
    const int part = blockIdx.x % parts, begin = part * length, end = min(begin + length, a.vocab);
    const T* const row = static_cast<const T*>(a.logits) + t * a.ld_logits;
    RunningSum r;
    TokenList list;
    if (parts == 1 && threadIdx.x < 64) list = TokenList(a, t);
    const auto add = [&](const Pack<T, G>(&v)[DT_UNROLL]) {
        float most = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < G; ++i) most = fmaxf(most, v[u][i]);
        const float m = fmaxf(r.m, most), ref = RunningSum::reference(m);
        float s = r.s * RunningSum::power(r.m, ref, c);
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < G; ++i) s += RunningSum::power(v[u][i], ref, c);
        r.m = m;
        r.s = s;
    };
    constexpr int STEP = DT_THREADS * G;
    int e = begin + static_cast<int>(threadIdx.x) * G;
    for (; e - static_cast<int>(threadIdx.x) * G + DT_UNROLL * STEP <= end; e += DT_UNROLL * STEP) {
        Pack<T, G> v[DT_UNROLL];
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u) v[u] = Pack<T, G>::template load<true>(row + e + u * STEP);
        add(v);
    }
    if (e - static_cast<int>(threadIdx.x) * G < end) {      // what is left of the part: -infinity beyond it
        Pack<T, G> v[DT_UNROLL];
        Pack<T, G> none = Pack<T, G>::zero();
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if constexpr (sizeof(T) == 2) none.put(i, 0xff80);
            else none.put(i, -__builtin_inff());
        }
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u) {
            const int at = e + u * STEP;
            v[u] = none;
            if (at + G <= end) v[u] = Pack<T, G>::template load<false>(row + at);
            else if (at < end) {
                Pack<T, G> some = Pack<T, G>::zero();
#pragma unroll
                for (int i = 0; i < G; ++i) some.put(i, at + i < end ? row[at + i] : none.get(i));
                v[u] = some;
            }
        }
        add(v);
    }
    const float m = group_reduce<64>(r.m, [](float x, float y) { return fmaxf(x, y); });
    const float s = group_sum<64>(r.s * RunningSum::power(r.m, RunningSum::reference(m), c));
    if ((threadIdx.x & 63) == 0) {
        top[threadIdx.x >> 6] = m;
        sum[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0;
    if (threadIdx.x >= 64) return;
    if (parts == 1) {
        const int lane = threadIdx.x;
        RunningSum mine;
        if (lane < DT_WAVES) mine.m = top[lane], mine.s = sum[lane];
        float loss;
        list.finish(a, t, c, mine, loss);
    } else if (threadIdx.x == 0) {
        RunningSum all;
        for (int w = 0; w < DT_WAVES; ++w) all.join(top[w], sum[w], c);
        reinterpret_cast<f32x2_t*>(a.partials)[blockIdx.x] = f32x2_t{all.m, all.s};
    }
}

// The workgroup that is done last adds up the losses.  LISTS: a wave for each token, its parts joined, its list, its loss; else these are there, and
// a thread for each token only adds.  (At most 256 workgroups: with one for every four tokens, 2048 of them at one counter took 96 us.)
constexpr int DF_THREADS = 1024, DF_WAVES = DF_THREADS / 64, DF_GROUPS = 256;
static int finish_groups(int64_t tokens, int each) { return static_cast<int>(tokens < each * DF_GROUPS ? (tokens + each - 1) / each : DF_GROUPS); }
template <bool LISTS>
__global__ __launch_bounds__(DF_THREADS) void distill_finish_kernel(const MuonDistill a, int parts) {
    __shared__ float sums[DF_WAVES];
    __shared__ int counts[DF_WAVES];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float total = 0.f;
    int taking = 0;
    if constexpr (LISTS) {
        const float c = LOG2E / a.temperature;
        for (int64_t t = static_cast<int64_t>(blockIdx.x) * DF_WAVES + wave; t < a.tokens; t += static_cast<int64_t>(gridDim.x) * DF_WAVES) {
            // All that the token has to be read for is requested together: each lane's entry of the list, the student's logit there, a part's sums.
            const f32x2_t* const p = reinterpret_cast<const f32x2_t*>(a.partials) + t * parts;
            const f32x2_t first = lane < parts ? p[lane] : f32x2_t{-__builtin_inff(), 0.f};
            const TokenList list(a, t);
            RunningSum r;
            r.join(first[0], first[1], c);
            for (int i = lane + 64; i < parts; i += 64) r.join(p[i][0], p[i][1], c);
            float loss;
            taking += list.finish(a, t, c, r, loss);
            total += loss;
        }
    } else {
        for (int64_t t = static_cast<int64_t>(blockIdx.x) * DF_THREADS + threadIdx.x; t < a.tokens; t += static_cast<int64_t>(gridDim.x) * DF_THREADS) {
            total += a.losses[t];
            taking += reinterpret_cast<const f32x4v*>(a.stats)[t][2] != -__builtin_inff();
        }
        total = group_sum<64>(total);
        taking = group_reduce<64>(taking, [](int u, int v) { return u + v; });
    }
    if (lane == 0) {
        sums[wave] = total;
        counts[wave] = taking;
    }
    __syncthreads();
    float* const left = a.partials + 2 * a.tokens * parts;           // {sum, tokens} of each workgroup
    if (threadIdx.x == 0) {
        float s = 0.f;
        int n = 0;
        for (int w = 0; w < DF_WAVES; ++w) {
            s += sums[w];
            n += counts[w];
        }
        __hip_atomic_store(&left[2 * blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&left[2 * blockIdx.x + 1], __int_as_float(n), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(a.counter, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.x) - 1;
    }
    __syncthreads();
    if (!last) return;
    float s = 0.f;
    int n = 0;
    for (unsigned g = threadIdx.x; g < gridDim.x; g += DF_THREADS) {
        s += __hip_atomic_load(&left[2 * g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        n += __float_as_int(__hip_atomic_load(&left[2 * g + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
    s = group_sum<64>(s);
    n = group_reduce<64>(n, [](int u, int v) { return u + v; });
    if (lane == 0) {
        sums[wave] = s;
        counts[wave] = n;
    }
    __syncthreads();
    if (threadIdx.x > 0) return;
    for (int w = 1; w < DF_WAVES; ++w) {
        s += sums[w];
        n += counts[w];
    }
    const float part = static_cast<float>(n > 0 ? n : 1);
    *a.part = part;
    if (a.loss) *a.loss = a.reduction == MUON_AMD_REDUCE_MEAN ? s / part : s;
}

// Packs of a thread in a workgroup's share of a row: one round of loads (8192 x 128256 bf16, both passes: 1140 us; 8 packs 1158, 16 packs 1176).
constexpr int DB_CHUNK_PACKS = DT_UNROLL;
template <typename T>
__global__ __launch_bounds__(DT_THREADS) void distill_backward_kernel(const MuonDistill a, int parts) {
    constexpr int G = pack_of<T>, STEP = DT_THREADS * G, LENGTH = STEP * DB_CHUNK_PACKS;
    __shared__ int at[DT_MAX_TOP];
    __shared__ float q[DT_MAX_TOP];
    const float c = LOG2E / a.temperature;
    const int64_t t = blockIdx.x / parts;
    const int begin = static_cast<int>(blockIdx.x % parts) * LENGTH, end = min(begin + LENGTH, a.vocab);
    const T* const row = static_cast<const T*>(a.logits) + t * a.ld_logits;
    T* const out = static_cast<T*>(a.dlogits) + t * a.vocab;
    const f32x4v st = reinterpret_cast<const f32x4v*>(a.stats)[t];
    const float m = st[0], l = st[1], tm = st[2], tl = st[3];
    if (tm == -__builtin_inff()) {                           // takes no part
        for (int e = begin + static_cast<int>(threadIdx.x) * G; e < end; e += STEP) store_pack<T, G, true>(out, e, end, Pack<T, G>::zero());
        return;
    }
    float g = *(a.dloss + (a.reduction == MUON_AMD_REDUCE_NONE ? t * a.ld_dloss : 0)) * a.temperature;
    if (a.reduction == MUON_AMD_REDUCE_MEAN) g /= *a.part;
    for (int k = threadIdx.x; k < a.top; k += DT_THREADS) {
        const int i = index_of(a, t, k);
        at[k] = i >= begin && i < end ? i : -1;
        q[k] = __builtin_amdgcn_exp2f((teacher_of(a, t * a.ld_teacher + k) - tm) * c - tl);
    }
    const auto gradient = [&](float x) { return g * __builtin_amdgcn_exp2f((x - m) * c - l); };
    const auto put = [&](const Pack<T, G>& v, int e) {
        float d[G];
#pragma unroll
        for (int i = 0; i < G; ++i) d[i] = gradient(v[i]);
        store_pack<T, G, true>(out, e, end, Pack<T, G>::of(d));
    };
    int e = begin + static_cast<int>(threadIdx.x) * G;
    if (begin + LENGTH <= end) {
        Pack<T, G> v[DT_UNROLL];
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u) v[u] = Pack<T, G>::template load<true>(row + e + u * STEP);
#pragma unroll
        for (int u = 0; u < DT_UNROLL; ++u) put(v[u], e + u * STEP);
    } else {
        for (; e < end; e += STEP) put(load_pack<T, G, true>(row, e, end), e);
    }
    // The teacher's entries go over what was written there: the barrier orders the two.  The first entry of an index
    // writes for all that have it.
    __syncthreads();
    for (int k = threadIdx.x; k < a.top; k += DT_THREADS) {
        const int i = at[k];
        if (i < 0) continue;
        float all = 0.f;
        bool first = true;
        for (int j = 0; j < a.top; ++j)
            if (at[j] == i) {
                first = first && j >= k;
                all += q[j];
            }
        if (!first) continue;
        const float d = g * (__builtin_amdgcn_exp2f((element<T>(row, i) - m) * c - l) - all);
        if constexpr (sizeof(T) == 2) out[i] = f2bf(d);
        else out[i] = d;
    }
}

// Parts that a token's logits are read in: one where there are tokens enough for every CU to have several workgroups, else up
// to as many as leave a workgroup two rounds of its loads.
static int distill_parts(int64_t tokens, int vocab, int dtype) {
    const int round = DT_THREADS * DT_UNROLL * (dtype == MUON_AMD_SRC_BF16 ? 8 : 4);
    const int64_t wanted = (1024 + tokens - 1) / tokens, most = (vocab + 2 * round - 1) / (2 * round);
    return static_cast<int>(wanted < most ? wanted : most);
}
// (a launch counts its threads in 32 bits)
static int check_distill_grid(int64_t groups, const MuonDistill& a, const char* what) {
    MUON_REQUIRE(groups <= 0xffffffffll / DT_THREADS, "%s: %lld tokens of %d logits are more than a launch holds", what, static_cast<long long>(a.tokens), a.vocab);
    return MUON_AMD_OK;
}
// Workgroups to a token's gradient.
static int64_t backward_parts(const MuonDistill& a) {
    const int64_t length = DT_THREADS * DB_CHUNK_PACKS * (a.dtype == MUON_AMD_SRC_BF16 ? 8 : 4);
    return (a.vocab + length - 1) / length;
}
static int part_length(int vocab, int parts) { return ((vocab + parts - 1) / parts + 7) / 8 * 8; }

static int check_distill(const MuonDistill* a, const char* what) {
    MUON_REQUIRE(a, "%s: null arguments", what);
    MUON_REQUIRE(a->tokens > 0 && a->tokens < (int64_t(1) << 24) && a->vocab > 0 && a->vocab <= (1 << 30), "%s: tokens=%lld vocab=%d", what,
                 static_cast<long long>(a->tokens), a->vocab);
    MUON_REQUIRE(a->top > 0 && a->top <= DT_MAX_TOP, "%s: top=%d (at most %d)", what, a->top, DT_MAX_TOP);
    MUON_REQUIRE(a->logits && a->teacher && a->indices && a->stats && a->part, "%s: null pointer", what);
    MUON_REQUIRE((a->dtype == MUON_AMD_SRC_F32 || a->dtype == MUON_AMD_SRC_BF16) && (a->teacher_dtype == MUON_AMD_SRC_F32 || a->teacher_dtype == MUON_AMD_SRC_BF16),
                 "%s: dtype=%d teacher_dtype=%d", what, a->dtype, a->teacher_dtype);
    MUON_REQUIRE(a->index_bits == 32 || a->index_bits == 64, "%s: index_bits=%d", what, a->index_bits);
    MUON_REQUIRE(a->reduction >= MUON_AMD_REDUCE_NONE && a->reduction <= MUON_AMD_REDUCE_MEAN, "%s: reduction=%d", what, a->reduction);
    // (its square and reciprocal are to be normal numbers)
    MUON_REQUIRE(a->temperature >= 1e-15f && a->temperature <= 1e15f, "%s: temperature=%g", what, static_cast<double>(a->temperature));
    return MUON_AMD_OK;
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_distill(void) { return sizeof(MuonDistill); }
int muon_amd_distill_max_top(void) { return DT_MAX_TOP; }

int64_t muon_amd_distill_partials(int64_t tokens, int vocab, int dtype) {
    if (tokens <= 0 || vocab <= 0) return 0;
    return 2 * tokens * distill_parts(tokens, vocab, dtype) + 2 * DF_GROUPS;
}

int muon_amd_distill(const MuonDistill* args, void* stream) {
    if (const int rc = check_distill(args, "distill")) return rc;
    const MuonDistill a = *args;
    MUON_REQUIRE(a.losses && a.partials && a.counter, "distill: null workspace or output");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int parts = distill_parts(a.tokens, a.vocab, a.dtype), length = part_length(a.vocab, parts);
    if (const int rc = check_distill_grid(a.tokens * parts, a, "distill")) return rc;
    if (a.differentiable)
        if (const int rc = check_distill_grid(a.tokens * backward_parts(a), a, "distill, whose gradient is wanted")) return rc;
    const dim3 grid(static_cast<unsigned>(a.tokens * parts));
    if (a.dtype == MUON_AMD_SRC_BF16) hipLaunchKernelGGL(distill_stats_kernel<uint16_t>, grid, dim3(DT_THREADS), 0, st, a, parts, length);
    else hipLaunchKernelGGL(distill_stats_kernel<float>, grid, dim3(DT_THREADS), 0, st, a, parts, length);
    if (const int rc = check_launch("distill")) return rc;
    if (parts > 1) hipLaunchKernelGGL(distill_finish_kernel<true>, dim3(finish_groups(a.tokens, DF_WAVES)), dim3(DF_THREADS), 0, st, a, parts);
    else hipLaunchKernelGGL(distill_finish_kernel<false>, dim3(finish_groups(a.tokens, DF_THREADS)), dim3(DF_THREADS), 0, st, a, parts);
    return check_launch("distill");
}

int muon_amd_distill_backward(const MuonDistill* args, void* stream) {
    if (const int rc = check_distill(args, "distill_backward")) return rc;
    const MuonDistill a = *args;
    MUON_REQUIRE(a.dloss && a.dlogits, "distill_backward: null gradient");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t parts = backward_parts(a);
    if (const int rc = check_distill_grid(a.tokens * parts, a, "distill_backward")) return rc;
    const dim3 grid(static_cast<unsigned>(a.tokens * parts));
    if (a.dtype == MUON_AMD_SRC_BF16) hipLaunchKernelGGL(distill_backward_kernel<uint16_t>, grid, dim3(DT_THREADS), 0, st, a, static_cast<int>(parts));
    else hipLaunchKernelGGL(distill_backward_kernel<float>, grid, dim3(DT_THREADS), 0, st, a, static_cast<int>(parts));
    return check_launch("distill_backward");
}

}  // extern "C"
