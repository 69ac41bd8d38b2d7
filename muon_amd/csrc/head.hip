// Cross entropy of a linear head over a large vocabulary, without its logits.  Over N tokens of D channels h, a matrix W of
// V rows, targets t:
//   x_nv = h_n . W_v,  lse_n = log sum_v exp(x_nv),  loss_n = lse_n - x_{n, t_n}
// Backward, from the gradients g_n of loss_n and z_n of lse_n:
//   e_nv = (g_n + z_n) exp(x_nv - lse_n) - g_n [v = t_n],   dh_n = sum_v e_nv W_v,   dW_v = sum_n e_nv h_n
//
// Forward is one matrix product whose epilogue leaves the maximum and the sum of exponentials of each row of its tile, 8 bytes for
// 256 logits, joined by a second launch.  Backward goes through the vocabulary in pieces: the logits of a piece are formed again
// (the same product; the same bits too, but where few tokens were streamed forward), e is written once in bf16 (rounding each term of sums over the
// vocabulary or the tokens by at most 2^-8 of itself, as the sums are rounded when they are written), and two products follow, whose second operand (and for
// dW the first one too) lies k-major and is read through transposing LDS reads, so nothing is written twice.  8 N V D operations
// instead of the 6 N V D of a backward pass that keeps N V logits.  8192 x 128256 x 4096: 6.4 ms forward, 6.6 + 6.4 + 6.9 ms backward (1254 to 1354
// TFLOP/s; a library's product of that size 1377).
//
// Tokens that are ignored leave the products: a first launch numbers those that take part, and their hidden states are copied
// to consecutive rows (zeros up to whole tiles).  The products take the tokens' number from the device; workgroups beyond it end
// at once.  Few tokens forward (evaluation, single tokens): the matrix is streamed once through registers instead.
//
// The products bound everything: matrix instructions at 256 x 256 tiles of 8 waves, k-blocks of 64 in an LDS ring filled by
// buffer_load ... lds a block and a half ahead, as in ns_gemm.hip.
#include "lanes.h"
#include "tile.h"

namespace muon_amd {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr int HD_TILE = 256;                        // rows of the copy of the hidden states are padded to this
constexpr int HD_CUS = 256;                         // compute units
constexpr int HD_FEW = 64;                          // tokens that the streaming kernel takes

// ---------------------------------------------------------------------------------------------
// The products
// ---------------------------------------------------------------------------------------------
enum HeadProduct {
    HEAD_STATS,      // x = h W^T: row statistics
    HEAD_GRAD,       // x = h W^T again: e
    HEAD_DHIDDEN,    // e W, a share of the vocabulary
    HEAD_DWEIGHT,    // e^T h
};

// acc[i][j] = sum_k P(i, k) Q(j, k).  An operand is row-major (k along the row) or k-major; `end_*` is the byte offset of the last
// 16 bytes that may be read from the base: what lies beyond (rows and columns of a tile that are in no output, rows that
// meet zeros of the other operand) is read from there instead.
struct HeadGemm {
    const uint16_t* P;
    const uint16_t* Q;
    int64_t ldp, ldq;
    int64_t end_p, end_q;
    const int32_t* count;          // tokens that take part
    const int32_t* splits;         // HEAD_DHIDDEN: shares of the k-blocks
    int row_tiles, col_tiles, most_splits;   // (row_tiles of a product over tokens: at most; the count decides)
    int rows, cols, kblocks;       // rows / cols of the output (rows of a product over tokens: from the count), k-blocks (HEAD_DWEIGHT: from the count)
    int col_limit;                 // columns of a k-major Q row that may be read
    int row_limit;                 // likewise of a k-major P row
    // HEAD_STATS, HEAD_GRAD
    int vocab_begin, vocab;        // first column in the vocabulary, size of the vocabulary
    const int32_t* target;         // of each row
    f32x2_t* stats;                // [column tile][row]: maximum, sum of 2^((x - maximum) log2 e)
    float* target_logit;
    int64_t ld_stats;
    const f32x4v* coef;            // of each row: (g + z) / scale, g / scale, the row's maximum, log2 of its sum
    const float* scale;            // HEAD_DWEIGHT: what the gradient is multiplied by
    // outputs
    uint16_t* out;                 // HEAD_GRAD, HEAD_DWEIGHT
    float* part;                   // HEAD_DHIDDEN: [split][row][column]
    int64_t ld_out, part_stride;
    int add;                       // HEAD_DHIDDEN: to what a piece before left there
};

template <int BT_, int WGM_, int WGN_, int MINB_, int NHALF_>
struct HeadCfg {
    static constexpr int BT = BT_, WGM = WGM_, WGN = WGN_, MINB = MINB_, NHALF = NHALF_;
    static constexpr int NW = WGM * WGN, NT = NW * 64, WM = BT / WGM, WN = BT / WGN, TM = WM / 32, TN = WN / 32;
    static constexpr int HALF_BYTES = BT * ROW_BYTES, DPH = BT / 8 / NW, RING = (NHALF - 1) / 2;
    static constexpr size_t LDS_BYTES = static_cast<size_t>(NHALF) * HALF_BYTES;
    static_assert(WN == 64, "an epilogue's strip is 64 columns");
    static_assert(2 * HALF_BYTES >= WGN * BT * 8 && 2 * HALF_BYTES >= NW * 4096, "what the epilogues leave in LDS");
    static_assert(RING == 2 && NHALF % 2 == 1, "one copy of the k-block for each of the last two");
    static_assert(LDS_BYTES * MINB <= 163840, "LDS of a CU");
};
typedef HeadCfg<256, 2, 4, 1, 5> HeadLarge;
typedef HeadCfg<128, 2, 2, 2, 5> HeadSmall;

// Tile `t` of row_tiles x col_tiles: strips of 8 column tiles, row by row, so that 32 neighbours are 4 x 8 tiles.
struct TileAt {
    int row, col;
};
__device__ __forceinline__ TileAt tile_at(int t, int row_tiles, int col_tiles) {
    const int strip = t / (8 * row_tiles), first = strip * 8, width = min(8, col_tiles - first), in = t - first * row_tiles;
    return {in / width, first + in % width};
}
// Workgroup b of `total` to its place in that order: workgroups are dealt to the eight XCDs in turn, and each XCD gets runs of 32
// neighbours, which share operand panels in its L2 (what is left over after whole sets of eight runs: one run for each XCD).
__device__ __forceinline__ int place_of(int b, int total) {
    const int full = total / 256 * 256;
    const int x = b % 8, s = b / 8;
    if (b < full) return ((s / 32) * 8 + x) * 32 + s % 32;
    const int rem = total - full;
    return full + x * (rem / 8) + min(x, rem % 8) + (b - full) / 8;
}

// Fragments of one k-step for a side of the product: N fragments, row-major or k-major.
template <int N, bool K>
struct Frags {
    u32x4 row[K ? 1 : N];
    u32x2 tr[K ? 2 * N : 1];
    __device__ __forceinline__ u32x4 get(int i) const {
        if constexpr (K) return u32x4{tr[2 * i].x, tr[2 * i].y, tr[2 * i + 1].x, tr[2 * i + 1].y};
        else return row[i];
    }
};
// The wait for the older fragments while CNT younger reads are in flight, tied to their registers.
template <int CNT, typename A, typename B>
__device__ __forceinline__ void wait_both(A& a, B& b) {
    constexpr bool ka = sizeof(a.tr) > sizeof(u32x2), kb = sizeof(b.tr) > sizeof(u32x2);
    if constexpr (!ka && !kb) {
        wait_frags<CNT>(a.row, b.row);
    } else if constexpr (!ka) {
        wait_frags_tr<CNT>(a.row, b.tr);
    } else if constexpr (sizeof(a.tr) / sizeof(u32x2) == 8) {
        static_assert(sizeof(b.tr) / sizeof(u32x2) == 4, "operand lists below");
        asm volatile("s_waitcnt lgkmcnt(%12)"
                     : "+v"(a.tr[0]), "+v"(a.tr[1]), "+v"(a.tr[2]), "+v"(a.tr[3]), "+v"(a.tr[4]), "+v"(a.tr[5]), "+v"(a.tr[6]), "+v"(a.tr[7]),
                       "+v"(b.tr[0]), "+v"(b.tr[1]), "+v"(b.tr[2]), "+v"(b.tr[3])
                     : "n"(CNT));
    } else {
        static_assert(sizeof(a.tr) / sizeof(u32x2) == 4 && sizeof(b.tr) / sizeof(u32x2) == 4, "operand lists below");
        asm volatile("s_waitcnt lgkmcnt(%8)"
                     : "+v"(a.tr[0]), "+v"(a.tr[1]), "+v"(a.tr[2]), "+v"(a.tr[3]), "+v"(b.tr[0]), "+v"(b.tr[1]), "+v"(b.tr[2]), "+v"(b.tr[3])
                     : "n"(CNT));
    }
}

// An operand's half-stages: where a lane's pieces lie from the tile's base, and how the base moves from k-block to k-block.
// TURN: the k-blocks are taken from number `turn` on, and from the first one after the last of `blocks`.
template <typename Cfg, bool K, bool TURN>
struct Source {
    uint32_t off[Cfg::DPH];
    uint64_t base;                 // (wave-uniform)
    int64_t step, end;
    int turn, blocks;
    // first: the tile's first row (k-major: column); limit: columns of a k-major row that may be read
    __device__ __forceinline__ void set(const uint16_t* p, int64_t ld, int64_t end_bytes, int first, int limit, int k0, int lane, int wave) {
        constexpr int ROWK = Cfg::BT * 2;
        const int gchunk = (lane & 7) ^ (((wave & 1) << 2) | (lane >> 4));
        const int64_t corner = K ? (static_cast<int64_t>(k0) * ld + first) * 2 : (static_cast<int64_t>(first) * ld + k0) * 2;
#pragma unroll
        for (int j = 0; j < Cfg::DPH; ++j) {
            if constexpr (K) {
                const int o = (j * Cfg::NW + wave) * 1024 + lane * 16, k = o / ROWK, w = o % ROWK;
                const int col = ((w / 64) ^ (k & 3)) * 32 + ((w % 64) >> 1);
                off[j] = static_cast<uint32_t>((k * ld + min(col, limit - first - 8)) * 2);
            } else {
                const int r = (j * Cfg::NW + wave) * 8 + (lane >> 3);
                off[j] = static_cast<uint32_t>((r * ld + gchunk * 8) * 2);
            }
        }
        base = reinterpret_cast<uint64_t>(p) + corner;
        end = end_bytes - corner;
        step = K ? BK * ld * 2 : BK * 2;
    }
    // Piece j of k-block kb.
    __device__ __forceinline__ void issue(int j, int kb, uint32_t lds_addr) const {
        if constexpr (TURN) kb = kb + turn < blocks ? kb + turn : kb + turn - blocks;
        const int64_t moved = kb * step, left = end - moved;
        const uint64_t b = base + moved;
        const u32x4 rsrc = {static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32) & 0xffffu, 0xffffffffu, 0x00020000u};
        const uint32_t last = left > 0xfffffff0ll ? 0xfffffff0u : static_cast<uint32_t>(left);
        dma16(rsrc, min(off[j], last), 0u, lds_addr);
    }
};

// TURN: for one row of tiles.  W is then read once, and its rows may lie a power of two apart: workgroups begin at different k-blocks, so
// that they read from different memory channels (128 x 128256 x 4096 forward, not in a cache: 250 -> 205 us, both passes 1199 -> 1110; with more rows of tiles those
// that are worked on together share what they read).
template <typename Cfg, int PRODUCT, bool TURN>
__global__ __launch_bounds__(Cfg::NT, Cfg::MINB) void head_gemm_kernel(const HeadGemm a) {
    constexpr int NW = Cfg::NW, WGN = Cfg::WGN, WM = Cfg::WM, WN = Cfg::WN, TM = Cfg::TM, TN = Cfg::TN, NHALF = Cfg::NHALF;
    constexpr int HALF_BYTES = Cfg::HALF_BYTES, DPH = Cfg::DPH, RING = Cfg::RING, ROWK = Cfg::BT * 2;
    constexpr bool PK = PRODUCT == HEAD_DWEIGHT, QK = PRODUCT == HEAD_DHIDDEN || PRODUCT == HEAD_DWEIGHT;
    extern __shared__ __align__(16) uint16_t lds[];
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint16_t*)lds));
    const int count = *a.count;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WGN;
    const int rows = PRODUCT == HEAD_DWEIGHT ? a.rows : count;
    const int row_tiles = (rows + Cfg::BT - 1) / Cfg::BT, tiles = row_tiles * a.col_tiles;
    const int id = static_cast<int>(blockIdx.x), splits = PRODUCT == HEAD_DHIDDEN ? *a.splits : 1;
    if (id >= tiles * splits) return;
    const int place = place_of(id, tiles * splits), split = place / tiles;
    const TileAt tile = tile_at(place - split * tiles, row_tiles, a.col_tiles);
    const int i0 = tile.row * Cfg::BT, j0 = tile.col * Cfg::BT;
    // A tile at the end of the rows or columns may have nothing in its second half: the waves there fetch their share of the operands and keep
    // the barriers, but leave the matrix pipes to the others.  Waves w and w + 4 share a SIMD: where columns are empty the second
    // row of waves is turned by two, so that every SIMD has one wave of either kind.
    const int cols = PRODUCT == HEAD_STATS || PRODUCT == HEAD_GRAD ? a.vocab - a.vocab_begin : a.cols;
    const bool narrow = cols - j0 <= Cfg::BT / 2, low = rows - i0 <= Cfg::BT / 2;
    const int wn = WGN == 4 && narrow ? (wave % WGN) ^ (wm * 2) : wave % WGN;
    const bool empty = (narrow && wn * WN >= Cfg::BT / 2) || (low && wm * WM >= Cfg::BT / 2);
    // k-blocks of this share
    const int all = PRODUCT == HEAD_DWEIGHT ? (count + BK - 1) / BK : a.kblocks;
    const int k0 = static_cast<int>(static_cast<int64_t>(all) * split / splits), nk = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / splits) - k0;

    f32x16 acc[TM][TN];
#pragma unroll
    for (int x = 0; x < TM; ++x)
#pragma unroll
        for (int y = 0; y < TN; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[x][y][i] = 0.f;

    if (nk > 0) {
        Source<Cfg, PK, TURN> sp_;
        Source<Cfg, QK, TURN> sq_;
        sp_.set(a.P, a.ldp, a.end_p, i0, a.row_limit, k0 * BK, lane, wave);
        sq_.set(a.Q, a.ldq, a.end_q, j0, a.col_limit, k0 * BK, lane, wave);
        if constexpr (TURN) {
            sp_.turn = sq_.turn = (a.vocab_begin / Cfg::BT + tile.col) % nk;
            sp_.blocks = sq_.blocks = nk;
        }
        const uint32_t dst0 = lds_base + wave * 1024;
#pragma unroll
        for (int h = 0; h < NHALF; ++h)
            if (h < 2 * nk) {
#pragma unroll
                for (int j = 0; j < DPH; ++j) {
                    if (h & 1) sq_.issue(j, h >> 1, dst0 + h * HALF_BYTES + j * NW * 1024);
                    else sp_.issue(j, h >> 1, dst0 + h * HALF_BYTES + j * NW * 1024);
                }
            }

        const int swz = (lane >> 1) & 7, c0 = (lane >> 5) ^ swz, r4 = (lane & 15) >> 2;
        const int koff[4] = {c0 * 16, (c0 ^ 2) * 16, (c0 ^ 4) * 16, (c0 ^ 6) * 16};
        const uint32_t pfrag = lds_base + (wm * WM + (lane & 31)) * ROW_BYTES, qfrag = lds_base + (wn * WN + (lane & 31)) * ROW_BYTES;
        uint32_t ptr_off[TM], qtr_off[TN];
#pragma unroll
        for (int x = 0; x < TM; ++x)
            ptr_off[x] = ((lane >> 5) * 8 + r4) * ROWK + (lane & 3) * 8 + ((wm * (WM / 32) + x) ^ r4) * 64 + ((lane >> 4) & 1) * 32;
#pragma unroll
        for (int y = 0; y < TN; ++y)
            qtr_off[y] = ((lane >> 5) * 8 + r4) * ROWK + (lane & 3) * 8 + ((wn * (WN / 32) + y) ^ r4) * 64 + ((lane >> 4) & 1) * 32;

        if (2 * nk >= NHALF) NS_WAIT_VMCNT((NHALF - 2) * DPH);
        else NS_WAIT_VMCNT(0);
        __syncthreads();

        // The loop is that of ns_gemm_kernel: fragments double buffered over k-steps across blocks, reads and waits written out, the
        // transfers of a pair of half-stages spread over four k-steps (there: why each is where it is).
        Frags<TM, PK> af[2];
        Frags<TN, QK> bf[2];
        constexpr int KSTEPS = BK / 16, NFRAG = (PK ? 2 * TM : TM) + (QK ? 2 * TN : TN), DPK = 2 * DPH / KSTEPS;
        static_assert(NFRAG < 16 && 2 * DPH % KSTEPS == 0 && DPH % DPK == 0 && DPK <= TM, "reads in flight, transfers per k-step");
        const auto load = [&](int buf, int sp, int sq, int ks) __attribute__((always_inline)) {
            if constexpr (PK) FragLoadTr<TM, ROWK>::run(af[buf].tr, ptr_off, lds_base + sp * HALF_BYTES + ks * 16 * ROWK);
            else FragLoad<TM>::run(af[buf].row, pfrag + sp * HALF_BYTES + koff[ks]);
            if constexpr (QK) FragLoadTr<TN, ROWK>::run(bf[buf].tr, qtr_off, lds_base + sq * HALF_BYTES + ks * 16 * ROWK);
            else FragLoad<TN>::run(bf[buf].row, qfrag + sq * HALF_BYTES + koff[ks]);
        };
        const auto multiply = [&](int x, int buf) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < TN; ++y)
                acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, bf[buf].get(y)),
                                                                    __builtin_bit_cast(bf16x8, af[buf].get(x)), acc[x][y], 0, 0, 0);
        };
        uint32_t ddst[2] = {0, 0};
        int dk[2] = {0, 0};
        const auto transfer = [&](int jj) __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            if (jj / DPH == 0) sq_.issue(jj % DPH, dk[0], ddst[0] + (jj % DPH) * NW * 1024);
            else sp_.issue(jj % DPH, dk[1], ddst[1] + (jj % DPH) * NW * 1024);
            __builtin_amdgcn_sched_barrier(0);
        };
        int sp = 0, sq = 1, kb = 0;
        const auto block = [&](auto more) __attribute__((always_inline)) {
            constexpr int MORE = decltype(more)::value;
            int spn = sp + 2, sqn = sq + 2;
            spn = spn >= NHALF ? spn - NHALF : spn;
            sqn = sqn >= NHALF ? sqn - NHALF : sqn;
#pragma unroll
            for (int ks = 0; ks + 1 < KSTEPS; ++ks) {
                const int cur = ks & 1, nxt = cur ^ 1;
                load(nxt, sp, sq, ks + 1);
                wait_both<NFRAG>(af[cur], bf[cur]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < TM; ++x) {
                    multiply(x, cur);
                    if (x < DPK && kb > 0 && (MORE == RING || (MORE == RING - 1 && (ks + 1) * DPK + x < DPH))) transfer((ks + 1) * DPK + x);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            constexpr int cur = (KSTEPS - 1) & 1, nxt = cur ^ 1;
            wait_both<0>(af[cur], bf[cur]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < TM / 2; ++x) multiply(x, cur);
            __builtin_amdgcn_sched_barrier(0);
            if (MORE > 0) {
                NS_WAIT_VMCNT((MORE == RING ? NHALF - 4 : MORE > 0 ? 2 * MORE - 2 : 0) * DPH);
                __builtin_amdgcn_s_barrier();
                const int h0 = 2 * kb + NHALF;
                ddst[0] = dst0 + sp * HALF_BYTES;
                ddst[1] = dst0 + sq * HALF_BYTES;
                dk[0] = h0 >> 1;
                dk[1] = (h0 + 1) >> 1;
                load(nxt, spn, sqn, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int x = TM / 2; x < TM; ++x) {
                multiply(x, cur);
                if (MORE == RING) {
#pragma unroll
                    for (int jj = 0; jj < DPK; ++jj)
                        if (jj * (TM - TM / 2) / DPK == x - TM / 2) transfer(jj);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (MORE > 0) wait_both<0>(af[0], bf[0]);
            sp = spn;
            sq = sqn;
        };
        if (empty) {
            const auto pass = [&](auto more) __attribute__((always_inline)) {
                constexpr int MORE = decltype(more)::value;
                if (kb > 0) {
#pragma unroll
                    for (int jj = DPK; jj < 2 * DPH; ++jj)
                        if (MORE == RING || (MORE == RING - 1 && jj < DPH)) transfer(jj);
                }
                if (MORE > 0) {
                    NS_WAIT_VMCNT((MORE == RING ? NHALF - 4 : MORE > 0 ? 2 * MORE - 2 : 0) * DPH);
                    __builtin_amdgcn_s_barrier();
                    const int h0 = 2 * kb + NHALF;
                    ddst[0] = dst0 + sp * HALF_BYTES;
                    ddst[1] = dst0 + sq * HALF_BYTES;
                    dk[0] = h0 >> 1;
                    dk[1] = (h0 + 1) >> 1;
                }
                if (MORE == RING) {
#pragma unroll
                    for (int jj = 0; jj < DPK; ++jj) transfer(jj);
                }
                sp = sp + 2 >= NHALF ? sp + 2 - NHALF : sp + 2;
                sq = sq + 2 >= NHALF ? sq + 2 - NHALF : sq + 2;
            };
            for (; kb < nk - RING; ++kb) pass(std::integral_constant<int, RING>{});
            if (nk - kb == 2) {
                pass(std::integral_constant<int, 1>{});
                ++kb;
            }
            pass(std::integral_constant<int, 0>{});
        } else {
            load(0, 0, 1, 0);
            wait_both<0>(af[0], bf[0]);
            for (; kb < nk - RING; ++kb) block(std::integral_constant<int, RING>{});
            if (nk - kb == 2) {
                block(std::integral_constant<int, 1>{});
                ++kb;
            }
            block(std::integral_constant<int, 0>{});
        }
        __syncthreads();            // every wave is done with the ring
    }

    // ---- epilogue: a lane's accumulators are 4 x 4 columns of row lane % 32 in each 32 x 32 tile --------------------
    int tid_e = threadIdx.x;
    asm volatile("" : "+v"(tid_e));            // (nothing of it is formed ahead of the loop and kept there)
    const int lane_e = tid_e & 63, lr = lane_e & 31, g = lane_e >> 5;
    const int row0 = i0 + wm * WM, col0 = j0 + wn * WN;
    if constexpr (PRODUCT == HEAD_STATS) {
        // columns beyond the vocabulary do not count
        const int limit = a.vocab - col0;
        f32x2_t* const red = reinterpret_cast<f32x2_t*>(lds);               // [wave column][row of the tile]
#pragma unroll
        for (int x = 0; x < TM; ++x) {
            if (limit < WN) {
#pragma unroll
                for (int y = 0; y < TN; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (y * 32 + (i / 4) * 8 + g * 4 + i % 4 >= limit) acc[x][y][i] = -__builtin_inff();
            }
            float m = acc[x][0][0];
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, acc[x][y][i]);
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float ref = m == -__builtin_inff() ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int i = 0; i < 16; ++i) s += __builtin_amdgcn_exp2f((acc[x][y][i] - ref) * LOG2E);
            s += __shfl_xor(s, 32, 64);
            if (g == 0) red[wn * Cfg::BT + wm * WM + x * 32 + lr] = f32x2_t{m, s};
            // the target's logit, where it is one of these columns
            const int row = row0 + x * 32 + lr, at = row < rows ? a.target[row] - col0 : -1;
            const bool mine = at >= 0 && at < WN && ((at >> 2) & 1) == g;
            if (__ballot(mine)) {
                float value = 0.f;
#pragma unroll
                for (int y = 0; y < TN; ++y)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (y * 32 + (i / 4) * 8 + g * 4 + i % 4 == at) value = acc[x][y][i];
                if (mine) a.target_logit[row] = value;
            }
        }
        __syncthreads();
        for (int r = tid_e; r < Cfg::BT; r += Cfg::NT) {
            float m = red[r][0], s = red[r][1];
#pragma unroll
            for (int w = 1; w < WGN; ++w) {
                const f32x2_t o = red[w * Cfg::BT + r];
                const float top = fmaxf(m, o[0]), ref = top == -__builtin_inff() ? 0.f : top;
                s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + o[1] * __builtin_amdgcn_exp2f((o[0] - ref) * LOG2E);
                m = top;
            }
            if (i0 + r < rows) a.stats[tile.col * a.ld_stats + i0 + r] = f32x2_t{m, s};
        }
    } else if constexpr (PRODUCT == HEAD_DHIDDEN) {
        float* const part = a.part + split * a.part_stride;
#pragma unroll
        for (int x = 0; x < TM; ++x) {
            const int row = row0 + x * 32 + lr;
            if (row >= rows) continue;
#pragma unroll
            for (int y = 0; y < TN; ++y)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = col0 + y * 32 + q * 8 + g * 4;           // (the columns are padded to 64)
                    if (col >= a.cols) continue;
                    f32x4v v = {acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2], acc[x][y][4 * q + 3]};
                    float* const at = part + row * a.ld_out + col;
                    if (a.add) v += load_as<false, f32x4v>(at);
                    store_as<false>(at, v);
                }
        }
    } else {
        // 32 rows at a time go through LDS, so that a store's lanes take 128 bytes of each of 8 rows (a piece of a row at another place in each
        // of 8 rows: other banks).  (dW of 2 tokens, 32000 x 4096: 70 -> 58 us; of 500 tokens, 50257 x 1024: 78 -> 71.)
        u32x4* const strip = reinterpret_cast<u32x4*>(lds) + wave * 256;
        const float scale = PRODUCT == HEAD_DWEIGHT ? *a.scale : 1.f;
#pragma unroll
        for (int x = 0; x < TM; ++x) {
            const int row = row0 + x * 32 + lr;
            [[maybe_unused]] float both = 0.f, own = 0.f, m = 0.f, l = 0.f;
            [[maybe_unused]] int at = -1;
            if constexpr (PRODUCT == HEAD_GRAD) {
                // (rows of the tile beyond the tokens are rows of zeros, and so are their coefficients)
                const f32x4v c = a.coef[row];
                both = c[0];
                own = c[1];
                m = c[2];
                l = c[3];
                at = row < rows ? a.target[row] - a.vocab_begin - col0 : -1;
            }
#pragma unroll
            for (int y = 0; y < TN; ++y) {
                uint32_t po[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float v[2] = {acc[x][y][2 * k], acc[x][y][2 * k + 1]};
                    if constexpr (PRODUCT == HEAD_GRAD) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int c = y * 32 + (k / 2) * 8 + g * 4 + (k % 2) * 2 + i;
                            v[i] = both * __builtin_amdgcn_exp2f((v[i] - m) * LOG2E - l) - (c == at ? own : 0.f);
                            if (a.vocab_begin + col0 + c >= a.vocab) v[i] = 0.f;
                        }
                    }
                    if constexpr (PRODUCT == HEAD_DWEIGHT) {
                        v[0] *= scale;
                        v[1] *= scale;
                    }
                    po[k] = pack2bf(v[0], v[1]);
                }
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                    const auto u = __builtin_amdgcn_permlane32_swap(po[2 * q], po[2 * q + 2], false, false);
                    const auto w = __builtin_amdgcn_permlane32_swap(po[2 * q + 1], po[2 * q + 3], false, false);
                    strip[lr * 8 + ((y * 4 + q + g) ^ (lr & 7))] = u32x4{u[0], w[0], u[1], w[1]};
                }
            }
            wave_order();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = i * 8 + lane_e / 8, to = row0 + x * 32 + at;
                const u32x4 v = strip[at * 8 + ((lane_e & 7) ^ (at & 7))];
                if (PRODUCT == HEAD_GRAD || to < rows) store_pack<uint16_t, 8, false>(a.out + to * a.ld_out, col0 + (lane_e & 7) * 8, a.cols, Pack<uint16_t, 8>{v});
            }
            wave_order();
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Few tokens: W streamed through registers
// ---------------------------------------------------------------------------------------------
// A workgroup takes 64 rows of W, its four waves every fourth block of 64 channels, against up to 64 tokens, which the caches hold.  A wave's loads
// take whole lines of 128 bytes of 8 rows each, a block ahead; through LDS (of its own, so there is nothing to wait for) they become the
// fragments of 16 rows x 32 channels.  Workgroups begin at different blocks, as rows that lie a power of two apart would otherwise all be read from
// the same memory channels at a time.  The waves' sums are added in LDS.  W's bytes bound it (128256 x 4096 not in a cache, one token: 207 -> 186 us
// against fragments straight from memory, every workgroup from the first block on; 32 tokens: 233 -> 184; 32000 x 2048, one token: 33.4 -> 31.0); beyond
// 32 tokens so do the hidden states' fragments, as many bytes again from the L2 (64 tokens: 214).
constexpr int HF_THREADS = 256, HF_VOCAB = 64;
typedef float f32x4a __attribute__((ext_vector_type(4)));
template <bool TAIL>
__device__ __forceinline__ u32x4 few_chunk(const uint16_t* row, int k, int width) {
    if constexpr (!TAIL) return Pack<uint16_t, 8>::load<false>(row + k).v;
    else return load_pack<uint16_t, 8, false>(row, k, width).v;
}
template <int NT>
__global__ __launch_bounds__(HF_THREADS, NT == 4 ? 2 : NT == 2 ? 3 : 4) void head_few_kernel(const uint16_t* hidden, int64_t ld_hidden, const uint16_t* weight, int64_t ld_weight, int tokens,
                                                              int width, int vocab, const void* targets, int target_bits, f32x2_t* stats, int64_t ld_stats,
                                                              float* target_logit, int32_t* counter) {
    // a row's columns exchanged by its number, four at a time: the lanes of a token's 16 then write to different banks
    constexpr int WAVES = NT == 4 ? 2 : 4;       // whose sums lie in LDS at once (what four of them take for 64 tokens would leave two workgroups a CU)
    constexpr int TILE = HF_VOCAB * 8;           // 16-byte pieces of a wave's block
    typedef float Sums[16 * NT][HF_VOCAB];
    __shared__ u32x4 pieces[4 * TILE];           // the waves' blocks, then their sums
    static_assert(sizeof(pieces) >= WAVES * sizeof(Sums), "the waves' sums");
    Sums* const sums = reinterpret_cast<Sums*>(pieces);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kq = (lane >> 4) * 8;
    const int v0 = blockIdx.x * HF_VOCAB;
    const uint16_t* wrow[8];
    const uint16_t* hrow[NT];
#pragma unroll
    for (int i = 0; i < 8; ++i) wrow[i] = weight + min(v0 + 8 * i + (lane >> 3), vocab - 1) * ld_weight + (lane & 7) * 8;
#pragma unroll
    for (int f = 0; f < NT; ++f) hrow[f] = hidden + min(16 * f + r, tokens - 1) * ld_hidden + kq;
    if (blockIdx.x == 0 && threadIdx.x == 0) *counter = 0;       // (of the launch that joins)
    // the target of the token that the thread has in the end, where it is a row of W (requested before the rows: at the end it is waited for)
    int target = -1;
    if (const int t = threadIdx.x / (HF_THREADS / (16 * NT)); t < tokens) {
        const int64_t at = target_bits == 64 ? static_cast<const int64_t*>(targets)[t] : static_cast<const int32_t*>(targets)[t];
        if (at >= 0 && at < vocab) target = static_cast<int>(at);
    }
    f32x4a acc[4][NT];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[f][t] = f32x4a{0.f, 0.f, 0.f, 0.f};
    u32x4 next[8], next_h[2][NT];
    const auto fetch = [&](auto tail, int k) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail)::value;
#pragma unroll
        for (int i = 0; i < 8; ++i) next[i] = few_chunk<TAIL>(wrow[i], k, width - (lane & 7) * 8);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) next_h[s][t] = few_chunk<TAIL>(hrow[t], k + 32 * s, width - kq);
    };
    // (piece c of row v lies at c ^ (v / 2 % 8) of the row's eight: sixteen rows next to each other are on all banks)
    u32x4* const tile = pieces + wave * TILE;
    const int to = (lane >> 3) * 8 + ((lane & 7) ^ (lane >> 4)), from = r * 8 + ((lane >> 4) ^ (r >> 1));
    const auto multiply = [&](auto more, int k) __attribute__((always_inline)) {
        u32x4 h[2][NT];
#pragma unroll
        for (int i = 0; i < 8; ++i) tile[64 * i + (to ^ (i & 1) * 4)] = next[i];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < NT; ++t) h[s][t] = next_h[s][t];
        if constexpr (decltype(more)::value) fetch(std::false_type{}, k);
        wave_order();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const bf16x8 w = __builtin_bit_cast(bf16x8, tile[128 * f + (from ^ s * 4)]);
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, __builtin_bit_cast(bf16x8, h[s][t]), acc[f][t], 0, 0, 0);
            }
        wave_order();
    };
    const int whole = width / 64, turn = whole > 0 ? blockIdx.x % whole : 0;
    const auto block = [&](int b) { return (b + turn < whole ? b + turn : b + turn - whole) * 64; };
    if (wave < whole) {
        fetch(std::false_type{}, block(wave));
        int b = wave;
#pragma unroll 1
        for (; b + 4 < whole; b += 4) multiply(std::true_type{}, block(b + 4));
        multiply(std::false_type{}, 0);
    }
    if (width % 64 && wave == whole % 4) {
        fetch(std::true_type{}, whole * 64);
        multiply(std::false_type{}, 0);
    }
    __syncthreads();                             // every wave is done with its block
    // a lane holds rows 4 (lane / 16) .. + 3 of W for token lane % 16
    const auto slot = [&](int f, int t) { return reinterpret_cast<f32x4a*>(&sums[wave % WAVES][16 * t + r][(16 * f + 4 * (lane >> 4)) ^ (r << 2)]); };
    if (wave >= 4 - WAVES) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int t = 0; t < NT; ++t) *slot(f, t) = acc[f][t];
    }
    if (WAVES < 4) __syncthreads();
    if (wave < 4 - WAVES) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int t = 0; t < NT; ++t) *slot(f, t) += acc[f][t];
    }
    __syncthreads();
    // as many threads to each token as there are: maximum and sum of the token's columns here, and its target where that is one of them
    constexpr int P = HF_THREADS / (16 * NT), C = HF_VOCAB / P;
    const int t = threadIdx.x / P, part = threadIdx.x % P, turned = (t & 15) << 2;
    float x[C], m = -__builtin_inff(), sum = 0.f;
#pragma unroll
    for (int j = 0; j < C / 4; ++j) {
        const int col = part * C + 4 * j;
        f32x4a v = *reinterpret_cast<const f32x4a*>(&sums[0][t][col ^ turned]) + *reinterpret_cast<const f32x4a*>(&sums[1][t][col ^ turned]);
        if constexpr (WAVES == 4) v += *reinterpret_cast<const f32x4a*>(&sums[2][t][col ^ turned]) + *reinterpret_cast<const f32x4a*>(&sums[3][t][col ^ turned]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[4 * j + i] = v0 + col + i < vocab ? v[i] : -__builtin_inff();
            m = fmaxf(m, x[4 * j + i]);
            if (target == v0 + col + i) target_logit[t] = v[i];
        }
    }
    m = group_reduce<P>(m, [](float u, float v) { return fmaxf(u, v); });
    const float ref = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int i = 0; i < C; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * LOG2E);
    sum = group_sum<P>(sum);
    if (part == 0 && t < tokens) stats[blockIdx.x * ld_stats + t] = f32x2_t{m, sum};
}

// ---------------------------------------------------------------------------------------------
// The launches around the products
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t target_of(const MuonHeadLoss& a, int64_t t) {
    return a.target_bits == 64 ? static_cast<const int64_t*>(a.targets)[t] : static_cast<const int32_t*>(a.targets)[t];
}
// A target as the other kernels see it: -1 where it is outside of the vocabulary.
__device__ __forceinline__ int target_in(const MuonHeadLoss& a, int64_t target) { return target >= 0 && target < a.vocab ? static_cast<int>(target) : -1; }

// Numbers the tokens that take part, in order: order[row] = token for the first `count` rows, after them ~token of the ignored
// ones (whose outputs are written here); rows[row] = target.  order[tokens] = count.
constexpr int HO_THREADS = 1024;
__global__ __launch_bounds__(HO_THREADS) void head_order_kernel(const MuonHeadLoss a) {
    __shared__ int before[HO_THREADS / 64 + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t each = (a.tokens + HO_THREADS - 1) / HO_THREADS, begin = min(threadIdx.x * each, a.tokens), end = min(begin + each, a.tokens);
    int n = 0;
    for (int64_t t = begin; t < end; ++t) n += target_of(a, t) != a.ignore_index;
    int upto = n;                                            // of this lane and those before it
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    if (lane == 63) before[wave + 1] = upto;
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 0; w < HO_THREADS / 64; ++w) before[w + 1] += before[w];
    __syncthreads();
    const int count = before[HO_THREADS / 64];
    int64_t at = before[wave] + upto - n, out = count + (begin - at);
    for (int64_t t = begin; t < end; ++t) {
        const int64_t target = target_of(a, t);
        const bool on = target != a.ignore_index;
        const int64_t row = on ? at++ : out++;
        a.order[row] = static_cast<int32_t>(on ? t : ~t);
        a.rows[row] = on ? target_in(a, target) : -1;
        if (!on) {
            a.losses[t] = 0.f;
            a.lse[t] = 0.f;
        }
    }
    if (threadIdx.x == 0) {
        a.order[a.tokens] = count;
        *a.part = static_cast<float>(count > 0 ? count : 1);
        *a.counter = 0;
    }
}

// The same for few tokens, and their hidden states' copy with it: every workgroup counts all of them, and a wave takes one (64 x 50257 x 768:
// 27.4 -> 25.0 us against a launch for each).
constexpr int HO_FEW = 1024, HO_EACH = 4, HO_WAVES = 4;
__global__ __launch_bounds__(HO_WAVES * 64) void head_order_few_kernel(const MuonHeadLoss a, uint16_t* rows, int ld, int64_t padded) {
    __shared__ int counted[HO_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tokens = static_cast<int>(a.tokens), first = blockIdx.x * HO_WAVES;
    int n = 0;                                               // those that take part, and in the upper half those before this workgroup's
#pragma unroll
    for (int i = 0; i < HO_EACH; ++i) {
        const int t = i * HO_WAVES * 64 + threadIdx.x;
        if (t < tokens && target_of(a, t) != a.ignore_index) n += t < first ? 0x10001 : 1;
    }
    static_assert(HO_EACH * HO_WAVES * 64 == HO_FEW, "all tokens are counted");
    const int t = first + wave;
    const int64_t target = t < tokens ? target_of(a, t) : a.ignore_index;
    const uint64_t here = __ballot(lane < HO_WAVES && first + lane < tokens && target_of(a, first + lane) != a.ignore_index);
    n = group_reduce<64>(n, [](int u, int v) { return u + v; });
    if (lane == 0) counted[wave] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < HO_WAVES; ++w) n += counted[w];
    const int count = n & 0xffff, before = (n >> 16) + __builtin_popcountll(here & ((1ull << wave) - 1));
    const bool on = target != a.ignore_index;
    if (t < tokens) {
        const int row = on ? before : count + (t - before);
        if (lane == 0) {
            a.order[row] = on ? t : ~t;
            a.rows[row] = on ? target_in(a, target) : -1;
            if (!on) {
                a.losses[t] = 0.f;
                a.lse[t] = 0.f;
            }
        }
        if (on) {
            const uint16_t* const from = static_cast<const uint16_t*>(a.hidden) + t * a.ld_hidden;
            for (int e = lane * 8; e < ld; e += 512) load_pack<uint16_t, 8, false>(from, e, a.width).template store<false>(rows + static_cast<int64_t>(row) * ld + e);
        }
    }
    if (t >= count && t < padded)
        for (int e = lane * 8; e < ld; e += 512) Pack<uint16_t, 8>::zero().template store<false>(rows + static_cast<int64_t>(t) * ld + e);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.order[tokens] = count;
        *a.part = static_cast<float>(count > 0 ? count : 1);
        *a.counter = 0;
    }
}

// The shares that the k-blocks of e W are cut into, formed by a wave.  A launch takes as many rounds of workgroups as it has tiles for the
// places on the GPU, a tile as long as its share and about six k-blocks more (its prologue and epilogue), and each share's sums
// are written and read once (in the time of a k-block 5 MB are): the number of shares with the least of that.  (4096 x 32000 x 2048:
// 504 -> 438 us against a fixed 4; 5003 x 50257 x 1600, a third ignored: 658 -> 534.)
constexpr int HD_SPLITS = 128;
__device__ __forceinline__ int splits_for(int64_t count, int ld, int kblocks, int most, int tile) {
    const int tiles = static_cast<int>((count + tile - 1) / tile) * ((ld + tile - 1) / tile), places = tile == 256 ? HD_CUS : 2 * HD_CUS;
    uint64_t least = ~0ull;
    for (int s = 1 + static_cast<int>(threadIdx.x & 63); s <= most; s += 64) {
        const int64_t cost = static_cast<int64_t>((tiles * s + places - 1) / places) * ((kblocks + s - 1) / s + 6) + s * count * ld / 625000;
        least = min(least, static_cast<uint64_t>(cost) << 8 | s);
    }
    return static_cast<int>(group_reduce<64>(least, [](uint64_t u, uint64_t v) { return min(u, v); }) & 255);
}

// The tokens' common factor g of a mean or sum, without its power of two: e is formed and rounded without it, and the products are
// multiplied by it.  With it in e, every target's entry near -g is rounded the same way, and the errors of the sums over tokens
// add up (1.7 times those of the rest together, 5003 tokens, 3352 of them taking part).
__device__ __forceinline__ float common_factor(const MuonHeadLoss& a) {
    if (a.reduction == MUON_AMD_REDUCE_NONE || !a.dloss) return 1.f;
    const float g = *a.dloss / (a.reduction == MUON_AMD_REDUCE_MEAN ? *a.part : 1.f), m = __builtin_amdgcn_frexp_mantf(g);
    return g != 0.f && fabsf(g) < __builtin_inff() ? m : 1.f;
}

// The hidden states of the rows, in bf16 rows of `ld` elements with zeros beyond the width, up to a whole tile of rows; backward their
// coefficients too.  A wave for each row.
__global__ __launch_bounds__(256) void head_gather_kernel(const MuonHeadLoss a, uint16_t* rows, int ld, f32x4v* coef, float* scale, int kblocks, int most_splits, int tile) {
    const int lane = threadIdx.x & 63;
    const float factor = coef ? common_factor(a) : 1.f;
    const int64_t count = a.order[a.tokens];
    if (coef && blockIdx.x == 0 && threadIdx.x < 64) {
        const int splits = splits_for(count, ld, kblocks, most_splits, tile);
        if (threadIdx.x == 0) {
            scale[0] = factor;
            reinterpret_cast<int32_t*>(scale)[1] = splits;
        }
    }
    const int64_t padded = (count + HD_TILE - 1) / HD_TILE * HD_TILE;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); r < padded; r += static_cast<int64_t>(gridDim.x) * 4) {
        const int token = r < count ? a.order[r] : -1;
        const uint16_t* const from = static_cast<const uint16_t*>(a.hidden) + (token >= 0 ? token : 0) * a.ld_hidden;
        for (int e = lane * 8; e < ld; e += 512)
            (token >= 0 ? load_pack<uint16_t, 8, false>(from, e, a.width) : Pack<uint16_t, 8>::zero()).template store<false>(rows + r * ld + e);
        if (coef && lane == 0) {
            f32x4v c = {0.f, 0.f, 0.f, 0.f};
            if (token >= 0) {
                float g = a.dloss ? a.dloss[a.reduction == MUON_AMD_REDUCE_NONE ? token * a.ld_dloss : 0] : 0.f;
                if (a.reduction == MUON_AMD_REDUCE_MEAN) g /= *a.part;
                const float z = a.dlse ? a.dlse[token * a.ld_dlse] : 0.f;
                // (a target outside of the vocabulary: no number, as the loss)
                c = f32x4v{a.rows[r] >= 0 ? (g + z) / factor : __builtin_nanf(""), g / factor, a.stats[2 * r], a.stats[2 * r + 1]};
            }
            coef[r] = c;
        }
    }
}

// W with rows of `ld` elements, zeros beyond its width: where its own rows are no multiples of 128 bytes at 16-byte addresses.
__global__ __launch_bounds__(256) void head_pad_kernel(const uint16_t* weight, int64_t ld_weight, int64_t vocab, int width, uint16_t* out, int ld) {
    const int64_t packs = vocab * (ld / 8);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < packs; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / (ld / 8);
        const int e = static_cast<int>(i % (ld / 8)) * 8;
        load_pack<uint16_t, 8, false>(weight + r * ld_weight, e, width).template store<false>(out + r * ld + e);
    }
}

// Joins the statistics of a row's column tiles, and forms its loss; the workgroup that is done last adds up the losses.  16 rows to a
// workgroup, 64 threads to each.  FEW: the rows are the tokens, order[token] = ~token where one is ignored, and nothing of that
// has been written yet.
constexpr int HJ_THREADS = 1024, HJ_ROWS = 16, HJ_SHARES = HJ_THREADS / HJ_ROWS;
template <bool FEW>
__global__ __launch_bounds__(HJ_THREADS) void head_join_kernel(const MuonHeadLoss a, const f32x2_t* stats, int64_t ld_stats, int tiles, const float* target_logit,
                                                               float* left) {
    __shared__ float tops[HJ_SHARES][HJ_ROWS], sums[HJ_SHARES][HJ_ROWS];
    __shared__ bool last;
    const int r = threadIdx.x % HJ_ROWS, share = threadIdx.x / HJ_ROWS;
    const int64_t count = FEW ? a.tokens : a.order[a.tokens], row = static_cast<int64_t>(blockIdx.x) * HJ_ROWS + r;
    const auto join = [](float& m, float& s, float m2, float s2) {
        const float top = fmaxf(m, m2), ref = top == -__builtin_inff() ? 0.f : top;
        s = s * __builtin_amdgcn_exp2f((m - ref) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * LOG2E);
        m = top;
    };
    float m = -__builtin_inff(), s = 0.f;
    if (row < count) {
        int i = share;
        for (; i + 3 * HJ_SHARES < tiles; i += 4 * HJ_SHARES) {
            f32x2_t v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = stats[(i + k * HJ_SHARES) * ld_stats + row];
#pragma unroll
            for (int k = 0; k < 4; ++k) join(m, s, v[k][0], v[k][1]);
        }
        for (; i < tiles; i += HJ_SHARES) {
            const f32x2_t v = stats[i * ld_stats + row];
            join(m, s, v[0], v[1]);
        }
    }
    tops[share][r] = m;
    sums[share][r] = s;
    __syncthreads();
    for (int half = HJ_SHARES / 2; half > 0; half >>= 1) {
        if (share < half) {
            float m1 = tops[share][r], s1 = sums[share][r];
            join(m1, s1, tops[share + half][r], sums[share + half][r]);
            tops[share][r] = m1;
            sums[share][r] = s1;
        }
        __syncthreads();
    }
    if (threadIdx.x < 64) {
        float loss = 0.f;
        int token = -1, target = -1;
        if (share == 0 && row < count) {
            if constexpr (FEW) {
                const int64_t t = target_of(a, row);
                token = static_cast<int>(t != a.ignore_index ? row : ~row);
                target = token >= 0 ? target_in(a, t) : -1;
                a.order[row] = token;
                a.rows[row] = target;
                if (token < 0) {
                    a.losses[row] = 0.f;
                    a.lse[row] = 0.f;
                }
            } else {
                token = a.order[row];
                target = a.rows[row];
            }
        }
        if (token >= 0) {
            m = tops[0][r] == -__builtin_inff() ? 0.f : tops[0][r];
            const float l = __log2f(sums[0][r]);
            a.stats[2 * row] = m;
            a.stats[2 * row + 1] = l;
            loss = target >= 0 ? fmaf(l, LN2, m - target_logit[row]) : __builtin_nanf("");
            a.losses[token] = loss;
            a.lse[token] = fmaf(l, LN2, m);
        }
        loss = group_sum<64>(loss);
        const int part = FEW ? __builtin_popcountll(__ballot(token >= 0)) : 0;
        if (threadIdx.x == 0) {
            __hip_atomic_store(&left[2 * blockIdx.x], loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (FEW) __hip_atomic_store(&left[2 * blockIdx.x + 1], __int_as_float(part), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = gridDim.x == 1 || __hip_atomic_fetch_add(a.counter, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.x) - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    if constexpr (FEW) {                         // (few workgroups)
        if (threadIdx.x > 0) return;
        float total = 0.f;
        int n = 0;
        for (unsigned g = 0; g < gridDim.x; ++g) {
            total += __hip_atomic_load(&left[2 * g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            n += __float_as_int(__hip_atomic_load(&left[2 * g + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        }
        const float part = static_cast<float>(n > 0 ? n : 1);
        a.order[a.tokens] = static_cast<int32_t>(a.tokens);
        *a.part = part;
        if (a.loss) *a.loss = a.reduction == MUON_AMD_REDUCE_MEAN ? total / part : total;
        return;
    }
    if (!a.loss) return;
    float total = 0.f;
    for (unsigned g = threadIdx.x; g < gridDim.x; g += HJ_THREADS) total += __hip_atomic_load(&left[2 * g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    total = group_sum<64>(total);
    if ((threadIdx.x & 63) == 0) tops[0][threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x > 0) return;
    total = 0.f;
    for (int w = 0; w < HJ_THREADS / 64; ++w) total += tops[0][w];
    *a.loss = a.reduction == MUON_AMD_REDUCE_MEAN ? total / *a.part : total;
}

// Adds the shares of the hidden states' gradient and writes it to the tokens; zeros for those that take no part.  A wave takes 512 channels
// of a row; where there are many shares (and few rows), the four waves of a workgroup share them.
constexpr int HH_MANY = 8;
__global__ __launch_bounds__(256) void head_dhidden_kernel(const MuonHeadLoss a, const float* part, int64_t stride, int ld, const float* scale) {
    __shared__ float sums[3][64][9];                         // (a place more, so that lanes fall on different banks)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, shares = reinterpret_cast<const int32_t*>(scale)[1], segments = (a.width + 511) / 512;
    const bool many = shares >= HH_MANY;
    const float factor = scale[0];
    const int64_t count = a.order[a.tokens], items = a.tokens * segments;
    const int first = many ? wave : 0, step = many ? 4 : 1;
    for (int64_t item = many ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + wave; item < items; item += many ? gridDim.x : static_cast<int64_t>(gridDim.x) * 4) {
        const int64_t r = item / segments;
        const int e = static_cast<int>(item % segments) * 512 + lane * 8, at = a.order[r];
        const bool on = at >= 0;
        float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (on && r < count && e < a.width) {
            const float* const p = part + r * ld + e;
            const auto add = [&](auto together, int s) __attribute__((always_inline)) {
                constexpr int K = decltype(together)::value;
                f32x4v v[K][2];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    v[k][0] = load_as<true, f32x4v>(p + (s + k * step) * stride);
                    v[k][1] = load_as<true, f32x4v>(p + (s + k * step) * stride + 4);
                }
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[i] += v[k][i / 4][i % 4];
            };
            int s = first;
            for (; s + 3 * step < shares; s += 4 * step) add(std::integral_constant<int, 4>{}, s);
            for (; s < shares; s += step) add(std::integral_constant<int, 1>{}, s);
        }
        if (many) {
            if (wave > 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[wave - 1][lane][i] = sum[i];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += sums[0][lane][i] + (sums[1][lane][i] + sums[2][lane][i]);
            __syncthreads();
            if (wave > 0) continue;
        }
        if (e >= a.width) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] *= factor;
        uint16_t* const out = static_cast<uint16_t*>(a.dhidden) + static_cast<int64_t>(on ? at : ~at) * a.width;
        store_pack<uint16_t, 8, false>(out, e, a.width, Pack<uint16_t, 8>::of(sum));
    }
}

// ---------------------------------------------------------------------------------------------
// How a call is laid out
// ---------------------------------------------------------------------------------------------
// Bytes of e: the larger the piece of the vocabulary, the less its sums' reading and writing weighs.  At least 4096 columns
// whatever the number of tokens.
constexpr int64_t HD_PIECE_BYTES = int64_t(1) << 30;

static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

struct HeadPlan {
    bool few, padded;              // streamed; W through a padded copy
    bool large;                    // 256 x 256 tiles in the products over tokens
    int64_t rows, ld;              // padded rows and width
    int tile, col_tiles;           // of the statistics
    int64_t piece;                 // columns of e
    int pieces, splits, dh_tile, dw_tile;
    // offsets in the workspace, in bytes
    int64_t hidden, weight, stats, logit, left, coef, scale, e, part, bytes;
};

// Whether the products of tokens with the vocabulary take less time in 256 x 256 tiles, one to a CU, than in 128 x 128 tiles, two to a CU: a round
// of the latter does half the work, and takes a little more than half the time.
static bool fewer_rounds(int64_t tokens, int64_t vocab) {
    const auto rounds = [&](int64_t tile, int64_t places) { return ((tokens + tile - 1) / tile * ((vocab + tile - 1) / tile) + places - 1) / places; };
    return 100 * rounds(256, HD_CUS) <= 62 * rounds(128, 2 * HD_CUS);
}

static HeadPlan head_plan(const MuonHeadLoss& a, bool backward) {
    HeadPlan p{};
    const int64_t n = a.tokens, d = a.width, v = a.vocab;
    p.ld = up(d, BK);
    p.rows = up(n, HD_TILE);
    p.padded = d % BK != 0 || a.ld_weight % 8 != 0 || reinterpret_cast<uintptr_t>(a.weight) % 16 != 0;
    // Streamed: up to 32 tokens (32 x 128256 x 4096: streamed 184 us, by tiles 244); up to 64 where the tiles would need a copy of W, or W is small, or its
    // rows are long.  W not in a cache, streamed and by tiles, on the side of the streams: 64 x 32000 x 2048 37 and 44 us, 40 x 128256 x 1024 58 and 62, 64 x
    // 20000 x 1024 21.0 and 26.5, 64 x 8000 x 512 15.2 and 18.4, 48 x 100000 x 1000 (copied) 74 and 132; of the tiles: 64 x 200000 x 128 38 and 31, 64 x
    // 262144 x 256 57 and 45, 64 x 128256 x 512 43.7 and 39.7, 64 x 128256 x 960 65 and 62, 64 x 50257 x 768 30.4 and 30.2 (in the last cache 26.6 and 24.6).
    // Shorter rows and more tokens are for the tiles, and whole rounds of them; near the border either may lose a tenth (48 x 100000 x 896 47 and 54, 33 x
    // 50257 x 768 27 and 30, 40 x 128256 x 512 39.5 both).
    p.few = !backward && (n <= HD_FEW / 2 || (n <= HD_FEW && (p.padded || d >= 1024 || v * d < (1 << 24))));
    p.padded = p.padded && !p.few;
    p.large = fewer_rounds(n, v);
    p.tile = p.few ? HF_VOCAB : p.large ? 256 : 128;
    p.col_tiles = static_cast<int>(up(v, p.tile) / p.tile);
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t begin = at;
        at += up(bytes, 256);
        return begin;
    };
    if (!p.few) p.hidden = take(p.rows * p.ld * 2);
    if (p.padded) p.weight = take(v * p.ld * 2);
    if (!backward) {
        p.stats = take(p.rows * p.col_tiles * 8);
        p.logit = take(p.rows * 4);
        p.left = take((n + HJ_ROWS - 1) / HJ_ROWS * 8);
    } else {
        p.coef = take(p.rows * 16);
        p.scale = take(8);
        const int64_t fit = HD_PIECE_BYTES / (p.rows * 2) / 256 * 256, most = fit < 4096 ? 4096 : fit;
        p.pieces = static_cast<int>((up(v, 256) + most - 1) / most);
        p.piece = up((v + p.pieces - 1) / p.pieces, 256);
        p.pieces = static_cast<int>((v + p.piece - 1) / p.piece);
        p.e = take(p.rows * p.piece * 2);
        // at most so many shares (the tokens that take part decide, on the device): of 8 k-blocks or more each, in half a GiB or one share.  Tiles of
        // 128 x 128 where those of 256 x 256 are few.
        // (dW: a few k-blocks of two 128 x 128 tiles keep a CU busier than those of a large one, 130 x 100000 x 768 234 and 243 us, but where tiles are
        // many their prologues add up: 65 x 128256 x 4096 617 us by large ones and 711, 250 x 128256 x 4096 736 and 867, 1000 x 50257 x 2048 948 and 963;
        // a single k-block has four small tiles to a CU: 2 x 32000 x 4096 151 and 146)
        const int64_t large_tiles = (up(v, 256) / 256) * (up(d, 256) / 256);
        p.dw_tile = p.rows > 512 || (n > BK && large_tiles >= 8 * HD_CUS) ? 256 : 128;
        p.dh_tile = (p.rows / 256) * ((p.ld + 255) / 256) >= 64 ? 256 : 128;
        int64_t most_splits = HD_SPLITS;
        if (most_splits > p.piece / BK / 8) most_splits = p.piece / BK / 8;
        if (most_splits > HD_PIECE_BYTES / 2 / (p.rows * p.ld * 4)) most_splits = HD_PIECE_BYTES / 2 / (p.rows * p.ld * 4);
        p.splits = static_cast<int>(most_splits > 0 ? most_splits : 1);
        p.part = take(p.splits * p.rows * p.ld * 4);
    }
    p.bytes = at;
    return p;
}

static int check_head(const MuonHeadLoss* a, const char* what) {
    MUON_REQUIRE(a, "%s: null arguments", what);
    MUON_REQUIRE(a->tokens > 0 && a->tokens <= (1 << 24) && a->vocab > 0 && a->vocab <= (1 << 24) && a->width > 0 && a->width <= (1 << 16),
                 "%s: tokens=%lld vocab=%d width=%d", what, static_cast<long long>(a->tokens), a->vocab, a->width);
    MUON_REQUIRE(a->hidden && a->weight && a->targets && a->order && a->rows && a->stats && a->part && a->workspace, "%s: null pointer", what);
    MUON_REQUIRE(a->target_bits == 32 || a->target_bits == 64, "%s: target_bits=%d", what, a->target_bits);
    MUON_REQUIRE(a->reduction >= MUON_AMD_REDUCE_NONE && a->reduction <= MUON_AMD_REDUCE_MEAN, "%s: reduction=%d", what, a->reduction);
    MUON_REQUIRE(reinterpret_cast<uintptr_t>(a->workspace) % 256 == 0, "%s: the workspace is not at a multiple of 256 bytes", what);
    MUON_REQUIRE(a->ld_weight >= 0 && a->ld_weight <= (int64_t(1) << 21), "%s: ld_weight=%lld", what, static_cast<long long>(a->ld_weight));
    return MUON_AMD_OK;
}

// `most` k-blocks in a workgroup: where these are few, the ring is as long as they need, and more workgroups share a CU (their prologues and
// epilogues are all there is; dW of 2 tokens, 32000 x 4096: 78 -> 70 us, of 20 tokens, 50257 x 768: 23.6 -> 21.0).
template <typename Cfg, int PRODUCT, bool TURN>
static int launch_product(const HeadGemm& g, int64_t most, hipStream_t s) {
    const int64_t grid = static_cast<int64_t>(g.row_tiles) * g.col_tiles * (g.most_splits > 0 ? g.most_splits : 1);
    MUON_REQUIRE(grid > 0 && grid <= 0xffffffffll / Cfg::NT, "linear_cross_entropy: %lld tiles", static_cast<long long>(grid));
    hipLaunchKernelGGL((head_gemm_kernel<Cfg, PRODUCT, TURN>), dim3(static_cast<unsigned>(grid)), dim3(Cfg::NT),
                       2 * most < Cfg::NHALF ? static_cast<size_t>(2 * most) * Cfg::HALF_BYTES : Cfg::LDS_BYTES, s, g);
    return check_launch("linear_cross_entropy");
}
template <typename Cfg, int PRODUCT>
static int launch_product(const HeadGemm& g, int64_t tokens, int64_t most, hipStream_t s) {
    if constexpr (PRODUCT == HEAD_STATS || PRODUCT == HEAD_GRAD)
        if (tokens <= Cfg::BT) return launch_product<Cfg, PRODUCT, true>(g, most, s);
    return launch_product<Cfg, PRODUCT, false>(g, most, s);
}
template <int PRODUCT>
static int launch_product(const HeadGemm& g, bool large, int64_t tokens, int64_t most, hipStream_t s) {
    return large ? launch_product<HeadLarge, PRODUCT>(g, tokens, most, s) : launch_product<HeadSmall, PRODUCT>(g, tokens, most, s);
}

template <typename Cfg, int PRODUCT, bool TURN = false>
static int raise_head_limit() {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(head_gemm_kernel<Cfg, PRODUCT, TURN>), hipFuncAttributeMaxDynamicSharedMemorySize,
                            static_cast<int>(Cfg::LDS_BYTES)) != hipSuccess) {
        (void)hipGetLastError();
        set_error("linear_cross_entropy: cannot raise dynamic LDS to %zu bytes", Cfg::LDS_BYTES);
        return MUON_AMD_ELAUNCH;
    }
    return MUON_AMD_OK;
}
template <typename Cfg>
static int raise_head_limits_of() {
    int rc = raise_head_limit<Cfg, HEAD_STATS>();
    if (rc == MUON_AMD_OK) rc = raise_head_limit<Cfg, HEAD_GRAD>();
    if (rc == MUON_AMD_OK) rc = raise_head_limit<Cfg, HEAD_DHIDDEN>();
    if (rc == MUON_AMD_OK) rc = raise_head_limit<Cfg, HEAD_DWEIGHT>();
    if (rc == MUON_AMD_OK) rc = raise_head_limit<Cfg, HEAD_STATS, true>();
    if (rc == MUON_AMD_OK) rc = raise_head_limit<Cfg, HEAD_GRAD, true>();
    return rc;
}
int raise_head_limits() {
    const int rc = raise_head_limits_of<HeadLarge>();
    return rc == MUON_AMD_OK ? raise_head_limits_of<HeadSmall>() : rc;
}

// The copies that the products read; W is then (w, ld).  Forward (no coefficients) numbers the tokens too.
static int gather(const MuonHeadLoss& a, const HeadPlan& p, char* ws, f32x4v* coef, const uint16_t** w, int64_t* ld, hipStream_t s) {
    const int64_t blocks = p.rows / 4 < 4096 ? p.rows / 4 : 4096;
    uint16_t* const rows = reinterpret_cast<uint16_t*>(ws + p.hidden);
    if (!coef && a.tokens <= HO_FEW) {
        hipLaunchKernelGGL(head_order_few_kernel, dim3(static_cast<unsigned>(p.rows / HO_WAVES)), dim3(HO_WAVES * 64), 0, s, a, rows, static_cast<int>(p.ld), p.rows);
    } else {
        if (!coef) {
            hipLaunchKernelGGL(head_order_kernel, dim3(1), dim3(HO_THREADS), 0, s, a);
            if (const int rc = check_launch("head_loss: order")) return rc;
        }
        hipLaunchKernelGGL(head_gather_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, rows, static_cast<int>(p.ld), coef,
                           reinterpret_cast<float*>(ws + p.scale), static_cast<int>(p.piece / BK), p.splits, p.dh_tile);
    }
    if (const int rc = check_launch("linear_cross_entropy: rows")) return rc;
    *w = static_cast<const uint16_t*>(a.weight);
    *ld = a.ld_weight;
    if (p.padded) {
        *w = reinterpret_cast<uint16_t*>(ws + p.weight);
        *ld = p.ld;
        hipLaunchKernelGGL(head_pad_kernel, dim3(4096), dim3(256), 0, s, static_cast<const uint16_t*>(a.weight), a.ld_weight, static_cast<int64_t>(a.vocab), a.width,
                           reinterpret_cast<uint16_t*>(ws + p.weight), static_cast<int>(p.ld));
        return check_launch("linear_cross_entropy: matrix");
    }
    return MUON_AMD_OK;
}

}  // namespace muon_amd

using namespace muon_amd;

extern "C" {

size_t muon_amd_sizeof_head_loss(void) { return sizeof(MuonHeadLoss); }

int64_t muon_amd_head_loss_workspace(const MuonHeadLoss* args, int backward) {
    if (!args || args->tokens <= 0 || args->vocab <= 0 || args->width <= 0) return 0;
    return head_plan(*args, backward != 0).bytes;
}

int muon_amd_head_loss(const MuonHeadLoss* args, void* stream) {
    if (const int rc = check_head(args, "head_loss")) return rc;
    const MuonHeadLoss a = *args;
    MUON_REQUIRE(a.losses && a.lse && a.counter, "head_loss: null output");
    const HeadPlan p = head_plan(a, false);
    MUON_REQUIRE(a.workspace_bytes >= p.bytes, "head_loss: a workspace of %lld bytes, %lld needed", static_cast<long long>(a.workspace_bytes), static_cast<long long>(p.bytes));
    if (const int rc = muon_amd_init()) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char* const ws = static_cast<char*>(a.workspace);
    f32x2_t* const stats = reinterpret_cast<f32x2_t*>(ws + p.stats);
    float* const logit = reinterpret_cast<float*>(ws + p.logit);
    const auto join = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((a.tokens + HJ_ROWS - 1) / HJ_ROWS)), dim3(HJ_THREADS), 0, s, a, stats, p.rows, p.col_tiles, logit,
                           reinterpret_cast<float*>(ws + p.left));
        return check_launch("head_loss: join");
    };
    if (p.few) {
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(p.col_tiles), dim3(HF_THREADS), 0, s, static_cast<const uint16_t*>(a.hidden), a.ld_hidden,
                               static_cast<const uint16_t*>(a.weight), a.ld_weight, static_cast<int>(a.tokens), a.width, a.vocab, a.targets, a.target_bits, stats, p.rows, logit, a.counter);
        };
        if (a.tokens <= 16) go(head_few_kernel<1>);
        else if (a.tokens <= 32) go(head_few_kernel<2>);
        else go(head_few_kernel<4>);
        if (const int rc = check_launch("head_loss: few")) return rc;
        return join(head_join_kernel<true>);
    } else {
        HeadGemm g{};
        if (const int rc = gather(a, p, ws, nullptr, &g.Q, &g.ldq, s)) return rc;
        g.P = reinterpret_cast<const uint16_t*>(ws + p.hidden);
        g.ldp = p.ld;
        g.end_p = (p.rows * p.ld - 8) * 2;
        g.end_q = ((a.vocab - 1) * g.ldq + p.ld - 8) * 2;
        g.count = a.order + a.tokens;
        g.row_tiles = static_cast<int>(p.rows / p.tile);
        g.col_tiles = p.col_tiles;
        g.kblocks = static_cast<int>(p.ld / BK);
        g.vocab = a.vocab;
        g.target = a.rows;
        g.stats = stats;
        g.ld_stats = p.rows;
        g.target_logit = logit;
        if (const int rc = launch_product<HEAD_STATS>(g, p.large, a.tokens, g.kblocks, s)) return rc;
    }
    return join(head_join_kernel<false>);
}

int muon_amd_head_loss_backward(const MuonHeadLoss* args, void* stream) {
    if (const int rc = check_head(args, "head_loss_backward")) return rc;
    const MuonHeadLoss a = *args;
    MUON_REQUIRE(a.dhidden || a.dweight, "head_loss_backward: no output");
    const HeadPlan p = head_plan(a, true);
    MUON_REQUIRE(a.workspace_bytes >= p.bytes, "head_loss_backward: a workspace of %lld bytes, %lld needed", static_cast<long long>(a.workspace_bytes),
                 static_cast<long long>(p.bytes));
    if (const int rc = muon_amd_init()) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char* const ws = static_cast<char*>(a.workspace);
    f32x4v* const coef = reinterpret_cast<f32x4v*>(ws + p.coef);
    const uint16_t* w;
    int64_t ldw;
    if (const int rc = gather(a, p, ws, coef, &w, &ldw, s)) return rc;
    uint16_t* const rows = reinterpret_cast<uint16_t*>(ws + p.hidden);
    uint16_t* const e = reinterpret_cast<uint16_t*>(ws + p.e);
    float* const part = reinterpret_cast<float*>(ws + p.part);
    const int32_t* const splits = reinterpret_cast<const int32_t*>(ws + p.scale) + 1;
    for (int i = 0; i < p.pieces; ++i) {
        const int begin = static_cast<int>(i * p.piece), size = static_cast<int>(a.vocab - begin < p.piece ? a.vocab - begin : p.piece);
        const uint16_t* const piece = w + begin * ldw;
        HeadGemm g{};
        g.count = a.order + a.tokens;
        // e of the piece
        const int tile = p.large ? 256 : 128;
        g.P = rows;
        g.ldp = p.ld;
        g.end_p = (p.rows * p.ld - 8) * 2;
        g.Q = piece;
        g.ldq = ldw;
        g.end_q = ((size - 1) * ldw + p.ld - 8) * 2;
        g.row_tiles = static_cast<int>(p.rows / tile);
        g.col_tiles = static_cast<int>(up(size, tile) / tile);
        g.cols = static_cast<int>(p.piece);
        g.kblocks = static_cast<int>(p.ld / BK);
        g.vocab_begin = begin;
        g.vocab = a.vocab;
        g.target = a.rows;
        g.coef = coef;
        g.out = e;
        g.ld_out = p.piece;
        if (const int rc = launch_product<HEAD_GRAD>(g, p.large, a.tokens, g.kblocks, s)) return rc;
        if (a.dhidden) {
            HeadGemm h{};
            h.count = g.count;
            h.P = e;
            h.ldp = p.piece;
            h.end_p = (p.rows * p.piece - 8) * 2;
            h.Q = piece;
            h.ldq = ldw;
            h.end_q = ((size - 1) * ldw + p.ld - 8) * 2;
            h.col_limit = static_cast<int>(p.ld);
            h.row_tiles = static_cast<int>(p.rows / p.dh_tile);
            h.col_tiles = static_cast<int>(up(p.ld, p.dh_tile) / p.dh_tile);
            h.splits = splits;
            h.most_splits = p.splits;
            h.cols = static_cast<int>(p.ld);
            h.kblocks = static_cast<int>(up(size, BK) / BK);
            h.part = part;
            h.add = i > 0;
            h.part_stride = p.rows * p.ld;
            h.ld_out = p.ld;
            if (const int rc = launch_product<HEAD_DHIDDEN>(h, p.dh_tile == 256, a.tokens, h.kblocks, s)) return rc;
        }
        if (a.dweight) {
            HeadGemm h{};
            h.count = g.count;
            h.P = e;
            h.ldp = p.piece;
            h.end_p = (p.rows * p.piece - 8) * 2;
            h.row_limit = static_cast<int>(p.piece);
            h.Q = rows;
            h.ldq = p.ld;
            h.end_q = (p.rows * p.ld - 8) * 2;
            h.col_limit = static_cast<int>(p.ld);
            h.rows = size;
            h.row_tiles = static_cast<int>(up(size, p.dw_tile) / p.dw_tile);
            h.col_tiles = static_cast<int>(up(a.width, p.dw_tile) / p.dw_tile);
            h.cols = a.width;
            h.scale = reinterpret_cast<const float*>(ws + p.scale);
            h.out = static_cast<uint16_t*>(a.dweight) + static_cast<int64_t>(begin) * a.width;
            h.ld_out = a.width;
            if (const int rc = launch_product<HEAD_DWEIGHT>(h, p.dw_tile == 256, a.tokens, up(a.tokens, BK) / BK, s)) return rc;
        }
    }
    if (a.dhidden) {
        const int64_t items = a.tokens * ((a.width + 511) / 512), blocks = items < 8192 ? items : 8192;
        hipLaunchKernelGGL(head_dhidden_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, a, part, p.rows * p.ld, static_cast<int>(p.ld),
                           reinterpret_cast<const float*>(ws + p.scale));
        return check_launch("head_loss_backward: hidden");
    }
    return MUON_AMD_OK;
}

}  // extern "C"
