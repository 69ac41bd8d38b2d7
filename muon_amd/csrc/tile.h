// What the matrix kernels are made of: operand tiles streamed into LDS, fragments read from it, result strips written.
#pragma once

#include "common.h"

namespace muon_amd {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int BK = 64;   // k extent of one ring stage (128 bytes per LDS row)
constexpr int ROW_BYTES = BK * 2;

// One wave-wide 16-byte-per-lane load from global memory straight into LDS at
// lds_addr + lane*16 (lds_addr wave-uniform): buffer_load_dwordx4 ... lds, the operand addressed as
// resource (base pointer) + per-lane byte offset + wave-uniform byte offset.  Issued through inline
// assembly so that the compiler's wait-count insertion does not serialise the ring; completion is
// awaited explicitly with s_waitcnt vmcnt(n) before the workgroup barrier that publishes a stage.
// The buffer form keeps the per-lane address in one register and the k-block offset in a scalar one
// (global_load_lds_dwordx4 needs a 64-bit address per lane): measured 1.3 % faster on the 256 x 256
// class, equal on the 128 x 128 class.
// rsrc: {base[31:0], base[47:32] (stride 0), number of bytes addressable, format word}.
__device__ __forceinline__ u32x4 dma_resource(const void* base) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32) & 0xffffu, 0xffffffffu, 0x00020000u};
}
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds\n"
                 :: "v"(voff), "s"(rsrc), "s"(soff), "s"(lds_addr) : "memory", "m0");
}
// s_waitcnt vmcnt(n) only (expcnt / lgkmcnt left unconstrained); n < 64 (bits 3:0 and 15:14).
#define NS_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt(0x0F70 | ((n) & 15) | (((n) >> 4) << 14))

// Fragment reads of the main loop: N ds_read_b128 from LDS byte address addr + i * 32 rows, issued
// through inline assembly so that the waits for them can be placed by hand (wait_frags).
template <int N, int I = 0>
struct FragLoad {
    static __device__ __forceinline__ void run(u32x4 (&f)[N], uint32_t addr) {
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f[I]) : "v"(addr), "n"(I * 32 * ROW_BYTES));
        if constexpr (I + 1 < N) FragLoad<N, I + 1>::run(f, addr);
    }
};
// The same for an operand that lies k-major in LDS (row = k, the tile's columns along the row: X
// itself as the second operand of B X): ds_read_b64_tr_b16 takes, in every group of 16 lanes, from
// lane 4r + c the address of columns 4c .. 4c+3 of row r of a 4 x 16 block and hands lane j the four
// rows of column j.  With lanes 0..15 / 16..31 on columns 0..15 / 16..31 of rows 0..3 and lanes 32..63
// on rows 8..11, two such reads (rows +0 and +4) leave lane l with k = 8 (l / 32) .. + 7 of column
// l % 32: exactly the second operand of v_mfma_f32_32x32x16_bf16 (checked on the device).
// f[2 i], f[2 i + 1]: the two halves of fragment i; addr[i]: its per-lane LDS byte address (the
// column blocks of a row are XOR-swizzled with row & 3, so it depends on i).
template <int N, int ROWQ, int I = 0>
struct FragLoadTr {
    static __device__ __forceinline__ void run(u32x2 (&f)[2 * N], const uint32_t (&addr)[N], uint32_t base) {
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:0" : "=v"(f[2 * I]) : "v"(addr[I] + base));
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f[2 * I + 1]) : "v"(addr[I] + base), "n"(4 * ROWQ));
        if constexpr (I + 1 < N) FragLoadTr<N, ROWQ, I + 1>::run(f, addr, base);
    }
};

// s_waitcnt lgkmcnt(CNT), tied to the fragment registers the following MFMAs read: the compiler
// sees them redefined here and cannot move a use above the wait.
template <int CNT, int TM, int TN>
__device__ __forceinline__ void wait_frags(u32x4 (&a)[TM], u32x4 (&b)[TN]) {
    static_assert(CNT >= 0 && CNT < 16, "lgkmcnt is a 4-bit counter");
    if constexpr (TM == 4 && TN == 2)
        asm volatile("s_waitcnt lgkmcnt(%6)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(b[0]), "+v"(b[1]) : "n"(CNT));
    else if constexpr (TM == 2 && TN == 2)
        asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(a[0]), "+v"(a[1]), "+v"(b[0]), "+v"(b[1]) : "n"(CNT));
    else if constexpr (TM == 1 && TN == 1)
        asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(a[0]), "+v"(b[0]) : "n"(CNT));
    else
        static_assert(TM == 2 && TN == 2, "wait_frags: add the operand list of this wave tile");
}
template <int CNT, int TM, int TN2>
__device__ __forceinline__ void wait_frags_tr(u32x4 (&a)[TM], u32x2 (&b)[TN2]) {
    static_assert(CNT >= 0 && CNT < 16, "lgkmcnt is a 4-bit counter");
    if constexpr (TM == 4 && TN2 == 4)
        asm volatile("s_waitcnt lgkmcnt(%8)" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(b[0]), "+v"(b[1]),
                     "+v"(b[2]), "+v"(b[3]) : "n"(CNT));
    else if constexpr (TM == 2 && TN2 == 4)
        asm volatile("s_waitcnt lgkmcnt(%6)" : "+v"(a[0]), "+v"(a[1]), "+v"(b[0]), "+v"(b[1]), "+v"(b[2]), "+v"(b[3]) : "n"(CNT));
    else if constexpr (TM == 1 && TN2 == 2)
        asm volatile("s_waitcnt lgkmcnt(%3)" : "+v"(a[0]), "+v"(b[0]), "+v"(b[1]) : "n"(CNT));
    else
        static_assert(TM == 2 && TN2 == 4, "wait_frags_tr: add the operand list of this wave tile");
}

// Result strips go through wave-private LDS, 32 rows of WN bf16 columns at a time, as 16-byte chunks;
// chunk c of row r sits at position c ^ f(r).  f spreads both the 16-byte accesses of 8 consecutive
// rows and the transposing reads of 4 rows x 16 columns over all banks.
template <int WN>
__device__ __forceinline__ uint32_t strip_pos(int r, int c) {
    static_assert(WN == 64 || WN == 32, "strip_pos: rows of 8 or 4 chunks");
    const int f = WN == 64 ? (((r & 3) << 1) | ((r >> 2) & 1)) : ((r & 2) | ((r >> 2) & 1));
    return static_cast<uint32_t>(r * WN * 2 + ((c ^ f) << 4));
}

// One 32 x 32 tile of packed bf16 pairs (lane = row l % 32, pair 2q + i = columns 8q + 4 (l / 32) + 2i) into
// columns 32b .. of the strip: the halves of two neighbouring 8-column chunks are exchanged between
// lanes l and l + 32, so that every lane holds 8 consecutive columns and writes them at once.
template <int WN>
__device__ __forceinline__ void strip_write(char* stage, int lr, int g, int b, const uint32_t (&po)[8]) {
#pragma unroll
    for (int q = 0; q < 4; q += 2) {
        const auto x = __builtin_amdgcn_permlane32_swap(po[2 * q], po[2 * q + 2], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(po[2 * q + 1], po[2 * q + 3], false, false);
        *reinterpret_cast<u32x4*>(stage + strip_pos<WN>(lr, b * 4 + q + g)) = u32x4{x[0], y[0], x[1], y[1]};
    }
}

}  // namespace muon_amd
