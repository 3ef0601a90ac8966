// Tile images and fragment accesses of the 32-rows-per-wave attention kernels (attn32.hip, packed_attn.hip): a [64 rows][64 bf16] LDS tile
// is 64 rows of eight 16-byte chunks, chunk c of row r at position c ^ ((r >> 1) & 7).  Internal to those files (anonymous namespace on purpose).
#pragma once
#include "e2k_device.h"
#include <e2k_asm.h>

namespace {

using namespace e2k;

// LDS row of a K-type tile that holds tile row R (and back: an involution): bits 2 and 3 trade places
__device__ __forceinline__ int swap23(int r) { return (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1); }
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

// the upper half-wave's x and the lower half-wave's y trade places (two dwords each)
__device__ __forceinline__ void swap_pair(u32x2& x, u32x2& y) {
    unsigned x0 = x[0], x1 = x[1], y0 = y[0], y1 = y[1];
    lane32_swap(x0, y0);
    lane32_swap(x1, y1);
    x = u32x2{x0, x1};
    y = u32x2{y0, y1};
}
__device__ __forceinline__ bf16x8 pack8f(const float* f) { return __builtin_bit_cast(bf16x8, pack8(f)); }

// the 16 x 4 fragment-read offsets of a lane inside a [64][64] tile: chunk 2 j + hi of row l31 (+ 32 per row block, added as an
// immediate)
__device__ __forceinline__ void frag_offsets(int l31, int hi, int (&off)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) off[j] = l31 * 128 + (((2 * j + hi) ^ swz(l31)) << 4);
}

// row-per-lane epilogue: acc[db][r] = column (32 db + (r & 3) + 8 (r >> 2) + 4 hi) of this lane's row, scaled and stored as bf16 in
// 16-byte pieces: the two half-waves exchange their 8-byte pieces (v_permlane32_swap), lower half stores columns 16 g .. + 7, upper half
// 16 g + 8 .. + 15 of every group of 16 columns
template <class F>
__device__ __forceinline__ void store_rows32(const f32x16 (&acc)[2], int hi, bool ok, F&& put) {
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            float a[4] = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
            float b[4] = {acc[db][4 * g + 4], acc[db][4 * g + 5], acc[db][4 * g + 6], acc[db][4 * g + 7]};
            put(db, g, hi, ok, a, b);
        }
}

// Transposing fragment reads (ds_read_b64_tr_b16) out of a K-type tile image: the A operand of an MFMA whose rows are the tile's 64
// COLUMNS (dh) and whose reduction slots are tile rows.  Lane l = (i = l & 31, hi): row block db gives MFMA row i = column 32 db + i;
// its eight slots 8 hi .. 8 hi + 7 of slab (kb, s2) are the tile rows 32 kb + 16 s2 + 8 hi + e, which sit at LDS rows
// 32 kb + 16 s2 + 4 hi + (e & 3) + 8 (e >> 2) (swap23).  One instruction serves a 16-lane group: lane (q16 = l & 15) passes the
// address of 4 consecutive columns 4 (q16 & 3) .. of LDS row (q16 >> 2) of the group's [4 rows][16 columns] block and receives
// column q16 of the four rows.  The group of lanes 16 .. 31 (and 48 .. 63) covers columns 16 .. 31 of the row block.
struct TrOff { int lo[2], hi_[2]; };      // [db]: byte offsets (inside the tile) of the reads for e = 0..3 and e = 4..7, slab (0, 0)
__device__ __forceinline__ TrOff tr_offsets(int lane) {
    const int q16 = lane & 15, cg = (lane >> 4) & 1, hi = lane >> 5;
    TrOff t;
#pragma unroll
    for (int db = 0; db < 2; ++db) {
        const int col = 32 * db + 16 * cg + 4 * (q16 & 3);           // first of the 4 columns this lane addresses
#pragma unroll
        for (int eh = 0; eh < 2; ++eh) {
            const int row = 4 * hi + (q16 >> 2) + 8 * eh;
            const int off = row * 128 + ((((col >> 3)) ^ swz(row)) << 4) + (col & 7) * 2;
            (eh ? t.hi_ : t.lo)[db] = off;
        }
    }
    return t;
}
// rows + 16 s2 + 32 kb: swz(row + 16 s2 + 32 kb) = swz(row) ^ ... only when 16 s2 >> 1 = 8 s2 leaves (row >> 1) & 7 alone: it does (8, 16 = 0 mod 8)
__device__ __forceinline__ bf16x8 tr_frag(const unsigned char* T, const TrOff& t, int db, int imm) {
    s16x4_ a, b;
    lds_tr_issue(a, T + t.lo[db], imm);
    lds_tr_issue(b, T + t.hi_[db], imm);
    lds_tr_wait(a, b);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// keeps a rarely taken, wave-uniform branch a branch (left alone the compiler turns its selects into unconditional ones on the hot path)
__device__ __forceinline__ void cold_path() { asm volatile("" ::: "memory"); }


}  // namespace
