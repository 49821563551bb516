// Pieces of the windowed attention's tile kernels: LDS tiles of head rows and their MFMA fragments.
#pragma once

#include "gemm16.hpp"

namespace vkh {

// B-operand fragment from two accumulator tiles (contraction rows 0-15 of
// tile a, 16-31 of tile b).
VKH_DEV bf16x8 frag_acc(const f32x4 &a, const f32x4 &b) {
    return cvt8(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]);
}

VKH_DEV bf16x8 ld_frag(const bf16 *p) { return *reinterpret_cast<const bf16x8 *>(p); }

// Maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that hold one row of a
// transposed score tile: the swaps give every lane both halves' values.
// (The compiler's builtin returned one register for both results here, so the two
// instructions are written out, with the two wait states they need after a VALU write.)
template <int L>
VKH_DEV void lane_halves(float v, float &a, float &b) {
    a = b = v;
    if constexpr (L == 32) asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    else asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
VKH_DEV float xrow_max(float v) {
    float a, b;
    lane_halves<32>(v, a, b);
    lane_halves<16>(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
VKH_DEV float xrow_sum(float v) {
    float a, b;
    lane_halves<16>(v, a, b);
    lane_halves<32>(a + b, a, b);
    return a + b;
}

template <int N>
VKH_DEV void wait_vm() {
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4 << 14));
}

// LDS tiles of bf16 head rows of HD values, as the DMA writes them: 16-byte chunk c of row r at
// chunk c ^ swz(r), so the 16 rows of a fragment read (frag_row) land in 16 different chunk columns of
// LDS's 256 bytes a cycle (rows of 128 bytes: two of them side by side).  A transposing read (tr4) takes
// two neighbouring chunks of each row, which rows r and r ^ 1 hold in the same two columns: half of the
// banks twice, two cycles more a read (a quarter to a third of the cycles that the kernels' LDS is active).
template <int HD>
struct TileRows {
    static_assert(HD == 64 || HD == 128, "head width");
    static VKH_DEV int swz(int r) { return HD == 128 ? r & 15 : (r >> 1) & 7; }
    // byte offset of (row r, element col)
    static VKH_DEV int toff(int r, int col) { return r * (HD * 2) + (((col >> 3) ^ swz(r)) << 4) + (col & 7) * 2; }
    // A or B operand: row r, values col .. col + 7
    static VKH_DEV bf16x8 frag_row(const char *tile, int r, int col) {
        return *reinterpret_cast<const bf16x8 *>(tile + toff(r, col));
    }
    // X[r0 + j][c0 + (lane % 16)], j = 0..3
    static VKH_DEV bf16x4 tr4(const char *tile, int r0, int c0, int l16) {
        const char *src = tile + toff(r0 + l16 / 4, c0 + 4 * (l16 % 4));
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4_t *)src);
    }
    // A operand whose rows are tile columns c0 + lane % 16 and whose contraction runs over the tile
    // rows k0 + {4g..4g+3, 16+4g..16+4g+3} (frag_acc's order)
    static VKH_DEV bf16x8 frag_t(const char *tile, int c0, int k0, int g, int l16) {
        const bf16x4 lo = tr4(tile, k0 + 4 * g, c0, l16);
        const bf16x4 hi = tr4(tile, k0 + 16 + 4 * g, c0, l16);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

}  // namespace vkh
