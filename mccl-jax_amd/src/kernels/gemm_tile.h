// Operand tiles of the tiled matrix products (gemm_tiled.hip, linear_xent.hip)
// in LDS: where a 16-byte chunk of a tile lies, and how a lane reads its MFMA
// operand.  gemm_tiled.hip's header has the reasons for both placements.
#pragma once

#include "attn_common.h"

namespace mk {

// chunk placement of a k-contiguous LDS row (BK / 8 chunks): the 16 rows one
// ds_read_b128 cycle reads at one chunk land on 16 different 16-byte bank
// groups (rows 2 (64 B) or 4 (32 B) apart share the row's bank offset)
template <int BK>
__device__ inline int kc_swizzle(int row) {
  return BK == 64 ? ((row >> 1) & 7) : ((row >> 2) & 3);
}

// chunk placement of an m- / n-contiguous LDS k-row (R / 8 chunks): the 4
// k-rows x 4 chunks of one ds_read_b64_tr_b16 half-wave land on 16 different
// bank groups; the XOR keeps each chunk inside its aligned group of 8 (R =
// 192) or 16 chunks
template <int R>
__device__ inline int nc_swizzle(int kr) {
  static_assert(R % 64 == 0, "k-row of whole 8-chunk groups");
  return R % 128 == 0 ? 4 * (kr & 3) : 4 * ((kr >> 1) & 1);
}

// MFMA operand (8 values of 16 bits) for rows rb .. rb + 31 of a tile of R rows
// and k-step ks (k = 16 ks .. 16 ks + 15): lane (c, g) gets row rb + c, k 16 ks
// + 8 g ..+7.
template <bool KC, int R, int BK>
__device__ inline u32x4_t read_operand16(const uint16_t* t, int rb, int ks, int lane) {
  if constexpr (KC) {
    const int row = rb + (lane & 31), ch = (2 * ks + (lane >> 5)) ^ kc_swizzle<BK>(row);
    return *reinterpret_cast<const u32x4_t*>(t + row * BK + 8 * ch);
  } else {
    // 16-lane group: lanes 4q .. 4q + 3 address k-row q of a 4 x 16 block,
    // 8 bytes (4 columns) each; lane i of the group receives column i.
    const int kr = 16 * ks + 8 * (lane >> 5) + ((lane & 15) >> 2);
    const int col = rb + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int at = 8 * ((col >> 3) ^ nc_swizzle<R>(kr)) + (col & 7);
    const uint2 lo = attn::lds_read_tr(t + kr * R + at);
    const uint2 hi = attn::lds_read_tr(t + (kr + 4) * R + at);  // k-row kr + 4 has kr's swizzle
    return u32x4_t{lo.x, lo.y, hi.x, hi.y};
  }
}

// s_waitcnt vmcnt(n) for a compile-time n, expcnt / lgkmcnt untouched
template <int N>
__device__ inline void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// Kernel shape: workgroup tile, wave grid, k-tile depth, LDS stages.
template <int TM_, int TN_, int WGM_, int WGN_, int BK_, int S_>
struct Shape {
  static constexpr int TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, BK = BK_, S = S_;
};

}  // namespace mk
