// Operands whose columns do not start on 16-byte boundaries, which TMA cannot address, are copied with padded columns
// before a fused or ragged product: dst[g][c][r] = src[g * group + c * ld + r], columns of ld_dst (a multiple of 8)
// elements, zeros behind the rows.  A copy at the rate of HBM against feeding the tensor cores by bounds-checked loads
// of two warps: 1000 x 777 x 1111, B unaligned, 140 us without it.
// A warp takes 256 rows of a column; its lanes take 8 each, whose 16 source bytes lie in two granules: the second one is
// the next lane's first.
#pragma once
#include "any_load.cuh"
#include "fused_epilogue.cuh"
#include "ptx.cuh"

namespace gk {

constexpr int kAlignThreads = 256;

struct AlignParams {
  const uint16_t* src; uint16_t* dst;
  int64_t ld, group, ld_dst, group_dst;
  int32_t rows, cols;
  int32_t skip_empty;      // 1: groups without columns (FusedParams) are not copied: their product is not computed
  FusedParams f;
};

static __global__ void __launch_bounds__(kAlignThreads) align_operand_kernel(const AlignParams p) {
  __shared__ int live;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = static_cast<int>(blockIdx.y);
  if (p.skip_empty) {
    if (warp == 0) {
      int carry = fused_first_offset(p.f), lo = 0, hi = 0;
      for (int base = 0; base <= g; base += 32) fused_group_chunk(p.f, base, lane, carry, lo, hi);
      if (lane == (g & 31)) live = hi > lo;
    }
    __syncthreads();
    if (!live) return;
  }
  const uint16_t* src = p.src + g * p.group;
  const uint16_t* end = src + static_cast<int64_t>(p.cols - 1) * p.ld + p.rows;
  uint16_t* dst = p.dst + g * p.group_dst;
  const int pieces = static_cast<int>(p.ld_dst / 8), segments = (pieces + 31) / 32;
  const int64_t units = static_cast<int64_t>(segments) * p.cols, step = static_cast<int64_t>(gridDim.x) * (kAlignThreads / 32);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kAlignThreads / 32) + warp; u < units; u += step) {
    const int64_t c = u / segments;
    const uint16_t* col = src + c * p.ld;
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(col) & 15);
    const uint16_t* granules = reinterpret_cast<const uint16_t*>(reinterpret_cast<uintptr_t>(col) & ~static_cast<uintptr_t>(15));
    const int q = static_cast<int>(u - c * segments) * 32 + lane;
    const uint4 lo = any_granule(granules + 8 * q, src, end);
    uint4 hi;
    hi.x = __shfl_down_sync(0xffffffffu, lo.x, 1); hi.y = __shfl_down_sync(0xffffffffu, lo.y, 1);
    hi.z = __shfl_down_sync(0xffffffffu, lo.z, 1); hi.w = __shfl_down_sync(0xffffffffu, lo.w, 1);
    if (lane == 31) hi = any_granule(granules + 8 * q + 8, src, end);
    if (q < pieces)
      *reinterpret_cast<uint4*>(dst + c * p.ld_dst + 8 * q) = any_keep(any_shift(lo, hi, shift), min(8, p.rows - 8 * q));
  }
}

}  // namespace gk
