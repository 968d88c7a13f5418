// Eight consecutive 16-bit elements from any address, by 16-byte loads.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gk {

// The 16-byte granule at `g` (16-byte aligned) of an array [first, last): whole if it lies inside, else the elements
// that do (nothing outside the array is read).
__device__ __forceinline__ uint4 any_granule(const uint16_t* g, const uint16_t* first, const uint16_t* last) {
  if (g >= first && g + 8 <= last) return *reinterpret_cast<const uint4*>(g);
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = (g + i >= first && g + i < last) ? g[i] : 0u;
  return make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
}

// 16 bytes starting `shift` bytes (even, below 16) into the 32 bytes of lo and hi.
__device__ __forceinline__ uint4 any_shift(const uint4& lo, const uint4& hi, int shift) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (shift & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (shift & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int bits = (shift & 2) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}

// Elements p .. p + 7 of the array [first, last); what lies outside reads as zero.
__device__ __forceinline__ uint4 any_load_8(const uint16_t* p, const uint16_t* first, const uint16_t* last) {
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
  const uint16_t* g = reinterpret_cast<const uint16_t*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15));
  const uint4 lo = any_granule(g, first, last);
  if (shift == 0) return lo;
  return any_shift(lo, any_granule(g + 8, first, last), shift);
}

// The first n (0 .. 8) of eight elements, zeros behind them.
__device__ __forceinline__ uint4 any_keep(uint4 v, int n) {
  auto word = [n](uint32_t w, int i) { return n >= 2 * i + 2 ? w : (n == 2 * i + 1 ? w & 0xffffu : 0u); };
  return make_uint4(word(v.x, 0), word(v.y, 1), word(v.z, 2), word(v.w, 3));
}

}  // namespace gk
