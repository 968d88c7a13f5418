// dZ = dD * act'(Z) and the bias gradient db[:, g] = sum over the columns of group g of dZ.
//
// Bytes: dD and Z are read once, dZ is written once; the sums are FP32 of the unrounded products and are made in a
// fixed order.  A CTA owns 64 rows of one strip of at most `strip` columns of one group: its 32 column slots of
// 8 lanes x 16 bytes (VEC elements per access) walk the strip, and the slots' sums meet in shared memory.  With one
// strip per group the CTA writes db; else it writes a row of `partial` and bias_gradient_sum_kernel adds the strips of
// each group in order.
#pragma once
#include "fused_epilogue.cuh"
#include "ptx.cuh"

namespace gk {

constexpr int kActGradThreads = 256;
constexpr int kActGradRows = 64;

struct ActGradParams {
  const void* dD; const void* Z; void* dZ;     // Z NULL: act' = 1; dZ NULL: only the sums are wanted
  float* db;                                   // NULL: no sums
  float* partial;                              // strips x M sums, NULL: one strip per group, straight to db
  int32_t M, act;
  int64_t ldd, ldz, lddz, lddb;
  int32_t strip;                               // columns per strip
  int32_t per_group;                           // 1: blockIdx.y is the group and the CTA walks all of its columns
  FusedParams f;                               // groups
};

template <typename T, int VEC> struct ActGradVec;
template <> struct ActGradVec<__half, 8> { using type = uint4; };
template <> struct ActGradVec<__nv_bfloat16, 8> { using type = uint4; };
template <> struct ActGradVec<float, 4> { using type = uint4; };
template <> struct ActGradVec<__half, 1> { using type = uint16_t; };
template <> struct ActGradVec<__nv_bfloat16, 1> { using type = uint16_t; };
template <> struct ActGradVec<float, 1> { using type = uint32_t; };

__device__ __forceinline__ float actgrad_float(float x) { return x; }
__device__ __forceinline__ float actgrad_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float actgrad_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T actgrad_round(float x);
template <> __device__ __forceinline__ float actgrad_round<float>(float x) { return x; }
template <> __device__ __forceinline__ __half actgrad_round<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 actgrad_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kActGradThreads, 3) activation_gradient_kernel(const ActGradParams p) {
  constexpr int kLanes = kActGradRows / VEC;              // threads along the rows
  constexpr int kSlots = kActGradThreads / kLanes;        // columns in flight
  using V = typename ActGradVec<T, VEC>::type;
  __shared__ float sums[kSlots][kActGradRows + 1];
  __shared__ int item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    int g, c0, n;
    if (p.per_group) {
      // this block's group, with all of its columns
      int carry = fused_first_offset(p.f), lo = 0, hi = 0;
      g = static_cast<int>(blockIdx.y);
      for (int base = 0; base <= g; base += 32) fused_group_chunk(p.f, base, lane, carry, lo, hi);
      c0 = __shfl_sync(0xffffffffu, lo, g & 31);
      n = __shfl_sync(0xffffffffu, hi, g & 31) - c0;
    } else {
      fused_find_item(p.f, blockIdx.y, p.strip, lane, g, c0, n);
    }
    if (lane == 0) { item[0] = g; item[1] = c0; item[2] = n; }
  }
  __syncthreads();
  const int g = item[0], c0 = item[1], n = item[2];
  if (n == 0 && !p.per_group) return;                     // the list of strips is shorter than the grid
  const int r = static_cast<int>(threadIdx.x) % kLanes, slot = static_cast<int>(threadIdx.x) / kLanes;
  const int row = static_cast<int>(blockIdx.x) * kActGradRows + r * VEC;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
  if (row < p.M) {                                        // VEC > 1: M is a multiple of it
    const T* dd = static_cast<const T*>(p.dD) + row + static_cast<int64_t>(c0) * p.ldd;
    const T* z = static_cast<const T*>(p.Z) + row + static_cast<int64_t>(c0) * p.ldz;
    T* dz = static_cast<T*>(p.dZ) + row + static_cast<int64_t>(c0) * p.lddz;
    // The loads of the next U columns are in flight while these are computed (8192 x 16384, GELU, on one machine: 163 us without, 148 with).
    constexpr int U = 2;
    V dv[U], zv[U], dn[U], zn[U];
    auto load = [&](int c, V (&d)[U], V (&w)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u * kSlots;
        if (col < n) {
          d[u] = *reinterpret_cast<const V*>(dd + col * p.ldd);
          if (ACT != FUSED_ACT_NONE) w[u] = *reinterpret_cast<const V*>(z + col * p.ldz);
        }
      }
    };
    load(slot, dn, zn);
    for (int c = slot; c < n; c += U * kSlots) {
#pragma unroll
      for (int u = 0; u < U; ++u) { dv[u] = dn[u]; zv[u] = zn[u]; }
      load(c + U * kSlots, dn, zn);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u * kSlots;
        if (col < n) {
          T* de = reinterpret_cast<T*>(&dv[u]);
          const T* ze = reinterpret_cast<const T*>(&zv[u]);
          if constexpr (VEC > 1) {                              // two elements at a time (fused_epilogue.cuh)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
              float2 v = make_float2(actgrad_float(de[i]), actgrad_float(de[i + 1]));
              if (ACT != FUSED_ACT_NONE)
                v = __fmul2_rn(v, fused_act_gradient2<ACT, sizeof(T) == 4>(make_float2(actgrad_float(ze[i]), actgrad_float(ze[i + 1]))));
              acc[i] += v.x; acc[i + 1] += v.y;
              de[i] = actgrad_round<T>(v.x); de[i + 1] = actgrad_round<T>(v.y);
            }
          } else {
            float v = actgrad_float(de[0]);
            if (ACT == FUSED_ACT_GELU) v = __fmul_rn(v, fused_gelu_gradient2<sizeof(T) == 4>(fused_2(actgrad_float(ze[0]))).x);
            else if (ACT != FUSED_ACT_NONE) v = __fmul_rn(v, fused_act_gradient(actgrad_float(ze[0]), ACT));
            acc[0] = __fadd_rn(acc[0], v);      // never contracted: the same sums whether dZ is stored or not
            de[0] = actgrad_round<T>(v);
          }
          if (p.dZ != nullptr) *reinterpret_cast<V*>(dz + col * p.lddz) = dv[u];
        }
      }
    }
  }
  if (p.db == nullptr) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[slot][r * VEC + i] = acc[i];
  __syncthreads();
  for (int half = kSlots / 2; half >= 4; half >>= 1) {     // pairwise: the order is fixed
    for (int i = threadIdx.x; i < half * kActGradRows; i += kActGradThreads)
      sums[i / kActGradRows][i % kActGradRows] += sums[i / kActGradRows + half][i % kActGradRows];
    __syncthreads();
  }
  if (threadIdx.x < kActGradRows) {
    const int m = static_cast<int>(blockIdx.x) * kActGradRows + threadIdx.x;
    const float s = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
    if (m < p.M) {
      if (p.partial) p.partial[static_cast<int64_t>(blockIdx.y) * p.M + m] = s;
      else p.db[m + g * p.lddb] = s;
    }
  }
}

// db[:, g] = the sum of group g's strips, in order (zero for a group without columns).
static __global__ void __launch_bounds__(kActGradThreads) bias_gradient_sum_kernel(const ActGradParams p) {
  __shared__ int item[2];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, g = static_cast<int>(blockIdx.y);
  if (threadIdx.x < 32) {
    int carry = fused_first_offset(p.f), before = 0, first = 0, count = 0;
    for (int base = 0; base <= g; base += 32) {
      int lo, hi;
      fused_group_chunk(p.f, base, lane, carry, lo, hi);
      const int items = (hi - lo + p.strip - 1) / p.strip;
      const int incl = fused_warp_scan(items, lane);
      first = before + __shfl_sync(0xffffffffu, incl - items, g & 31);
      count = __shfl_sync(0xffffffffu, items, g & 31);
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) { item[0] = first; item[1] = count; }
  }
  __syncthreads();
  const int m = static_cast<int>(blockIdx.x) * kActGradThreads + threadIdx.x;
  if (m >= p.M) return;
  const float* src = p.partial + static_cast<int64_t>(item[0]) * p.M + m;
  float s = 0.0f;
#pragma unroll 8
  for (int i = 0; i < item[1]; ++i) s += src[static_cast<int64_t>(i) * p.M];
  p.db[m + g * p.lddb] = s;
}

}  // namespace gk
