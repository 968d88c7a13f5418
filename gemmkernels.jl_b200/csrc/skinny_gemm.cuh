// Products with a few columns (a few tokens): D[:, J] = epilogue(op(A_g) B[:, J]) for at most NT columns at a time.
//
// With one to a few columns every weight is used that often and no more: the product is a stream of A at the rate of
// HBM, 2 * NT flop per 2 bytes, far below what the FP32 FMA pipe does (NT = 4: 13 TFMA/s at 6.6 TB/s of 36).  The
// tensor-core kernel reaches its first MMA only after barrier, TMEM and first-copy latencies that are as long as
// the whole stream of a 4096 x 4096 layer (5.1 us at 6.57 TB/s), so plain 16-byte loads feed FMAs directly.
//
// A cluster of S CTAs owns 64 rows of D; its CTA r takes the r-th run of K, so that a layer with few rows still has
// loads in flight on every SM (S is chosen on the host: one round of resident CTAs).  The CTAs' partial sums meet in
// distributed shared memory, where each CTA adds one slice of the 64 x NT outputs in the order of the ranks (the
// result does not depend on timing) and applies the epilogue.
//   K_MAJOR  (A stored with consecutive k): a warp owns 8 rows, its lanes 8 consecutive k each
//   M_MAJOR  (A stored with consecutive rows): 8 lanes own 8 rows each; the other 32 slots of the CTA (4 per warp)
//            take 8 consecutive k each
// Either way a thread has eight 16-byte loads of A in flight and 8 x NT accumulators.
//
// ANY drops the conditions of the plain form (K, and for M_MAJOR also M, a multiple of 8; every address 16-byte aligned; B
// with consecutive k): eight elements are cut from two 16-byte granules, what lies behind K is zeroed.
#pragma once
#include "any_load.cuh"
#include "fused_epilogue.cuh"
#include "ptx.cuh"

namespace gk {

constexpr int kSkinnyThreads = 256;
constexpr int kSkinnyRows = 64;        // rows of D per cluster
constexpr int kSkinnyStep = 256;       // K consumed per step of a CTA (K runs are multiples of it)
// CTAs per SM, which the registers are limited to: the loads in flight are what hides the latency of HBM (4096 x 4096,
// one column: 12.3 us with two, 8.3 us with four).
__host__ __device__ constexpr int skinny_ctas(int nt, bool any) { return any ? 2 : (nt == 1 ? 4 : (nt == 2 ? 3 : 2)); }

struct SkinnyParams {
  const void* A; const void* B; const void* C; void* D;
  int32_t M, K;
  int64_t lda, b_sk, b_sn, ldc, ldd;   // B(k, n) at k * b_sk + n * b_sn
  int64_t a_group;             // elements between the groups' A
  float alpha, beta;
  const float* bias;
  int32_t bias_axis, act;      // 0 none, 1 per row, 2 per column
  int32_t dtype_d;             // of C, D and Z: 0 F16, 1 BF16, 2 F32
  int32_t k_per_rank;          // K run of a CTA, a multiple of kSkinnyStep
  FusedParams f;
};

__device__ __forceinline__ uint4 skinny_load_stream(const void* p) {   // weights: used once, not kept in L1
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <typename T> __device__ __forceinline__ void skinny_unpack(const uint4& v, float (&f)[8]);
template <> __device__ __forceinline__ void skinny_unpack<__nv_bfloat16>(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void skinny_unpack<__half>(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ float skinny_load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Sums v over the lanes that differ in bits `kFrom` .. `kTo` (powers of two, kFrom > kTo), halving the number of
// values a lane holds at every step while there are several; returns the index of the lane's first value.
template <int V, int kFrom, int kTo>
__device__ __forceinline__ int skinny_reduce(float (&v)[V], int lane) {
  int n = V, first = 0;
#pragma unroll
  for (int o = kFrom; o >= kTo; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if (i < n) {
          const float send = up ? v[i] : v[i + n];
          const float keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
      if (up) first += n;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return first;
}

// The end of both kernels: the cluster's sums ([column][row], n columns) are added in rank order, each CTA taking a
// slice of the outputs, and the epilogue is applied.
__device__ __forceinline__ void skinny_finish(const SkinnyParams& p, const float* sum, int g, int c0, int n, int row0, uint32_t ranks, uint32_t rank) {
  __syncthreads();
  if (ranks > 1) cluster_sync_all();
  const int outputs = n * kSkinnyRows, mine = (outputs + static_cast<int>(ranks) - 1) / static_cast<int>(ranks);
  const int first = static_cast<int>(rank) * mine, last = min(first + mine, outputs);
  const uint32_t sum_addr = smem_u32(sum);
  for (int o = first + static_cast<int>(threadIdx.x); o < last; o += kSkinnyThreads) {
    float s = 0.0f;
    for (uint32_t r = 0; r < ranks; ++r) s += skinny_load_cluster(map_to_cta(sum_addr + 4u * o, r));
    const int m = row0 + o % kSkinnyRows;
    if (m >= p.M) continue;
    const int64_t col = c0 + o / kSkinnyRows;
    const float bias = p.bias_axis == 1 ? p.bias[m + g * p.f.bias_group] : (p.bias_axis == 2 ? p.bias[col] : 0.0f);
    fused_put(p.D, m + col * p.ldd, p.dtype_d,
              fused_finish(p.f, fmaf(p.alpha, s, bias), p.beta, p.C, m + col * p.ldc, p.dtype_d, p.act, m, col));
  }
  if (ranks > 1) cluster_sync_all();     // the peers have read this CTA's sums
}

template <typename T> struct SkinnyIsHalf { static constexpr bool value = false; };
template <> struct SkinnyIsHalf<__half> { static constexpr bool value = true; };

template <typename T, bool K_MAJOR, int NT, bool ANY>
__global__ void __launch_bounds__(kSkinnyThreads, skinny_ctas(NT, ANY)) skinny_gemm_kernel(const SkinnyParams p) {
  constexpr int kOut = kSkinnyRows * NT;
  __shared__ float part[K_MAJOR ? 1 : 8][kOut];   // M_MAJOR: sums of each warp
  __shared__ float sum[kOut];                     // sums of this CTA's K run, [column][row]
  __shared__ int item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const uint32_t rank = cluster_cta_rank();
  const int row0 = static_cast<int>(blockIdx.x / ranks) * kSkinnyRows;

  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    int g, c0, n;
    fused_find_item(p.f, blockIdx.y, NT, lane, g, c0, n);
    if (lane == 0) { item[0] = g; item[1] = c0; item[2] = n; }
  }
  __syncthreads();
  const int g = item[0], c0 = item[1], n = item[2];
  if (n == 0) return;    // the list is shorter than the grid; the same for every CTA of the cluster

  const T* A = static_cast<const T*>(p.A) + g * p.a_group;
  const T* B = static_cast<const T*>(p.B) + c0 * p.b_sn;
  // ANY: where this group's A and the columns of B end
  const uint16_t* a_first = reinterpret_cast<const uint16_t*>(A);
  const uint16_t* a_last = a_first + (K_MAJOR ? static_cast<int64_t>(p.M - 1) * p.lda + p.K : static_cast<int64_t>(p.K - 1) * p.lda + p.M);
  const int k_begin = static_cast<int>(rank) * p.k_per_rank;
  const int k_end = min(k_begin + p.k_per_rank, p.K);
  float acc[8 * NT];     // [row][column]
#pragma unroll
  for (int i = 0; i < 8 * NT; ++i) acc[i] = 0.0f;

  const int slot = K_MAJOR ? lane : warp * 4 + (lane >> 3);
  const int row = K_MAJOR ? row0 + warp * 8 : row0 + (lane & 7) * 8;    // the thread's first row
  const bool row_ok = row < p.M;
  for (int k = k_begin + slot * 8; k < k_end; k += kSkinnyStep) {
    uint4 w[8], x[NT];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // rows behind the last one re-read it (their sums are not stored); M_MAJOR has whole runs of 8 rows
      const T* src = K_MAJOR ? A + static_cast<int64_t>(min(row + i, p.M - 1)) * p.lda + k
                             : A + static_cast<int64_t>(k + i) * p.lda + (row_ok ? row : 0);
      if constexpr (!ANY) {
        w[i] = skinny_load_stream(src);
      } else if constexpr (K_MAJOR) {
        w[i] = any_keep(any_load_8(reinterpret_cast<const uint16_t*>(src), a_first, a_last), min(8, p.K - k));
      } else {
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        if (k + i < k_end) w[i] = any_load_8(reinterpret_cast<const uint16_t*>(src), a_first, a_last);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      x[t] = make_uint4(0u, 0u, 0u, 0u);
      if (t < n) {
        if constexpr (!ANY) {
          x[t] = *reinterpret_cast<const uint4*>(B + t * p.b_sn + k);
        } else {
          const uint16_t* src = reinterpret_cast<const uint16_t*>(B) + t * p.b_sn + k * p.b_sk;
          uint32_t e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = k + j < k_end ? src[j * p.b_sk] : 0u;
          x[t] = make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
        }
      }
    }
    float xf[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) skinny_unpack<T>(x[t], xf[t]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float wf[8];
      skinny_unpack<T>(w[i], wf);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (K_MAJOR) acc[i * NT + t] = fmaf(wf[j], xf[t][j], acc[i * NT + t]);
          else acc[j * NT + t] = fmaf(wf[j], xf[t][i], acc[j * NT + t]);
        }
    }
  }

  if constexpr (K_MAJOR) {
    const int first = skinny_reduce<8 * NT, 16, 1>(acc, lane);
    constexpr int kCopies = NT >= 4 ? 1 : 4 / NT;     // lanes that end up with the same value
    if (lane % kCopies == 0) sum[(first % NT) * kSkinnyRows + warp * 8 + first / NT] = acc[0];
  } else {
    const int first = skinny_reduce<8 * NT, 16, 8>(acc, lane);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i)
      part[warp][((first + i) % NT) * kSkinnyRows + (lane & 7) * 8 + (first + i) / NT] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < kOut; o += kSkinnyThreads) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += part[w][o];
      sum[o] = s;
    }
  }
  skinny_finish(p, sum, g, c0, n, row0, ranks, rank);
}

// Several columns, up to 16, of A with consecutive k: the same stream with the warp-level matrix instructions (m16n8k16,
// FP32 accumulators) in place of FMAs - the columns are its 16 rows, eight rows of A its 8 columns - so that the weights
// need no unpacking and the accumulators of 16 columns fit four registers.  (tcgen05 would want its operands staged in
// shared memory and tensor memory set up: the latency that this kernel avoids.  The rate is that of the loads: eight
// columns of a 4096 x 4096 layer 11.0 us against 16.1 with tcgen05.)  Lane 4 * g + t holds k0 + 8 t .. + 7 of row g of the
// warp's 8 rows and of columns g and g + 8: the instruction's K is permuted, in both operands alike, so that a lane's 16
// bytes feed two instructions.
constexpr int kSkinnyMmaCols = 16;
constexpr int kSkinnyMmaCtas = 4;      // per SM: 64 registers, eight loads of A in flight per thread (three: 13.0 us)

template <typename T>
__device__ __forceinline__ void skinny_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (SkinnyIsHalf<T>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T>
__global__ void __launch_bounds__(kSkinnyThreads, kSkinnyMmaCtas) skinny_mma_kernel(const SkinnyParams p) {
  __shared__ float sum[kSkinnyMmaCols * kSkinnyRows];                                    // [column][row]
  __shared__ int item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const uint32_t rank = cluster_cta_rank();
  const int row0 = static_cast<int>(blockIdx.x / ranks) * kSkinnyRows;

  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    int g, c0, n;
    fused_find_item(p.f, blockIdx.y, kSkinnyMmaCols, lane, g, c0, n);
    if (lane == 0) { item[0] = g; item[1] = c0; item[2] = n; }
  }
  __syncthreads();
  const int g = item[0], c0 = item[1], n = item[2];
  if (n == 0) return;    // the list is shorter than the grid; the same for every CTA of the cluster

  const T* A = static_cast<const T*>(p.A) + g * p.a_group;
  const T* B = static_cast<const T*>(p.B) + c0 * p.b_sn;
  const int k_begin = static_cast<int>(rank) * p.k_per_rank;
  const int k_end = min(k_begin + p.k_per_rank, p.K);
  const T* x0 = B + g4 * p.b_sn;                       // this lane's columns of B (read only if they exist)
  const T* x1 = B + (g4 + 8) * p.b_sn;
  const bool has0 = g4 < n, has1 = g4 + 8 < n;

  constexpr int U = 8;                               // steps of 32 k whose loads are in flight together
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const T* a_row = A + static_cast<int64_t>(min(row0 + warp * 8 + g4, p.M - 1)) * p.lda;
  for (int k = k_begin + t4 * 8; k < k_end + t4 * 8; k += 32 * U) {      // the same count for all lanes
    uint4 w[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      w[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k + 32 * i < k_end) w[i] = skinny_load_stream(a_row + k + 32 * i);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {                    // B comes from L1, which the CTA's other warps have filled
      uint4 u = make_uint4(0u, 0u, 0u, 0u), v = u;
      if (has0 && k + 32 * i < k_end) u = *reinterpret_cast<const uint4*>(x0 + k + 32 * i);
      if (has1 && k + 32 * i < k_end) v = *reinterpret_cast<const uint4*>(x1 + k + 32 * i);
      skinny_mma<T>(acc, u.x, v.x, u.y, v.y, w[i].x, w[i].y);
      skinny_mma<T>(acc, u.z, v.z, u.w, v.w, w[i].z, w[i].w);
    }
  }
  // acc: columns g4 and g4 + 8, rows 2 * t4 and 2 * t4 + 1 of the warp's
  const int r = warp * 8 + 2 * t4;
  sum[g4 * kSkinnyRows + r] = acc[0]; sum[g4 * kSkinnyRows + r + 1] = acc[1];
  sum[(g4 + 8) * kSkinnyRows + r] = acc[2]; sum[(g4 + 8) * kSkinnyRows + r + 1] = acc[3];
  skinny_finish(p, sum, g, c0, n, row0, ranks, rank);
}

// The same for A with consecutive rows and 5 to 8 columns, which are the instruction's 8 columns here (8 columns of 4096 x
// 4096: 12.4 us against 16.3-17.2 with tcgen05, of 2048 x 2048: 7.7 and 10.3; 8192 x 2048 and 8192 x 8192: even, within 0.7
// us; 16 columns would need 32 accumulators: 15.7 us, no better than tcgen05).  Lane 4 * g + t holds
// rows 8 g .. + 7 at k0 + 2 t, + 1, + 8, + 9; byte permutations put the pairs of k together, and instruction j takes rows
// 8 g + 2 j and 8 g + 2 j + 1 of every g as its rows g and g + 8.  The warps of a CTA take turns along K.
constexpr int kSkinnyMmaRowsCols = 8;
constexpr int kSkinnyMmaRowsCtas = 2;  // per SM: K is cut less (three: 14.4 us at 8 columns of 4096 x 4096; one: 15.7)

template <typename T>
__global__ void __launch_bounds__(kSkinnyThreads, kSkinnyMmaRowsCtas) skinny_mma_rows_kernel(const SkinnyParams p) {
  __shared__ float part[8][kSkinnyMmaRowsCols * kSkinnyRows];     // sums of each warp, [column][row]
  __shared__ float sum[kSkinnyMmaRowsCols * kSkinnyRows];
  __shared__ int item[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const uint32_t rank = cluster_cta_rank();
  const int row0 = static_cast<int>(blockIdx.x / ranks) * kSkinnyRows;

  pdl_launch_dependents();
  pdl_wait();
  if (warp == 0) {
    int g, c0, n;
    fused_find_item(p.f, blockIdx.y, kSkinnyMmaRowsCols, lane, g, c0, n);
    if (lane == 0) { item[0] = g; item[1] = c0; item[2] = n; }
  }
  __syncthreads();
  const int g = item[0], c0 = item[1], n = item[2];
  if (n == 0) return;    // the list is shorter than the grid; the same for every CTA of the cluster

  const int k_begin = static_cast<int>(rank) * p.k_per_rank;
  const int k_end = min(k_begin + p.k_per_rank, p.K);
  const T* x = static_cast<const T*>(p.B) + (c0 + g4) * p.b_sn;      // this lane's column of B (read only if it exists)
  const bool has = g4 < n;
  const int row = row0 + g4 * 8;
  const T* a_col = static_cast<const T*>(p.A) + g * p.a_group + (row < p.M ? row : 0);   // M is a multiple of 8; rows behind it are not stored
  float acc[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) { acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f; }
  constexpr int U = 2;                               // steps of 16 k whose loads are in flight together
  for (int k = k_begin + warp * 16 * U; k < k_end; k += 8 * 16 * U) {
    uint4 w[U][4];
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {                  // k_end is a multiple of 8: pairs of k exist together
        const int kk = k + 16 * i + 2 * t4 + (h & 1) + 8 * (h >> 1);
        w[i][h] = make_uint4(0u, 0u, 0u, 0u);
        if (kk < k_end) w[i][h] = skinny_load_stream(a_col + static_cast<int64_t>(kk) * p.lda);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int kk = k + 16 * i + 2 * t4;
      uint32_t b0 = 0u, b1 = 0u;
      if (has && kk < k_end) b0 = *reinterpret_cast<const uint32_t*>(x + kk);
      if (has && kk + 8 < k_end) b1 = *reinterpret_cast<const uint32_t*>(x + kk + 8);
      const uint32_t w0[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w}, w1[4] = {w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
      const uint32_t w2[4] = {w[i][2].x, w[i][2].y, w[i][2].z, w[i][2].w}, w3[4] = {w[i][3].x, w[i][3].y, w[i][3].z, w[i][3].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        skinny_mma<T>(acc[j], __byte_perm(w0[j], w1[j], 0x5410), __byte_perm(w0[j], w1[j], 0x7632), __byte_perm(w2[j], w3[j], 0x5410),
                      __byte_perm(w2[j], w3[j], 0x7632), b0, b1);
    }
  }
  // acc[j]: rows 8 * g4 + 2 * j and + 1, columns 2 * t4 and 2 * t4 + 1
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 8 * g4 + 2 * j;
    part[warp][2 * t4 * kSkinnyRows + r] = acc[j][0]; part[warp][(2 * t4 + 1) * kSkinnyRows + r] = acc[j][1];
    part[warp][2 * t4 * kSkinnyRows + r + 1] = acc[j][2]; part[warp][(2 * t4 + 1) * kSkinnyRows + r + 1] = acc[j][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < n * kSkinnyRows; o += kSkinnyThreads) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[w][o];
    sum[o] = s;
  }
  skinny_finish(p, sum, g, c0, n, row0, ranks, rank);
}

}  // namespace gk
