// C ABI of the library (include/gemmkernels_b200.h): handle, dispatch, error reporting.
#include <algorithm>
#include <type_traits>
#include <cmath>
#include <cstring>
#include <new>

#include "common.h"
#include "diag_gemm.cuh"
#include "fpu_gemm.cuh"
#include "fpu_gemm_f64.cuh"
#include "simt_gemm.cuh"
#include "split_planes.cuh"
#include "tc_plan.h"

namespace gk {

static thread_local char g_error[512] = "";

gk_status set_error(gk_status s, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return s;
}
void clear_error() { g_error[0] = 0; }

// ------------------------------------------------------------------------------------------------
// descriptor validation shared by every path
// ------------------------------------------------------------------------------------------------
gk_status validate_desc(const gk_gemm_desc* d, const gk_epilogue_desc* epi) {
  if (!d) return set_error(GK_ERR_INVALID_ARGUMENT, "descriptor is NULL");
  if (d->struct_size != sizeof(gk_gemm_desc))
    return set_error(GK_ERR_INVALID_ARGUMENT, "gk_gemm_desc.struct_size is %u, this library expects %zu",
                     d->struct_size, sizeof(gk_gemm_desc));
  if (epi && epi->struct_size != sizeof(gk_epilogue_desc))
    return set_error(GK_ERR_INVALID_ARGUMENT, "gk_epilogue_desc.struct_size is %u, this library expects %zu",
                     epi->struct_size, sizeof(gk_epilogue_desc));
  if (d->m < 0 || d->n < 0 || d->k < 0)
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: negative extent (%lld, %lld, %lld)",
                     (long long)d->m, (long long)d->n, (long long)d->k);
  const int64_t a_rows = d->trans_a ? d->k : d->m;
  const int64_t b_rows = d->trans_b ? d->n : d->k;
  if (d->layout_a == GK_LAYOUT_DENSE && d->lda < (a_rows > 0 ? a_rows : 1))
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: lda = %lld < %lld stored rows of A",
                     (long long)d->lda, (long long)a_rows);
  if (d->layout_b == GK_LAYOUT_DENSE && d->ldb < (b_rows > 0 ? b_rows : 1))
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: ldb = %lld < %lld stored rows of B",
                     (long long)d->ldb, (long long)b_rows);
  if (d->ldd < (d->m > 0 ? d->m : 1))
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: ldd = %lld < M = %lld",
                     (long long)d->ldd, (long long)d->m);
  if (d->layout_c == GK_LAYOUT_DENSE && d->beta != 0.0 && d->ldc < (d->m > 0 ? d->m : 1))
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: ldc = %lld < M = %lld",
                     (long long)d->ldc, (long long)d->m);
  if (dtype_size(d->dtype_a) == 0 || dtype_size(d->dtype_b) == 0 || dtype_size(d->dtype_c) == 0 ||
      dtype_size(d->dtype_d) == 0)
    return set_error(GK_ERR_UNSUPPORTED, "unknown element type in descriptor");
  if (d->number < GK_REAL || d->number > GK_DUAL)
    return set_error(GK_ERR_INVALID_CONFIG, "unknown number system %d", d->number);
  if (d->batch > 1) {
    if (d->number != GK_REAL)
      return set_error(GK_ERR_INVALID_CONFIG, "batched products are real products (number = %d)", d->number);
    if (d->layout_a == GK_LAYOUT_DIAGONAL)
      return set_error(GK_ERR_INVALID_CONFIG, "batched products do not take a Diagonal A");
    if (d->batch_stride_a < 0 || d->batch_stride_b < 0 || d->batch_stride_c < 0 || d->batch_stride_d < 0)
      return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: negative batch stride");
    if (d->m > 0 && d->n > 0 && d->batch_stride_d < d->ldd * (d->n - 1) + d->m)
      return set_error(GK_ERR_DIMENSION_MISMATCH,
                       "Dimensions do not match: batch_stride_d = %lld makes the outputs of the batch overlap",
                       (long long)d->batch_stride_d);
  }
  if (epi) {
    if (epi->bias_axis < GK_BIAS_NONE || epi->bias_axis > GK_BIAS_COL)
      return set_error(GK_ERR_UNSUPPORTED, "bias axis %d is not none/row/column", epi->bias_axis);
    if (epi->activation < GK_ACT_NONE || epi->activation > GK_ACT_GELU)
      return set_error(GK_ERR_UNSUPPORTED, "activation %d is not one of none/ReLU/GELU", epi->activation);
  }
  return GK_OK;
}

// FP32 FFMA fast path: the reference's UnsafeAligned* conditions (tile-multiple sizes, 16-byte
// aligned columns), all four matrices Float32.
static bool fpu_eligible(const gk_gemm_desc& d, const void* a, const void* b, const void* c, const void* dd,
                         const gk_epilogue_desc* epi) {
  if (d.op == GK_OP_FPU_TROPICAL || d.op == GK_OP_TCGEN05 || d.number != GK_REAL) return false;
  if (d.dtype_a != d.dtype_b || d.dtype_d != GK_F32) return false;
  if (d.dtype_a != GK_F32 && d.dtype_a != GK_F16 && d.dtype_a != GK_BF16) return false;
  if (d.compute != GK_F32 && d.compute != d.dtype_a) return false;
  if (d.layout_a != GK_LAYOUT_DENSE || d.layout_b != GK_LAYOUT_DENSE) return false;
  const bool has_c = d.layout_c == GK_LAYOUT_DENSE && d.beta != 0.0;
  if (has_c && (d.dtype_c != GK_F32 || d.ldc % 4)) return false;
  if (d.m < kFpuBM || d.n < kFpuBN || d.k < kFpuBK) return false;
  if (d.m % kFpuBM || d.n % kFpuBN || d.k % kFpuBK) return false;
  if (d.m > INT32_MAX / 2 || d.n > INT32_MAX / 2 || d.k > INT32_MAX / 2) return false;
  const int chunk = d.dtype_a == GK_F32 ? 4 : 8;   // elements per 16-byte copy
  if (d.lda % chunk || d.ldb % chunk || d.ldd % 4) return false;
  auto misaligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (misaligned(a) || misaligned(b) || misaligned(dd) || (has_c && misaligned(c))) return false;
  if (epi && epi->bias_axis != GK_BIAS_NONE && misaligned(epi->bias)) return false;
  return true;
}

// FP64 fast path (fpu_gemm_f64.cuh): the same conditions with all four matrices Float64.
static bool f64_eligible(gk_handle h, const gk_gemm_desc& d, const void* a, const void* b, const void* c, const void* dd,
                         const gk_epilogue_desc* epi) {
  if (d.op == GK_OP_FPU_TROPICAL || d.op == GK_OP_TCGEN05 || d.number != GK_REAL) return false;
  if (d.dtype_a != GK_F64 || d.dtype_b != GK_F64 || d.dtype_d != GK_F64) return false;
  if (d.compute != GK_F64) return false;
  if (d.layout_a != GK_LAYOUT_DENSE || d.layout_b != GK_LAYOUT_DENSE) return false;
  const bool has_c = d.layout_c == GK_LAYOUT_DENSE && d.beta != 0.0;
  if (has_c && (d.dtype_c != GK_F64 || d.ldc % 2)) return false;
  if (d.m < kF64BM || d.n < kF64BN || d.k < kF64BK) return false;
  if (d.m % kF64BM || d.n % kF64BN || d.k % kF64BK) return false;
  if (d.m > INT32_MAX / 2 || d.n > INT32_MAX / 2 || d.k > INT32_MAX / 2) return false;
  // One 128 x 128 tile per SM at a time: below three quarters of a round the generic kernel's 64 x 64 tiles
  // fill the GPU better (1024^3: 13.7 TFLOP/s there, 9.9 here; 2048^3: 16.6 against 20.2).
  if (4 * (d.m / kF64BM) * (d.n / kF64BN) < 3 * static_cast<int64_t>(h->sm_count)) return false;
  if (d.lda % 2 || d.ldb % 2 || d.ldd % 2) return false;
  auto misaligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  if (misaligned(a) || misaligned(b) || misaligned(dd) || (has_c && misaligned(c))) return false;
  return true;
}

static gk_status launch_f64(gk_handle h, const gk_gemm_desc& d, const gk_epilogue_desc* epi, const void* a,
                            const void* b, const void* c, void* dd, cudaStream_t stream) {
  F64Params p{};
  p.A = static_cast<const double*>(a); p.B = static_cast<const double*>(b);
  p.C = static_cast<const double*>(c); p.D = static_cast<double*>(dd);
  p.M = static_cast<int>(d.m); p.N = static_cast<int>(d.n); p.K = static_cast<int>(d.k);
  p.lda = d.lda; p.ldb = d.ldb; p.ldc = d.ldc; p.ldd = d.ldd;
  p.alpha = d.alpha;
  p.beta = (d.layout_c == GK_LAYOUT_DENSE && c) ? d.beta : 0.0;
  if (epi) { p.bias = epi->bias; p.bias_axis = epi->bias_axis; p.act = epi->activation; }
  p.tiles_m = p.M / kF64BM; p.tiles_n = p.N / kF64BN;
  int group = d.raster_group > 0 ? d.raster_group : static_cast<int>(std::lround(std::sqrt(static_cast<double>(h->sm_count))));
  if (d.raster == GK_RASTER_IDENTITY) group = p.tiles_m;
  p.raster_group = std::max(1, std::min(group, p.tiles_m));
  const dim3 grid(static_cast<unsigned>(p.tiles_m) * static_cast<unsigned>(p.tiles_n));
  const bool ak = d.trans_a != 0;   // stored K x M: K is the contiguous index of A
  const bool bk = d.trans_b == 0;   // stored K x N: K is the contiguous index of B
  cudaError_t attr_err = cudaSuccess;
  auto run = [&](auto kernel, int slot) {
    std::lock_guard<std::mutex> lock(h->mu);
    bool& set = h->f64_attr_set[slot];
    if (!set) {
      attr_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kF64SmemBytes);
      if (attr_err != cudaSuccess) return;
      set = true;
    }
    kernel<<<grid, kF64Threads, kF64SmemBytes, stream>>>(p);
  };
  if (ak && bk) run(fpu_gemm_f64_kernel<true, true>, 3);
  else if (ak && !bk) run(fpu_gemm_f64_kernel<true, false>, 2);
  else if (!ak && bk) run(fpu_gemm_f64_kernel<false, true>, 1);
  else run(fpu_gemm_f64_kernel<false, false>, 0);
  GK_CUDA_CHECK(attr_err);
  GK_CUDA_CHECK(cudaGetLastError());
  return GK_OK;
}

// K split of the FFMA kernel (fpu_gemm.cuh): how many parts the tiles of the last round - or, when the
// whole grid is smaller than half a round, all tiles - are cut into (1 = none), the first split tile,
// and the workspace the partial sums need.
struct FpuSplit { int q = 1, first = 0; int64_t bytes = 0; };
static FpuSplit fpu_plan_split(gk_handle h, const gk_gemm_desc& d) {
  FpuSplit sp;
  const int64_t tiles = (d.m / kFpuBM) * (d.n / kFpuBN);
  const int64_t slots = 2 * static_cast<int64_t>(h->sm_count);     // two CTAs per SM
  const int64_t rem = tiles % slots;
  const int64_t kt = d.k / kFpuBK;
  if (2 * tiles <= slots) {
    // Fewer tiles than half the slots: every tile is cut along K so that the grid fills the GPU.
    int q = static_cast<int>(std::min<int64_t>(slots / tiles, 8));
    while (q > 1 && kt / q < 8) --q;
    if (q < 2) return sp;
    sp.q = q; sp.first = 0;
    sp.bytes = tiles * q * static_cast<int64_t>(kFpuBM) * kFpuBN * 4;
    return sp;
  }
  if (tiles <= slots || rem == 0 || 2 * rem > slots || kt < 64) return sp;   // one round, a full last round, or a short K
  int q = static_cast<int>(std::min<int64_t>(slots / rem, 4));
  while (q > 1 && kt / q < 16) --q;
  if (q < 2) return sp;
  sp.q = q; sp.first = static_cast<int>(tiles - rem);
  sp.bytes = rem * q * static_cast<int64_t>(kFpuBM) * kFpuBN * 4;
  return sp;
}

static gk_status launch_fpu(gk_handle h, const gk_gemm_desc& d, const gk_epilogue_desc* epi, const void* a,
                            const void* b, const void* c, void* dd, cudaStream_t stream, void* workspace = nullptr,
                            int64_t workspace_bytes = 0) {
  FpuParams p{};
  p.A = a; p.B = b;
  p.C = static_cast<const float*>(c); p.D = static_cast<float*>(dd);
  p.M = static_cast<int>(d.m); p.N = static_cast<int>(d.n); p.K = static_cast<int>(d.k);
  p.lda = d.lda; p.ldb = d.ldb; p.ldc = d.ldc; p.ldd = d.ldd;
  p.alpha = static_cast<float>(d.alpha);
  p.beta = (d.layout_c == GK_LAYOUT_DENSE && c) ? static_cast<float>(d.beta) : 0.0f;
  if (epi) { p.bias = epi->bias; p.bias_axis = epi->bias_axis; p.act = epi->activation; }
  p.tiles_m = p.M / kFpuBM; p.tiles_n = p.N / kFpuBN;
  // 2 CTAs per SM run together: make the set of tiles in flight roughly square
  int group = d.raster_group > 0 ? d.raster_group
                                 : static_cast<int>(std::lround(std::sqrt(2.0 * h->sm_count)));
  if (d.raster == GK_RASTER_IDENTITY) group = p.tiles_m;
  p.raster_group = std::max(1, std::min(group, p.tiles_m));
  p.split_q = 1; p.split_first = 0; p.kt_per_part = 0; p.ws = nullptr;
  unsigned blocks = static_cast<unsigned>(p.tiles_m) * static_cast<unsigned>(p.tiles_n);
  const FpuSplit sp = fpu_plan_split(h, d);
  if (sp.q > 1 && workspace && workspace_bytes >= sp.bytes && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0) {
    p.split_q = sp.q; p.split_first = sp.first; p.ws = static_cast<float*>(workspace);
    const int kt = p.K / kFpuBK;
    p.kt_per_part = (kt + sp.q - 1) / sp.q;
    blocks = static_cast<unsigned>(sp.first) + (blocks - static_cast<unsigned>(sp.first)) * static_cast<unsigned>(sp.q);
  }
  const dim3 grid(blocks);
  const bool ak = d.trans_a != 0;   // stored K x M: K is the contiguous index of A
  const bool bk = d.trans_b == 0;   // stored K x N: K is the contiguous index of B
  // The kernels ask for more dynamic shared memory than the default limit: raise it once per instance and device.
  cudaError_t attr_err = cudaSuccess;
  auto run = [&](auto kernel, int slot) {
    std::lock_guard<std::mutex> lock(h->mu);
    bool& set = h->fpu_attr_set[slot];
    if (!set) {
      attr_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFpuSmemBytes);
      if (attr_err != cudaSuccess) return;
      set = true;
    }
    kernel<<<grid, kFpuThreads, kFpuSmemBytes, stream>>>(p);
  };
  auto launch = [&](auto tag, int type_slot) {
    using TIn = decltype(tag);
    const int slot = type_slot * 4 + (ak ? 2 : 0) + (bk ? 1 : 0);
    if (ak && bk) run(fpu_gemm_kernel<true, true, TIn>, slot);
    else if (ak && !bk) run(fpu_gemm_kernel<true, false, TIn>, slot);
    else if (!ak && bk) run(fpu_gemm_kernel<false, true, TIn>, slot);
    else run(fpu_gemm_kernel<false, false, TIn>, slot);
  };
  if (d.dtype_a == GK_F16) launch(__half{}, 1);
  else if (d.dtype_a == GK_BF16) launch(__nv_bfloat16{}, 2);
  else launch(float{}, 0);
  GK_CUDA_CHECK(attr_err);
  GK_CUDA_CHECK(cudaGetLastError());
  if (p.split_q > 1) {
    const unsigned n_split = static_cast<unsigned>(p.tiles_m) * static_cast<unsigned>(p.tiles_n) - static_cast<unsigned>(p.split_first);
    fpu_tail_reduce_kernel<<<n_split, 256, 0, stream>>>(p);
    GK_CUDA_CHECK(cudaGetLastError());
  }
  return GK_OK;
}

// Interleaved complex / dual operands (plane_x == 0) are split into planes in the workspace first.
// Layout of the workspace: A planes, then B planes; leading dimensions rounded up to 8 elements.
struct SplitPlan {
  bool a = false, b = false;
  int64_t a_rows = 0, a_cols = 0, a_ld = 0, b_rows = 0, b_cols = 0, b_ld = 0;
  int64_t a_bytes = 0, b_bytes = 0;
};

static SplitPlan plan_split(const gk_gemm_desc& d) {
  SplitPlan sp;
  if (d.number == GK_REAL || d.layout_a != GK_LAYOUT_DENSE || d.layout_b != GK_LAYOUT_DENSE) return sp;
  auto up8 = [](int64_t x) { return (x + 7) / 8 * 8; };
  const int64_t es = dtype_size(d.dtype_a);
  if (d.plane_a == 0) {
    sp.a = true; sp.a_rows = d.trans_a ? d.k : d.m; sp.a_cols = d.trans_a ? d.m : d.k; sp.a_ld = up8(sp.a_rows);
    sp.a_bytes = (2 * sp.a_ld * sp.a_cols * es + 255) / 256 * 256;
  }
  if (d.plane_b == 0) {
    sp.b = true; sp.b_rows = d.trans_b ? d.n : d.k; sp.b_cols = d.trans_b ? d.k : d.n; sp.b_ld = up8(sp.b_rows);
    sp.b_bytes = (2 * sp.b_ld * sp.b_cols * dtype_size(d.dtype_b) + 255) / 256 * 256;
  }
  return sp;
}

static gk_status launch_split(int dtype, const void* in, void* out, int64_t rows, int64_t cols, int64_t ld_in,
                              int64_t ld_out, int sm_count, cudaStream_t stream) {
  const int64_t total = rows * cols;
  if (total == 0) return GK_OK;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((total + 255) / 256, static_cast<int64_t>(sm_count) * 16)));
  const int64_t plane = ld_out * cols;
  if (dtype == GK_F16 || dtype == GK_BF16)
    split_planes_kernel<ushort2, unsigned short><<<grid, 256, 0, stream>>>(
        static_cast<const ushort2*>(in), static_cast<unsigned short*>(out), rows, cols, ld_in, ld_out, plane);
  else if (dtype == GK_F32)
    split_planes_kernel<float2, float><<<grid, 256, 0, stream>>>(
        static_cast<const float2*>(in), static_cast<float*>(out), rows, cols, ld_in, ld_out, plane);
  else
    return set_error(GK_ERR_UNSUPPORTED, "interleaved operands must be Float16, BFloat16 or Float32 pairs");
  GK_CUDA_CHECK(cudaGetLastError());
  return GK_OK;
}

// Diagonal A: row scaling of B (HBM-bound).
static gk_status launch_diag(gk_handle h, const gk_gemm_desc& d, const gk_epilogue_desc* epi, const void* a,
                             const void* b, const void* c, void* dd, cudaStream_t stream, gk_gemm_plan* plan_only) {
  auto dt3 = [](int32_t t) { return t == GK_F16 ? 0 : t == GK_BF16 ? 1 : t == GK_F32 ? 2 : -1; };
  if (d.m != d.k)
    return set_error(GK_ERR_INVALID_CONFIG, "Diagonal only supports square A matrix (M == K), got M = %lld, K = %lld",
                     (long long)d.m, (long long)d.k);
  if (d.number != GK_REAL || d.op == GK_OP_FPU_TROPICAL)
    return set_error(GK_ERR_INVALID_CONFIG, "Diagonal layout is for real products only");
  if (d.dtype_a != d.dtype_b || dt3(d.dtype_a) < 0 || dt3(d.dtype_d) < 0 || dt3(d.dtype_c) < 0)
    return set_error(GK_ERR_UNSUPPORTED, "Diagonal layout takes Float16/BFloat16/Float32 operands (A and B of one type)");
  if (d.layout_b != GK_LAYOUT_DENSE)
    return set_error(GK_ERR_INVALID_CONFIG, "Diagonal A needs a dense B");
  DiagParams p{};
  p.v = a; p.B = b; p.C = c; p.D = dd; p.M = d.m; p.N = d.n;
  p.b_sm = d.trans_b ? d.ldb : 1; p.b_sn = d.trans_b ? 1 : d.ldb;   // op(B)(m, n): B is K x N, K == M
  p.ldc = d.ldc; p.ldd = d.ldd;
  p.dtype_ab = dt3(d.dtype_a); p.dtype_c = dt3(d.dtype_c); p.dtype_d = dt3(d.dtype_d);
  p.alpha = static_cast<float>(d.alpha); p.beta = static_cast<float>(d.beta);
  p.has_c = (d.layout_c == GK_LAYOUT_DENSE && c != nullptr && d.beta != 0.0) ? 1 : 0;
  if (epi) { p.bias = epi->bias; p.bias_axis = epi->bias_axis; p.act = epi->activation; }
  auto al16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  const bool vec = !d.trans_b && (d.dtype_a == GK_F16 || d.dtype_a == GK_BF16) && d.dtype_d == GK_F32 &&
                   (!p.has_c || d.dtype_c == GK_F32) && d.m % 8 == 0 && d.ldb % 8 == 0 && d.ldd % 4 == 0 &&
                   (!p.has_c || d.ldc % 4 == 0) && (plan_only || (al16(a) && al16(b) && al16(dd) && (!p.has_c || al16(c))));
  const int64_t work = vec ? (d.m / 8) * d.n : d.m * d.n;
  const int64_t want = (work + 255) / 256;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, static_cast<int64_t>(h->sm_count) * 16)));
  if (plan_only) {
    plan_only->kernel = 4; plan_only->grid = grid; plan_only->block = 256; plan_only->cluster = 1;
    plan_only->tile_m = vec ? 8 : 1; plan_only->tile_n = 1; plan_only->tile_k = 1; plan_only->stages = 1;
    return GK_OK;
  }
  if (d.m == 0 || d.n == 0) return GK_OK;
  void (*kern)(const DiagParams) = !vec ? diag_gemm_scalar_kernel
                                        : (d.dtype_a == GK_F16 ? diag_gemm_vec_kernel<__half> : diag_gemm_vec_kernel<__nv_bfloat16>);
  GK_CUDA_CHECK(launch_dependent(kern, dim3(grid), dim3(256), 0, stream, p));
  GK_CUDA_CHECK(cudaGetLastError());
  return GK_OK;
}

// Which kernel family serves this descriptor: 1 tcgen05, 2 FP32 FFMA, 3 generic SIMT, 4 diagonal.
// *generic_loads is set when the tensor-core kernel must read its operands with ordinary loads
// (TMA cannot address them: alignment), which the reference's bounds-checked layouts correspond to
// (src/layout.jl:111-184, chosen in src/matmul.jl:121-156).
static int choose_family(const gk_gemm_desc& d, const void* a, const void* b, std::string* why, bool* generic_loads = nullptr) {
  if (generic_loads) *generic_loads = false;
  if (d.layout_a == GK_LAYOUT_DIAGONAL) return 4;
  if (d.m == 0 || d.n == 0) return 3;          // nothing to write: no launch follows
  // Nothing to multiply (Layout.Zero operands, alpha == 0, K == 0): D = act(beta * C + bias),
  // which the generic kernel does without touching A or B.
  const bool no_product = d.layout_a == GK_LAYOUT_ZERO || d.layout_b == GK_LAYOUT_ZERO ||
                          d.alpha == 0.0 || d.k == 0;
  if (no_product && d.number == GK_REAL) return 3;
  const bool tc_types = (d.compute == GK_F16 || d.compute == GK_BF16 || d.compute == GK_TF32);
  if (d.op == GK_OP_TCGEN05 || (d.op == GK_OP_AUTO && tc_types)) {
    if (tc_eligible(d, a, b, why)) return 1;
    // Only TMA's alignment rule stands in the way: the same kernel, fed by bounds-checked loads.
    std::string why2;
    if (generic_loads && tc_eligible_generic(d, &why2)) { *generic_loads = true; return 1; }
    return -1;                                 // no SIMT complex/dual kernel; an FP32 SIMT result is not a TF32 result
  }
  if (d.number != GK_REAL) { if (why) *why = "complex and dual products need the TCGen05Operator"; return -1; }
  return 3;
}

// ------------------------------------------------------------------------------------------------
// generic SIMT dispatch
// ------------------------------------------------------------------------------------------------
template <typename TIn, typename TOut, typename TAcc>
static gk_status launch_simt_typed(const SimtParams& p, bool tropical, cudaStream_t stream) {
  // 128 x 128 tiles (8 x 8 outputs per thread) for FP32 accumulation once there are enough of them to fill
  // the GPU; 64 x 64 tiles otherwise (measured: the larger tile gains 8 % on Float16 -> Float32, nothing
  // on Int32, and loses on Int16)
  constexpr bool kFloatAcc = std::is_same<TAcc, float>::value;
  const bool big = kFloatAcc && ((p.M + 127) / 128) * ((p.N + 127) / 128) >= 96;
  const int tile = big ? 128 : kSimtTile;
  dim3 grid(static_cast<unsigned>((p.M + tile - 1) / tile), static_cast<unsigned>((p.N + tile - 1) / tile));
  if (grid.y > 65535u) return set_error(GK_ERR_INVALID_CONFIG, "N too large for the generic kernel");
  if constexpr (kFloatAcc) {
    if (big) {
      if (tropical) simt_gemm_kernel<TIn, TOut, TAcc, true, 8><<<grid, kSimtThreads, 0, stream>>>(p);
      else simt_gemm_kernel<TIn, TOut, TAcc, false, 8><<<grid, kSimtThreads, 0, stream>>>(p);
      GK_CUDA_CHECK(cudaGetLastError());
      return GK_OK;
    }
  }
  if (tropical)
    simt_gemm_kernel<TIn, TOut, TAcc, true, 4><<<grid, kSimtThreads, 0, stream>>>(p);
  else
    simt_gemm_kernel<TIn, TOut, TAcc, false, 4><<<grid, kSimtThreads, 0, stream>>>(p);
  GK_CUDA_CHECK(cudaGetLastError());
  return GK_OK;
}

static gk_status launch_simt(const gk_gemm_desc& d, const gk_epilogue_desc* epi, const void* a,
                             const void* b, const void* c, void* dd, cudaStream_t stream) {
  if (d.dtype_a != d.dtype_b)
    return set_error(GK_ERR_UNSUPPORTED, "A (%s) and B (%s) must have the same element type",
                     dtype_name(d.dtype_a), dtype_name(d.dtype_b));
  if (d.dtype_c != d.dtype_d)
    return set_error(GK_ERR_UNSUPPORTED, "C (%s) and D (%s) must have the same element type",
                     dtype_name(d.dtype_c), dtype_name(d.dtype_d));
  if (d.m == 0 || d.n == 0) return GK_OK;
  SimtParams p{};
  p.A = a; p.B = b; p.C = c; p.D = dd;
  p.M = d.m; p.N = d.n; p.K = d.k;
  p.a_sm = d.trans_a ? d.lda : 1; p.a_sk = d.trans_a ? 1 : d.lda;
  p.b_sk = d.trans_b ? d.ldb : 1; p.b_sn = d.trans_b ? 1 : d.ldb;
  p.ldc = d.ldc; p.ldd = d.ldd;
  p.alpha = d.alpha; p.beta = d.beta;
  p.has_c = (d.layout_c != GK_LAYOUT_ZERO && c != nullptr && d.beta != 0.0) ? 1 : 0;
  p.a_zero = (d.layout_a == GK_LAYOUT_ZERO || d.layout_b == GK_LAYOUT_ZERO || d.alpha == 0.0 || d.k == 0) ? 1 : 0;
  if (d.layout_a == GK_LAYOUT_DIAGONAL)
    return set_error(GK_ERR_UNSUPPORTED, "Diagonal layout is not handled by the generic kernel");
  if (epi) { p.bias = epi->bias; p.bias_axis = epi->bias_axis; p.act = epi->activation; }
  const bool trop = d.op == GK_OP_FPU_TROPICAL;
  const int ti = d.dtype_a, to = d.dtype_d;
  if (ti == GK_F16 && to == GK_F32) return launch_simt_typed<__half, float, float>(p, trop, stream);
  if (ti == GK_F16 && to == GK_F16) return launch_simt_typed<__half, __half, float>(p, trop, stream);
  if (ti == GK_BF16 && to == GK_F32) return launch_simt_typed<__nv_bfloat16, float, float>(p, trop, stream);
  if (ti == GK_BF16 && to == GK_BF16) return launch_simt_typed<__nv_bfloat16, __nv_bfloat16, float>(p, trop, stream);
  if (ti == GK_F32 && to == GK_F32) return launch_simt_typed<float, float, float>(p, trop, stream);
  if (ti == GK_F32 && to == GK_F64) return launch_simt_typed<float, double, double>(p, trop, stream);
  if (ti == GK_F64 && to == GK_F64) return launch_simt_typed<double, double, double>(p, trop, stream);
  if (ti == GK_I16 && to == GK_I16) return launch_simt_typed<int16_t, int16_t, int16_t>(p, trop, stream);
  if (ti == GK_I32 && to == GK_I32) return launch_simt_typed<int32_t, int32_t, int32_t>(p, trop, stream);
  if (ti == GK_I64 && to == GK_I64) return launch_simt_typed<int64_t, int64_t, int64_t>(p, trop, stream);
  return set_error(GK_ERR_UNSUPPORTED, "no kernel for element types A/B %s, C/D %s", dtype_name(ti), dtype_name(to));
}

}  // namespace gk

using namespace gk;

// Register-only FP32 FMA throughput probe: kFmaPeakChains independent packed-FMA chains per thread.
constexpr int kFmaPeakChains = 16;
__global__ void __launch_bounds__(256) fma_peak_kernel(float* sink, int iters, float seed) {
  float2 acc[kFmaPeakChains];
#pragma unroll
  for (int i = 0; i < kFmaPeakChains; ++i) acc[i] = make_float2(seed + i, seed - i);
  const float2 a = make_float2(1.0f + 1e-7f * threadIdx.x, 1.0f - 1e-7f * threadIdx.x);
  const float2 b = make_float2(1e-9f, -1e-9f);
  for (int it = 0; it < iters; ++it) {
#pragma unroll
    for (int i = 0; i < kFmaPeakChains; ++i) acc[i] = __ffma2_rn(acc[i], a, b);
  }
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < kFmaPeakChains; ++i) s += acc[i].x + acc[i].y;
  if (s == 12345.678f) *sink = s;   // keeps the chains alive; practically never true
}

extern "C" {

int32_t gk_version(void) { return GK_VERSION_MAJOR * 1000 + GK_VERSION_MINOR; }

const char* gk_last_error_message(void) { return g_error; }

gk_status gk_create(gk_handle* out) {
  clear_error();
  if (!out) return set_error(GK_ERR_INVALID_ARGUMENT, "out is NULL");
  *out = nullptr;
  int dev = 0;
  GK_CUDA_CHECK(cudaGetDevice(&dev));
  cudaDeviceProp prop{};
  GK_CUDA_CHECK(cudaGetDeviceProperties(&prop, dev));
  if (prop.major != 10)
    return set_error(GK_ERR_CUDA, "device %d is sm_%d%d; this library is built for sm_100a only", dev,
                     prop.major, prop.minor);
  gk_handle h = new (std::nothrow) gk_handle_s();
  if (!h) return set_error(GK_ERR_CUDA, "out of host memory");
  h->device = dev;
  h->sm_count = prop.multiProcessorCount;
  h->cc_major = prop.major; h->cc_minor = prop.minor;
  h->max_smem_optin = static_cast<int>(prop.sharedMemPerBlockOptin);
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn) {
    delete h;
    return set_error(GK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
  }
  h->encode_tiled = reinterpret_cast<EncodeTiledFn>(fn);
  e = cudaHostAlloc(reinterpret_cast<void**>(&h->status_host), 16 * sizeof(int32_t), cudaHostAllocMapped);
  if (e != cudaSuccess) { delete h; return set_error(GK_ERR_CUDA, "cudaHostAlloc failed: %s", cudaGetErrorString(e)); }
  for (int i = 0; i < 16; ++i) h->status_host[i] = 0;
  e = cudaHostGetDevicePointer(reinterpret_cast<void**>(&h->status_dev), h->status_host, 0);
  if (e != cudaSuccess) {
    cudaFreeHost(h->status_host); delete h;
    return set_error(GK_ERR_CUDA, "cudaHostGetDevicePointer failed: %s", cudaGetErrorString(e));
  }
  *out = h;
  return GK_OK;
}

gk_status gk_destroy(gk_handle h) {
  clear_error();
  if (!h) return GK_OK;
  mgpu_release(h);
  for (int i = 0; i < 5; ++i)
    if (h->stage_dev[i]) cudaFree(h->stage_dev[i]);
  for (cudaEvent_t e : h->events) cudaEventDestroy(e);
  if (h->copy_in) cudaStreamDestroy(h->copy_in);
  if (h->copy_out) cudaStreamDestroy(h->copy_out);
  if (h->status_host) cudaFreeHost(h->status_host);
  delete h;
  return GK_OK;
}

gk_status gk_poll_status(gk_handle h, int32_t* raw_code) {
  clear_error();
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  const int32_t code = *reinterpret_cast<volatile int32_t*>(h->status_host);
  if (raw_code) *raw_code = code;
  if (code == 0) return GK_OK;
  *reinterpret_cast<volatile int32_t*>(h->status_host) = 0;
  return set_error(GK_ERR_TIMEOUT, "a device-side wait gave up (code %d: %s)", code,
                   code == 101 ? "TMA producer" : code == 102 ? "MMA issuer"
                   : code == 103 ? "epilogue" : code == 104 ? "drain" : "unknown");
}

gk_status gk_debug_marks(gk_handle h, int32_t* out16) {
  clear_error();
  if (!h || !out16) return set_error(GK_ERR_INVALID_ARGUMENT, "handle or output is NULL");
  for (int i = 0; i < 16; ++i) out16[i] = reinterpret_cast<volatile int32_t*>(h->status_host)[i];
  return GK_OK;
}

gk_status gk_measure_fp32_fma(gk_handle h, double* tflops, gk_stream stream) {
  clear_error();
  if (!h || !tflops) return set_error(GK_ERR_INVALID_ARGUMENT, "handle or output is NULL");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* sink = nullptr;
  GK_CUDA_CHECK(cudaMalloc(&sink, sizeof(float)));
  cudaEvent_t e0, e1;
  GK_CUDA_CHECK(cudaEventCreate(&e0));
  GK_CUDA_CHECK(cudaEventCreate(&e1));
  const int blocks = h->sm_count * 8, threads = 256, iters = 4096;
  fma_peak_kernel<<<blocks, threads, 0, st>>>(sink, iters, 1.0f);   // warm-up (clocks, instruction cache)
  double best_ms = 1e30;
  for (int rep = 0; rep < 5; ++rep) {
    cudaEventRecord(e0, st);
    fma_peak_kernel<<<blocks, threads, 0, st>>>(sink, iters, 1.0f);
    cudaEventRecord(e1, st);
    cudaError_t e = cudaEventSynchronize(e1);
    float ms = 0.0f;
    if (e == cudaSuccess) e = cudaEventElapsedTime(&ms, e0, e1);
    if (e != cudaSuccess) {
      cudaEventDestroy(e0); cudaEventDestroy(e1); cudaFree(sink);
      return set_error(GK_ERR_CUDA, "FMA measurement failed: %s", cudaGetErrorString(e));
    }
    best_ms = std::min(best_ms, static_cast<double>(ms));
  }
  cudaEventDestroy(e0); cudaEventDestroy(e1); cudaFree(sink);
  const double fmas = static_cast<double>(blocks) * threads * iters * kFmaPeakChains * 2;   // 2 lanes per packed FMA
  *tflops = 2.0 * fmas / (best_ms * 1e-3) / 1e12;
  return GK_OK;
}

gk_status gk_load_tuning(gk_handle h, const gk_tuning_entry* entries, int32_t count) {
  clear_error();
  if (!h || count < 0 || (count > 0 && !entries)) return set_error(GK_ERR_INVALID_ARGUMENT, "handle or entries is NULL, or a negative count");
  for (int i = 0; i < count; ++i) {
    const gk_tuning_entry& e = entries[i];
    const bool tile_ok = e.tile_n == 0 || e.tile_n == 512 || (e.tile_n >= 32 && e.tile_n <= 256 && e.tile_n % 32 == 0);
    if (!tile_ok || e.cta_group < 0 || e.cta_group > 2 || e.stages < 0 || e.raster_group < 0 || e.m < 1 || e.n < 1 || e.k < 1 ||
        e.k_blocks_per_stage < 0 || e.k_blocks_per_stage > 2)
      return set_error(GK_ERR_INVALID_CONFIG, "tuning entry %d is not usable (tile_n %d, cta_group %d, stages %d)", i, e.tile_n,
                       e.cta_group, e.stages);
  }
  std::lock_guard<std::mutex> lock(h->mu);
  h->tuning.assign(entries, entries + count);
  return GK_OK;
}

gk_status gk_gemm_query(gk_handle h, const gk_gemm_desc* desc, const gk_epilogue_desc* epi,
                        gk_gemm_plan* plan) {
  clear_error();
  if (!h || !plan) return set_error(GK_ERR_INVALID_ARGUMENT, "handle or plan is NULL");
  gk_status s = validate_desc(desc, epi);
  if (s != GK_OK) return s;
  std::memset(plan, 0, sizeof(*plan));
  std::string why;
  gk_gemm_desc planar = *desc;          // what the kernel sees once interleaved operands are split
  const SplitPlan sp = plan_split(*desc);
  if (sp.a) { planar.lda = sp.a_ld; planar.plane_a = sp.a_ld * sp.a_cols; }
  if (sp.b) { planar.ldb = sp.b_ld; planar.plane_b = sp.b_ld * sp.b_cols; }
  desc = &planar;
  bool generic_loads = false;
  const int fam = choose_family(*desc, nullptr, nullptr, &why, &generic_loads);
  if (fam < 0) return set_error(GK_ERR_INVALID_CONFIG, "no kernel takes this GEMM: %s", why.c_str());
  plan->kernel = fam;
  if (fam == 4) return launch_diag(h, *desc, epi, nullptr, nullptr, nullptr, nullptr, nullptr, plan);
  if (fam == 1) {
    TcLaunch L;
    TcProblem pr;
    tc_problem_from_gemm(*desc, epi, nullptr, nullptr, nullptr, nullptr, &pr);
    pr.generic = generic_loads;
    s = tc_plan(h, pr, false, &L);
    if (s != GK_OK) return s;
    plan->grid = L.grid; plan->block = tc_threads(L.planes); plan->cluster = L.cg;
    plan->smem_bytes = L.smem_bytes; plan->tmem_columns = static_cast<int32_t>(L.params.tmem_cols);
    plan->tile_m = kTcTileM * L.cg; plan->tile_n = L.params.bn * L.params.n_sub; plan->tile_k = L.params.bk * L.params.kps;
    plan->stages = L.params.stages;
    plan->workspace_bytes = sp.a_bytes + sp.b_bytes;
    if (!(sp.a || sp.b) && desc->batch <= 1) plan->workspace_bytes = tc_split_workspace_bytes(h, pr, L);   // optional: enables split-K
  } else if (fam == 3 && fpu_eligible(*desc, nullptr, nullptr, nullptr, nullptr, nullptr)) {
    plan->kernel = 2;
    plan->grid = static_cast<int32_t>((desc->m / kFpuBM) * (desc->n / kFpuBN));
    plan->block = kFpuThreads; plan->cluster = 1;
    plan->smem_bytes = kFpuSmemBytes;
    plan->tile_m = kFpuBM; plan->tile_n = kFpuBN; plan->tile_k = kFpuBK; plan->stages = kFpuStages;
    if (desc->batch <= 1) plan->workspace_bytes = fpu_plan_split(h, *desc).bytes;   // optional: splits the last round's tiles along K
  } else if (fam == 3 && f64_eligible(h, *desc, nullptr, nullptr, nullptr, nullptr, nullptr)) {
    plan->kernel = 2;
    plan->grid = static_cast<int32_t>((desc->m / kF64BM) * (desc->n / kF64BN));
    plan->block = kF64Threads; plan->cluster = 1;
    plan->smem_bytes = kF64SmemBytes;
    plan->tile_m = kF64BM; plan->tile_n = kF64BN; plan->tile_k = kF64BK; plan->stages = kF64Stages;
  } else {
    // same rule as launch_simt_typed: 128 x 128 tiles for 4-byte accumulators once there are 96 of them
    const bool float_acc = desc->dtype_d == GK_F32 || desc->dtype_d == GK_F16 || desc->dtype_d == GK_BF16;
    const int tile = (float_acc && ((desc->m + 127) / 128) * ((desc->n + 127) / 128) >= 96) ? 128 : kSimtTile;
    plan->grid = static_cast<int32_t>(((desc->m + tile - 1) / tile) * ((desc->n + tile - 1) / tile));
    plan->block = kSimtThreads; plan->cluster = 1;
    plan->tile_m = tile; plan->tile_n = tile; plan->tile_k = kSimtK; plan->stages = 1;
  }
  return GK_OK;
}

// Host-side checks of the pointers a launch would dereference: a caller's mistake must come back as a
// status code, not as a device fault.
static gk_status check_pointers(const gk_gemm_desc& d, const gk_epilogue_desc* epi, const void* a, const void* b,
                                const void* c, const void* dd) {
  if (d.m == 0 || d.n == 0) return GK_OK;
  if (!dd) return set_error(GK_ERR_INVALID_ARGUMENT, "D is NULL");
  const bool product = d.k > 0 && d.alpha != 0.0 && d.layout_a != GK_LAYOUT_ZERO && d.layout_b != GK_LAYOUT_ZERO;
  if (product && !a) return set_error(GK_ERR_INVALID_ARGUMENT, "A is NULL but its layout is not Zero");
  if (product && !b) return set_error(GK_ERR_INVALID_ARGUMENT, "B is NULL but its layout is not Zero");
  if (d.layout_c != GK_LAYOUT_ZERO && d.beta != 0.0 && !c)
    return set_error(GK_ERR_INVALID_ARGUMENT, "beta = %g but C is NULL (pass C, or beta = 0 / layout_c = ZERO)", d.beta);
  if (epi && epi->bias_axis != GK_BIAS_NONE && !epi->bias)
    return set_error(GK_ERR_INVALID_ARGUMENT, "bias axis set but bias pointer is NULL");
  return GK_OK;
}

// One product of a batch (or the only one) on the kernels that have no batch index of their own.
static gk_status gemm_single(gk_handle h, const gk_gemm_desc* desc, const void* a, const void* b, const void* c,
                             void* d, const gk_epilogue_desc* epi, void* workspace, int64_t workspace_bytes,
                             cudaStream_t st);

gk_status gk_gemm(gk_handle h, const gk_gemm_desc* desc, const void* a, const void* b,
                  const void* c, void* d, const gk_epilogue_desc* epi, void* workspace,
                  int64_t workspace_bytes, gk_stream stream) {
  clear_error();
  // argument checks first (they need no device), so that a caller's mistake is reported as such
  gk_status s = validate_desc(desc, epi);
  if (s != GK_OK) return s;
  if ((s = check_pointers(*desc, epi, a, b, c, d)) != GK_OK) return s;
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return set_error(GK_ERR_INVALID_ARGUMENT, "workspace_bytes = %lld with a %s workspace", (long long)workspace_bytes,
                     workspace ? "non-NULL" : "NULL");
  if (!workspace) workspace_bytes = 0;
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  return gemm_single(h, desc, a, b, c, d, epi, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

static gk_status gemm_single(gk_handle h, const gk_gemm_desc* desc, const void* a, const void* b, const void* c,
                             void* d, const gk_epilogue_desc* epi, void* workspace, int64_t workspace_bytes,
                             cudaStream_t st) {
  gk_status s = GK_OK;
  std::string why;
  gk_gemm_desc planar = *desc;
  const SplitPlan sp = plan_split(*desc);
  if (sp.a || sp.b) {
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < sp.a_bytes + sp.b_bytes)
      return set_error(GK_ERR_INVALID_ARGUMENT,
                       "interleaved complex/dual operands are split into planes first: pass a 256-byte aligned "
                       "workspace of %lld bytes (gk_gemm_query reports it); got %lld bytes",
                       (long long)(sp.a_bytes + sp.b_bytes), (long long)workspace_bytes);
    char* ws = static_cast<char*>(workspace);
    if (sp.a) {
      s = launch_split(desc->dtype_a, a, ws, sp.a_rows, sp.a_cols, desc->lda, sp.a_ld, h->sm_count, st);
      if (s != GK_OK) return s;
      a = ws; planar.lda = sp.a_ld; planar.plane_a = sp.a_ld * sp.a_cols;
    }
    if (sp.b) {
      s = launch_split(desc->dtype_b, b, ws + sp.a_bytes, sp.b_rows, sp.b_cols, desc->ldb, sp.b_ld, h->sm_count, st);
      if (s != GK_OK) return s;
      b = ws + sp.a_bytes; planar.ldb = sp.b_ld; planar.plane_b = sp.b_ld * sp.b_cols;
    }
    desc = &planar;
  }
  bool generic_loads = false;
  int fam = choose_family(*desc, a, b, &why, &generic_loads);
  if (fam < 0) return set_error(GK_ERR_INVALID_CONFIG, "no kernel takes this GEMM: %s", why.c_str());
  if (fam == 4) return launch_diag(h, *desc, epi, a, b, c, d, st, nullptr);
  if (desc->m == 0 || desc->n == 0) return GK_OK;
  if (fam == 1 && (desc->k == 0 || desc->alpha == 0.0)) fam = 3;  // nothing to multiply
  const int batch = desc->batch > 1 ? desc->batch : 1;
  if (fam == 1) {
    TcLaunch L;
    TcProblem pr;
    tc_problem_from_gemm(*desc, epi, a, b, c, d, &pr);
    pr.generic = generic_loads;
    s = tc_plan(h, pr, true, &L);
    if (s != GK_OK) return s;
    if (L.params.debug & 8) {
      if (!workspace || workspace_bytes < static_cast<int64_t>(L.grid) * 16 * 8)
        return set_error(GK_ERR_INVALID_ARGUMENT, "debug counters need a workspace of %lld bytes",
                         (long long)L.grid * 16 * 8);
      L.params.dbg_out = static_cast<long long*>(workspace);
      return tc_launch(L, st);
    }
    return tc_run(h, pr, L, (sp.a || sp.b || batch > 1) ? nullptr : workspace, workspace_bytes, st);
  }
  // The SIMT families have no batch index: one launch per product of the batch.
  // (the FFMA kernel's vector loads need every product of a batch 16-byte aligned like the first)
  auto stride_ok = [&](int64_t stride, int dtype) { return batch == 1 || (stride * dtype_size(dtype)) % 16 == 0; };
  const bool fpu = desc->k > 0 && desc->alpha != 0.0 && fpu_eligible(*desc, a, b, c, d, epi) &&
                   stride_ok(desc->batch_stride_a, desc->dtype_a) && stride_ok(desc->batch_stride_b, desc->dtype_b) &&
                   stride_ok(desc->batch_stride_c, desc->dtype_c) && stride_ok(desc->batch_stride_d, desc->dtype_d);
  const bool f64 = !fpu && desc->k > 0 && desc->alpha != 0.0 && f64_eligible(h, *desc, a, b, c, d, epi) &&
                   stride_ok(desc->batch_stride_a, desc->dtype_a) && stride_ok(desc->batch_stride_b, desc->dtype_b) &&
                   stride_ok(desc->batch_stride_c, desc->dtype_c) && stride_ok(desc->batch_stride_d, desc->dtype_d);
  for (int i = 0; i < batch; ++i) {
    auto at = [i](const void* p, int64_t stride, int dtype) -> const void* {
      return p ? static_cast<const char*>(p) + static_cast<size_t>(i) * stride * dtype_size(dtype) : nullptr;
    };
    const void* ai = at(a, desc->batch_stride_a, desc->dtype_a);
    const void* bi = at(b, desc->batch_stride_b, desc->dtype_b);
    const void* ci = at(c, desc->batch_stride_c, desc->dtype_c);
    void* di = const_cast<void*>(at(d, desc->batch_stride_d, desc->dtype_d));
    s = fpu ? launch_fpu(h, *desc, epi, ai, bi, ci, di, st, batch == 1 ? workspace : nullptr, workspace_bytes)
        : f64 ? launch_f64(h, *desc, epi, ai, bi, ci, di, st)
              : launch_simt(*desc, epi, ai, bi, ci, di, st);
    if (s != GK_OK) return s;
  }
  return GK_OK;
}

// Bytes an operand occupies, from its first to its last addressed element.
static size_t operand_bytes(int64_t ld, int64_t cols, int64_t plane, int number, int dtype) {
  const size_t es = static_cast<size_t>(dtype_size(dtype));
  if (cols <= 0) return 0;
  if (number == GK_REAL) return static_cast<size_t>(ld) * cols * es;
  if (plane == 0) return 2 * static_cast<size_t>(ld) * cols * es;  // interleaved pairs
  return (static_cast<size_t>(plane) + static_cast<size_t>(ld) * cols) * es;
}

}  // extern "C"

namespace gk {
gk_status stage_reserve(gk_handle h, int slot, size_t bytes) {
  if (bytes <= h->stage_bytes[slot]) return GK_OK;
  if (h->stage_dev[slot]) { cudaFree(h->stage_dev[slot]); h->stage_dev[slot] = nullptr; h->stage_bytes[slot] = 0; }
  GK_CUDA_CHECK(cudaMalloc(&h->stage_dev[slot], bytes));
  h->stage_bytes[slot] = bytes;
  return GK_OK;
}

gk_status host_streams_reserve(gk_handle h, size_t n_events) {
  if (!h->copy_in) GK_CUDA_CHECK(cudaStreamCreateWithFlags(&h->copy_in, cudaStreamNonBlocking));
  if (!h->copy_out) GK_CUDA_CHECK(cudaStreamCreateWithFlags(&h->copy_out, cudaStreamNonBlocking));
  while (h->events.size() < n_events) {
    cudaEvent_t e;
    GK_CUDA_CHECK(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
    h->events.push_back(e);
  }
  return GK_OK;
}
}  // namespace gk

extern "C" {

// Block (r0.., c0..) of a column-major matrix with leading dimension ld, between host and device images
// that share the layout.
static cudaError_t copy_block(void* dst, const void* src, int64_t ld, size_t es, int64_t r0, int64_t nr, int64_t c0,
                              int64_t nc, cudaMemcpyKind kind, cudaStream_t st) {
  const size_t off = (static_cast<size_t>(c0) * ld + r0) * es;
  return cudaMemcpy2DAsync(static_cast<char*>(dst) + off, ld * es, static_cast<const char*>(src) + off, ld * es,
                           nr * es, nc, kind, st);
}

// gk_gemm_host for large real products: D is cut into row-chunk x column-chunk blocks; the chunks of A
// and B go up on one copy stream in the order the blocks need them, each block is multiplied as soon as
// its two chunks have landed, and finished blocks go back on a second copy stream, so host-to-device
// traffic, the kernels and device-to-host traffic overlap (PCIe carries both directions at once).
// Returns GK_ERR_UNSUPPORTED (without setting the error text) when the problem is too small to cut.
static gk_status gemm_host_pipelined(gk_handle h, const gk_gemm_desc& d, const void* a_host, const void* b_host,
                                     const void* c_host, void* d_host, const gk_epilogue_desc* epi, bool read_c,
                                     size_t a_bytes, size_t b_bytes, bool a_resident, cudaStream_t st) {
  // chunk size: host_chunk_mib megabytes when set (a tuning aid), else 32 MiB
  const size_t target = static_cast<size_t>(d.host_chunk_mib > 0 ? d.host_chunk_mib : 32) << 20;
  auto chunks = [target](size_t bytes) {
    const int n = static_cast<int>((bytes + target / 2) / target);
    return std::max(1, std::min(n, 8));
  };
  auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  // A already on the device: nothing of it to upload, so only the columns are cut
  const int64_t mr = a_resident ? ceil_div(d.m, 256) * 256 : ceil_div(ceil_div(d.m, chunks(a_bytes)), 256) * 256;
  const int64_t nc = ceil_div(ceil_div(d.n, chunks(b_bytes)), 512) * 512;   // columns per chunk
  const int R = static_cast<int>(ceil_div(d.m, mr)), Cn = static_cast<int>(ceil_div(d.n, nc));
  if (R * Cn <= 1) return GK_ERR_UNSUPPORTED;
  {
    const gk_status rs = host_streams_reserve(h, 2 * static_cast<size_t>(R) * Cn + 2);
    if (rs != GK_OK) return rs;
  }
  const size_t es_a = dtype_size(d.dtype_a), es_b = dtype_size(d.dtype_b), es_c = dtype_size(d.dtype_c),
               es_d = dtype_size(d.dtype_d);
  char* a_dev = a_resident ? static_cast<char*>(const_cast<void*>(a_host)) : static_cast<char*>(h->stage_dev[0]);
  char* b_dev = static_cast<char*>(h->stage_dev[1]);
  char* c_dev = static_cast<char*>(h->stage_dev[2]);
  char* d_dev = static_cast<char*>(h->stage_dev[3]);
  size_t ev = 0;
  // The copy streams start after whatever the caller queued before this call — except that with A
  // resident the uploads of B do not wait for the caller's stream (where A may still be arriving from a
  // broadcast): the kernels run on that stream and are ordered after it anyway.
  GK_CUDA_CHECK(cudaEventRecord(h->events[ev], st));
  if (!a_resident) GK_CUDA_CHECK(cudaStreamWaitEvent(h->copy_in, h->events[ev], 0));
  GK_CUDA_CHECK(cudaStreamWaitEvent(h->copy_out, h->events[ev], 0));
  ++ev;
  gk_epilogue_desc epi_blk;
  if (epi) epi_blk = *epi;
  if (epi && epi->bias_axis != GK_BIAS_NONE) {
    const size_t bias_bytes = sizeof(float) * static_cast<size_t>(epi->bias_axis == GK_BIAS_ROW ? d.m : d.n);
    GK_CUDA_CHECK(cudaMemcpyAsync(h->stage_dev[4], epi->bias, bias_bytes, cudaMemcpyHostToDevice, h->copy_in));
  }
  auto load_a = [&](int i) -> cudaError_t {
    if (a_resident) return cudaSuccess;
    const int64_t i0 = i * mr, mi = std::min<int64_t>(mr, d.m - i0);
    return d.trans_a ? copy_block(a_dev, a_host, d.lda, es_a, 0, d.k, i0, mi, cudaMemcpyHostToDevice, h->copy_in)
                     : copy_block(a_dev, a_host, d.lda, es_a, i0, mi, 0, d.k, cudaMemcpyHostToDevice, h->copy_in);
  };
  auto load_b = [&](int j) -> cudaError_t {
    const int64_t j0 = j * nc, nj = std::min<int64_t>(nc, d.n - j0);
    return d.trans_b ? copy_block(b_dev, b_host, d.ldb, es_b, j0, nj, 0, d.k, cudaMemcpyHostToDevice, h->copy_in)
                     : copy_block(b_dev, b_host, d.ldb, es_b, 0, d.k, j0, nj, cudaMemcpyHostToDevice, h->copy_in);
  };
  // One block of D: waits for everything queued on the copy-in stream so far, multiplies, sends back.
  auto block = [&](int i, int j) -> gk_status {
    const int64_t i0 = i * mr, mi = std::min<int64_t>(mr, d.m - i0);
    const int64_t j0 = j * nc, nj = std::min<int64_t>(nc, d.n - j0);
    if (read_c) GK_CUDA_CHECK(copy_block(c_dev, c_host, d.ldc, es_c, i0, mi, j0, nj, cudaMemcpyHostToDevice, h->copy_in));
    GK_CUDA_CHECK(cudaEventRecord(h->events[ev], h->copy_in));
    GK_CUDA_CHECK(cudaStreamWaitEvent(st, h->events[ev], 0));
    ++ev;
    gk_gemm_desc blk = d;
    blk.m = mi; blk.n = nj;
    if (epi && epi->bias_axis != GK_BIAS_NONE)
      epi_blk.bias = static_cast<const float*>(h->stage_dev[4]) + (epi->bias_axis == GK_BIAS_ROW ? i0 : j0);
    const size_t a_off = (d.trans_a ? static_cast<size_t>(i0) * d.lda : static_cast<size_t>(i0)) * es_a;
    const size_t b_off = (d.trans_b ? static_cast<size_t>(j0) : static_cast<size_t>(j0) * d.ldb) * es_b;
    const size_t c_off = (static_cast<size_t>(j0) * d.ldc + i0) * es_c;
    const size_t d_off = (static_cast<size_t>(j0) * d.ldd + i0) * es_d;
    const gk_status s = gk_gemm(h, &blk, a_dev + a_off, b_dev + b_off, read_c ? c_dev + c_off : nullptr, d_dev + d_off,
                                epi ? &epi_blk : nullptr, nullptr, 0, st);
    if (s != GK_OK) return s;
    GK_CUDA_CHECK(cudaEventRecord(h->events[ev], st));
    GK_CUDA_CHECK(cudaStreamWaitEvent(h->copy_out, h->events[ev], 0));
    ++ev;
    GK_CUDA_CHECK(copy_block(d_host, d_dev, d.ldd, es_d, i0, mi, j0, nj, cudaMemcpyDeviceToHost, h->copy_out));
    return GK_OK;
  };
  // Chunks go up alternately (A_0 B_0 B_1 A_1 B_2 A_2 ...): with a rows of A and b columns of B on the
  // device a*b blocks can be done, so growing both together releases blocks soonest and leaves the
  // smallest batch of blocks behind the last chunk.
  gk_status s = GK_OK;
  auto fail = [&](gk_status code) {
    cudaStreamSynchronize(h->copy_in); cudaStreamSynchronize(st); cudaStreamSynchronize(h->copy_out);
    return code;
  };
  GK_CUDA_CHECK(load_a(0));
  GK_CUDA_CHECK(load_b(0));
  if ((s = block(0, 0)) != GK_OK) return fail(s);
  for (int step = 1; step < std::max(R, Cn); ++step) {
    if (step < Cn) {
      GK_CUDA_CHECK(load_b(step));
      for (int i = 0; i < std::min(step, R); ++i)
        if ((s = block(i, step)) != GK_OK) return fail(s);
    }
    if (step < R) {
      GK_CUDA_CHECK(load_a(step));
      for (int j = 0; j <= std::min(step, Cn - 1); ++j)
        if ((s = block(step, j)) != GK_OK) return fail(s);
    }
  }
  GK_CUDA_CHECK(cudaEventRecord(h->events[ev], h->copy_out));
  GK_CUDA_CHECK(cudaStreamWaitEvent(st, h->events[ev], 0));
  GK_CUDA_CHECK(cudaStreamSynchronize(st));
  return GK_OK;
}

gk_status gk_gemm_host(gk_handle h, const gk_gemm_desc* desc, const void* a_host, const void* b_host,
                       const void* c_host, void* d_host, const gk_epilogue_desc* epi,
                       gk_stream stream) {
  clear_error();
  gk_status s = validate_desc(desc, epi);
  if (s != GK_OK) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const gk_gemm_desc& d = *desc;
  if ((s = check_pointers(d, epi, a_host, b_host, c_host, d_host)) != GK_OK) return s;
  if (d.batch > 1) return set_error(GK_ERR_INVALID_CONFIG, "gk_gemm_host takes single products (batch = %d)", d.batch);
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  const bool read_ab = d.layout_a == GK_LAYOUT_DENSE && d.layout_b == GK_LAYOUT_DENSE;
  const bool read_c = c_host != nullptr && d.layout_c == GK_LAYOUT_DENSE && d.beta != 0.0;
  const bool a_resident = d.a_resident != 0 && read_ab;   // `a_host` is a device pointer: A stays where it is
  const size_t a_bytes = read_ab && !a_resident ? operand_bytes(d.lda, d.trans_a ? d.m : d.k, d.plane_a, d.number, d.dtype_a) : 0;
  const size_t b_bytes = read_ab ? operand_bytes(d.ldb, d.trans_b ? d.k : d.n, d.plane_b, d.number, d.dtype_b) : 0;
  const size_t c_bytes = read_c ? operand_bytes(d.ldc, d.n, d.plane_c, d.number, d.dtype_c) : 0;
  const size_t d_bytes = operand_bytes(d.ldd, d.n, d.plane_d, d.number, d.dtype_d);
  size_t bias_bytes = 0;
  if (epi && epi->bias_axis != GK_BIAS_NONE)
    bias_bytes = sizeof(float) * static_cast<size_t>(epi->bias_axis == GK_BIAS_ROW ? d.m : d.n);
  std::lock_guard<std::mutex> lock(h->host_mu);  // the staging buffers are shared per handle
  const size_t need[5] = {a_bytes, b_bytes, c_bytes, d_bytes, bias_bytes};
  for (int i = 0; i < 5; ++i)
    if (need[i] && (s = stage_reserve(h, i, need[i])) != GK_OK) return s;
  if (d.number == GK_REAL && read_ab && d.m > 0 && d.n > 0 && d.k > 0 && a_bytes + b_bytes + d_bytes >= (64u << 20)) {
    s = gemm_host_pipelined(h, d, a_host, b_host, c_host, d_host, epi, read_c, a_bytes, b_bytes, a_resident, st);
    if (s == GK_OK) {
      int32_t code = 0;
      return gk_poll_status(h, &code);
    }
    if (s != GK_ERR_UNSUPPORTED) return s;
  }
  if (a_bytes) GK_CUDA_CHECK(cudaMemcpyAsync(h->stage_dev[0], a_host, a_bytes, cudaMemcpyHostToDevice, st));
  if (b_bytes) GK_CUDA_CHECK(cudaMemcpyAsync(h->stage_dev[1], b_host, b_bytes, cudaMemcpyHostToDevice, st));
  if (c_bytes) GK_CUDA_CHECK(cudaMemcpyAsync(h->stage_dev[2], c_host, c_bytes, cudaMemcpyHostToDevice, st));
  gk_epilogue_desc epi_dev;
  const gk_epilogue_desc* epi_use = epi;
  if (bias_bytes) {
    GK_CUDA_CHECK(cudaMemcpyAsync(h->stage_dev[4], epi->bias, bias_bytes, cudaMemcpyHostToDevice, st));
    epi_dev = *epi;
    epi_dev.bias = static_cast<const float*>(h->stage_dev[4]);
    epi_use = &epi_dev;
  }
  s = gk_gemm(h, desc, a_resident ? a_host : h->stage_dev[0], h->stage_dev[1], read_c ? h->stage_dev[2] : nullptr,
              h->stage_dev[3], epi_use, nullptr, 0, stream);
  if (s != GK_OK) return s;
  if (d_bytes) GK_CUDA_CHECK(cudaMemcpyAsync(d_host, h->stage_dev[3], d_bytes, cudaMemcpyDeviceToHost, st));
  GK_CUDA_CHECK(cudaStreamSynchronize(st));
  int32_t code = 0;
  return gk_poll_status(h, &code);
}

}  // extern "C"
