// Layer-level entry points of the C ABI: products with a fused epilogue (gk_gemm_fused), alone or over groups of
// columns or of K known on the device, and the activation gradient with its bias sums (gk_activation_gradient).
//
// The reference stops at one product with one epilogue; these have no counterpart there.
#include <algorithm>
#include <cstring>

#include "activation_gradient.cuh"
#include "align_operand.cuh"
#include "common.h"
#include "skinny_gemm.cuh"
#include "tc_plan.h"

namespace gk {

static int fused_dtype(int32_t dt) { return dt == GK_F16 ? TC_F16 : dt == GK_BF16 ? TC_BF16 : dt == GK_F32 ? TC_F32 : -1; }

static gk_status check_offsets(int32_t groups, int32_t offsets_dtype, const void* offsets) {
  if (groups < 1 || groups > GK_MAX_GROUPS)
    return set_error(GK_ERR_INVALID_CONFIG, "groups must be between 1 and %d, got %d", GK_MAX_GROUPS, groups);
  if (!offsets) return set_error(GK_ERR_INVALID_ARGUMENT, "offsets is NULL");
  if (offsets_dtype != GK_I32 && offsets_dtype != GK_I64)
    return set_error(GK_ERR_UNSUPPORTED, "offsets must be Int32 or Int64");
  if (reinterpret_cast<uintptr_t>(offsets) % dtype_size(offsets_dtype))
    return set_error(GK_ERR_INVALID_ARGUMENT, "offsets is not aligned to its element type");
  return GK_OK;
}

// Everything that can be refused without looking at the device.
static gk_status validate_fused(const gk_gemm_desc* d, const gk_fused_desc* fu, const gk_group_desc* gr) {
  gk_status s = validate_desc(d, nullptr);
  if (s != GK_OK) return s;
  if (!fu) return set_error(GK_ERR_INVALID_ARGUMENT, "fused descriptor is NULL");
  if (fu->struct_size != sizeof(gk_fused_desc))
    return set_error(GK_ERR_INVALID_ARGUMENT, "gk_fused_desc.struct_size is %u, this library expects %zu", fu->struct_size, sizeof(gk_fused_desc));
  if (gr && gr->struct_size != sizeof(gk_group_desc))
    return set_error(GK_ERR_INVALID_ARGUMENT, "gk_group_desc.struct_size is %u, this library expects %zu", gr->struct_size, sizeof(gk_group_desc));
  if (d->number != GK_REAL || d->batch > 1 || d->debug != 0 || (d->op != GK_OP_AUTO && d->op != GK_OP_TCGEN05))
    return set_error(GK_ERR_INVALID_CONFIG, "fused and ragged products are single real products of the TCGen05Operator, without diagnostic bits");
  if (d->layout_a != GK_LAYOUT_DENSE || d->layout_b != GK_LAYOUT_DENSE || (d->layout_c != GK_LAYOUT_DENSE && d->layout_c != GK_LAYOUT_ZERO))
    return set_error(GK_ERR_INVALID_CONFIG, "fused and ragged products take dense operands (and a dense or Zero C)");
  const bool f16 = d->dtype_a == GK_F16 && d->compute == GK_F16, bf16 = d->dtype_a == GK_BF16 && d->compute == GK_BF16;
  if (d->dtype_a != d->dtype_b || !(f16 || bf16))
    return set_error(GK_ERR_INVALID_CONFIG, "fused and ragged products multiply Float16 or BFloat16 operands (A is %s, B is %s, compute %s)",
                     dtype_name(d->dtype_a), dtype_name(d->dtype_b), dtype_name(d->compute));
  if (fused_dtype(d->dtype_d) < 0)
    return set_error(GK_ERR_INVALID_CONFIG, "D must be Float16, BFloat16 or Float32, not %s", dtype_name(d->dtype_d));
  const bool has_c = d->layout_c == GK_LAYOUT_DENSE && d->beta != 0.0;
  if (has_c && d->dtype_c != d->dtype_d)
    return set_error(GK_ERR_INVALID_CONFIG, "C (%s) must have the element type of D (%s)", dtype_name(d->dtype_c), dtype_name(d->dtype_d));
  if (d->m > INT32_MAX / 2 || d->n > INT32_MAX / 2 || d->k > INT32_MAX / 2) return set_error(GK_ERR_INVALID_CONFIG, "dimension too large");
  if (fu->form < GK_FUSED_STANDARD || fu->form > GK_FUSED_GRADIENT) return set_error(GK_ERR_UNSUPPORTED, "epilogue form %d is unknown", fu->form);
  if (fu->bias_axis < GK_BIAS_NONE || fu->bias_axis > GK_BIAS_COL)
    return set_error(GK_ERR_UNSUPPORTED, "bias axis %d is not none/row/column", fu->bias_axis);
  if (fu->activation < GK_ACT_NONE || fu->activation > GK_ACT_SILU)
    return set_error(GK_ERR_UNSUPPORTED, "activation %d is not one of none/ReLU/GELU/SiLU", fu->activation);
  if (fu->form == GK_FUSED_GRADIENT && fu->bias_axis != GK_BIAS_NONE)
    return set_error(GK_ERR_INVALID_CONFIG, "the gradient form takes no bias");
  if (fu->z && fu->ldz < std::max<int64_t>(d->m, 1))
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: ldz = %lld < M = %lld", (long long)fu->ldz, (long long)d->m);
  if (!gr) return GK_OK;
  if (gr->ragged != GK_RAGGED_COLUMNS && gr->ragged != GK_RAGGED_DEPTH) return set_error(GK_ERR_UNSUPPORTED, "ragged = %d is unknown", gr->ragged);
  if ((s = check_offsets(gr->groups, gr->offsets_dtype, gr->offsets)) != GK_OK) return s;
  if (gr->stride_a < 0 || gr->stride_c < 0 || gr->stride_d < 0 || gr->stride_bias < 0)
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: negative group stride");
  if (gr->ragged == GK_RAGGED_COLUMNS) {
    if (fu->bias_axis == GK_BIAS_COL) return set_error(GK_ERR_INVALID_CONFIG, "grouped products take one bias per row of each group");
  } else {
    if (fu->form != GK_FUSED_STANDARD || fu->bias_axis != GK_BIAS_NONE || fu->activation != GK_ACT_NONE || fu->z)
      return set_error(GK_ERR_INVALID_CONFIG, "products with a ragged depth take alpha, beta and C only");
    if (gr->groups > 1 && d->m > 0 && d->n > 0 && gr->stride_d < d->ldd * (d->n - 1) + d->m)
      return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: stride_d = %lld makes the outputs of the groups overlap", (long long)gr->stride_d);
  }
  return GK_OK;
}

static bool off_element(const void* p, int32_t dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) != 0; }

static gk_status check_fused_pointers(const gk_gemm_desc& d, const gk_fused_desc& fu, const gk_group_desc* gr, const void* a, const void* b,
                                      const void* c, const void* dd) {
  if (d.m == 0 || d.n == 0) return GK_OK;
  if (!dd) return set_error(GK_ERR_INVALID_ARGUMENT, "D is NULL");
  if (d.k > 0 && d.alpha != 0.0 && (!a || !b)) return set_error(GK_ERR_INVALID_ARGUMENT, "%s is NULL", a ? "B" : "A");
  if (d.layout_c == GK_LAYOUT_DENSE && d.beta != 0.0 && !c)
    return set_error(GK_ERR_INVALID_ARGUMENT, "beta = %g but C is NULL (pass C, or beta = 0 / layout_c = ZERO)", d.beta);
  if (fu.bias_axis != GK_BIAS_NONE && !fu.bias) return set_error(GK_ERR_INVALID_ARGUMENT, "bias axis set but bias pointer is NULL");
  if (fu.form == GK_FUSED_GRADIENT && !fu.z) return set_error(GK_ERR_INVALID_ARGUMENT, "the gradient form needs Z");
  if (fu.form != GK_FUSED_GRADIENT && fu.z && (fu.z == dd || fu.z == c))
    return set_error(GK_ERR_INVALID_ARGUMENT, "Z is kept beside D: it cannot share memory with D or C");
  const bool has_c = d.layout_c == GK_LAYOUT_DENSE && d.beta != 0.0;
  if (off_element(a, d.dtype_a) || off_element(b, d.dtype_b) || off_element(dd, d.dtype_d) || (has_c && off_element(c, d.dtype_c)) ||
      off_element(fu.z, d.dtype_d) || (fu.bias_axis != GK_BIAS_NONE && off_element(fu.bias, GK_F32)))
    return set_error(GK_ERR_INVALID_ARGUMENT, "an array is not aligned to its element type");
  // In place, every element is read and written by one thread: the two must be laid out alike.
  const bool depth = gr && gr->ragged == GK_RAGGED_DEPTH && gr->groups > 1;
  if ((has_c && c == dd && (d.ldc != d.ldd || (depth && gr->stride_c != gr->stride_d))) || (fu.z == dd && fu.ldz != d.ldd))
    return set_error(GK_ERR_INVALID_ARGUMENT, "C or Z in place of D must have D's leading dimension and strides");
  return GK_OK;
}

// The tensor-core problem of a validated call.
static void fused_problem(const gk_gemm_desc& d, const gk_fused_desc& fu, const gk_group_desc* gr, const gk_epilogue_desc* epi,
                          const void* a, const void* b, const void* c, void* dd, TcProblem* out) {
  tc_problem_from_gemm(d, epi, a, b, c, dd, out);
  TcProblem& pr = *out;
  pr.form = !gr ? kTcFused : gr->ragged == GK_RAGGED_COLUMNS ? kTcRaggedCols : kTcRaggedDepth;
  pr.f.form = fu.form; pr.f.Z = fu.z; pr.f.z_sn = fu.ldz; pr.f.dtype_z = fused_dtype(d.dtype_d);
  pr.f.groups = 1; pr.f.total = static_cast<int32_t>(pr.form == kTcRaggedDepth ? d.k : d.n);
  if (gr) {
    pr.f.groups = gr->groups; pr.f.offsets = gr->offsets; pr.f.offsets64 = gr->offsets_dtype == GK_I64 ? 1 : 0;
    pr.f.bias_group = gr->stride_bias;
    if (pr.form == kTcRaggedCols) pr.batch_a = gr->stride_a;
    else { pr.batch_c = gr->stride_c; pr.batch_d = gr->stride_d; }
  }
  if (d.alpha == 0.0) {      // nothing to multiply: A and B are not read
    pr.K = 0;
    if (pr.form == kTcRaggedDepth) pr.f.total = 0;
  }
}

// How a tensor-core product gets at its operands.  TMA takes 16-byte aligned columns (and, along a ragged depth, only
// operands whose K is the strided index: a group's run may start anywhere); an operand that is not aligned is copied
// with padded columns into the workspace first.  Without the room for that, or with the wrong order along a ragged depth,
// the generic instances read the operands with bounds-checked loads.
struct OperandCopy { bool copy = false; int64_t rows = 0, cols = 0, ld = 0, group = 0, bytes = 0; int32_t groups = 1; };
struct FusedFeed {
  bool possible = true;            // TMA can be used once the copies are made
  OperandCopy a, b;
  int64_t bytes() const { return a.bytes + b.bytes; }
};

static FusedFeed fused_feed(const gk_gemm_desc& d, const gk_group_desc* gr, const void* a, const void* b) {
  FusedFeed f;
  if (gr && gr->ragged == GK_RAGGED_DEPTH && (d.trans_a || !d.trans_b)) { f.possible = false; return f; }
  if (d.k < 1 || d.alpha == 0.0) return f;      // nothing is loaded
  const bool cols = gr && gr->ragged == GK_RAGGED_COLUMNS;
  auto plan = [&](OperandCopy& c, const void* p, int64_t ld, bool trans, int64_t mn, bool is_a) {
    const int64_t stride = is_a && cols && gr->groups > 1 ? gr->stride_a : 0;
    c.copy = (reinterpret_cast<uintptr_t>(p) & 15) || ld % 8 || stride % 8;
    if (!c.copy) return;
    // stored rows x columns: op(A) is M x K, op(B) is K x N
    c.rows = trans == is_a ? d.k : mn; c.cols = trans == is_a ? mn : d.k;
    c.ld = (c.rows + 7) / 8 * 8; c.groups = stride > 0 ? gr->groups : 1; c.group = c.ld * c.cols;
    c.bytes = (c.group * c.groups * 2 + 255) / 256 * 256;
  };
  plan(f.a, a, d.lda, d.trans_a != 0, d.m, true);
  plan(f.b, b, d.ldb, d.trans_b != 0, d.n, false);
  return f;
}

static gk_status launch_copy(gk_handle h, const OperandCopy& c, const void* src, int64_t ld, int64_t stride, void* dst, const FusedParams& f,
                             bool skip_empty, cudaStream_t stream) {
  AlignParams p{};
  p.src = static_cast<const uint16_t*>(src); p.dst = static_cast<uint16_t*>(dst);
  p.ld = ld; p.group = c.groups > 1 ? stride : 0; p.ld_dst = c.ld; p.group_dst = c.group;
  p.rows = static_cast<int32_t>(c.rows); p.cols = static_cast<int32_t>(c.cols);
  p.skip_empty = skip_empty ? 1 : 0;
  p.f = f;
  const int per_block = kAlignThreads / 32;
  const int64_t want = std::max<int64_t>(1, 16 * static_cast<int64_t>(h->sm_count) / c.groups);
  const int64_t units = (c.ld / 8 + 31) / 32 * c.cols;      // a warp's share: 256 rows of a column
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((units + per_block - 1) / per_block, want));
  GK_CUDA_CHECK(launch_dependent(&align_operand_kernel, dim3(blocks, static_cast<unsigned>(c.groups)), dim3(kAlignThreads), 0, stream, p));
  return GK_OK;
}

// ------------------------------------------------------------------------------------------------
// a few columns: the streaming kernel
// ------------------------------------------------------------------------------------------------
// How the columns fall on the groups is known on the device only.  At this size the streaming kernel and the tensor cores are even
// when all columns fall on one group, whose weights the tensor cores read once, and streaming is ahead when they are spread
// (us, streaming / tensor cores; transposed A of 2048 x 2048, 64 groups: 8 columns spread 11.8 / 16.0, on one group 10.1 /
// 12.0; 16 columns 22.5 / 25.9 and 15.2 / 11.8; 32 columns 37.3 / 38.0 and 25.9 / 12.0; 64 columns 62.8 / 57.3 and 45.3 / 12.0.
// 256 groups of 1024 x 1024, 64 columns: 25.9 / 38.6 and 16.8 / 15.8.  8 groups of 4096 x 4096, 4 columns: 24.7 / 26.5
// and 15.5 / 16.1.  Operands off 16 bytes, 64 groups of 2047 x 2049, 16 columns: 87 / 143 and 59 / 66, 32 columns: 170 / 165
// and 110 / 68).
constexpr int64_t kSkinnyGroupBytes = 1 << 27;

struct SkinnyPlan { int nt = 0, ranks = 1, items = 0, rows = 0, k_per_rank = 0; bool any = false; };

static bool skinny_plan(gk_handle h, const gk_gemm_desc& d, const gk_group_desc* gr, const void* a, const void* b, int64_t group_bytes,
                        SkinnyPlan* out) {
  if (gr && gr->ragged != GK_RAGGED_COLUMNS) return false;
  if (d.tile_n || d.cta_group || d.stages || d.max_ctas) return false;      // a tensor-core tile was asked for
  if (d.k < 1 || d.alpha == 0.0 || d.n < 1 || d.m < 1) return false;
  const int64_t groups = gr ? gr->groups : 1;
  const int64_t active = std::min<int64_t>(groups, d.n);
  if (d.n > 4096) return false;
  SkinnyPlan p;
  auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  p.any = !al(a) || !al(b) || d.lda % 8 || d.ldb % 8 || d.k % 8 || (!d.trans_a && d.m % 8) || d.trans_b ||
          (gr && groups > 1 && gr->stride_a % 8);
  // Groups: one column at a time, while there are no more of them than groups and what they stream, counting a group's weights
  // once for each of its columns, stays below `group_bytes`.  One product: up to 16 columns of a
  // transposed A (4096 x 4096, 8 columns: 11.0 us, 16.1 with tcgen05; 16: 13.0 and 16.2), else up to eight (12.4 and
  // 16.3-17.2), of these with FMAs up to four (2048 x 2048, 4 columns: 6.0 us, 7.1 with warp-level matrix instructions; 4096 x
  // 4096: 11.6 and 11.8) and up to four in all where 16-byte loads do not serve.
  const int mma = groups != 1 || p.any ? 0 : d.trans_a ? (d.n > 1 ? kSkinnyMmaCols : 0) : (d.n > 4 ? kSkinnyMmaRowsCols : 0);
  if (d.n > (groups > 1 ? active : mma ? mma : 4)) return false;
  if (groups > 1 && d.n > 1 && 2 * d.m * d.k > group_bytes / d.n) return false;
  p.nt = d.n <= active ? 1 : mma ? mma : (d.n <= 2 ? 2 : 4);
  p.items = static_cast<int>(std::min<int64_t>(d.n, d.n / p.nt + active));
  if (groups == 1) p.items = static_cast<int>((d.n + p.nt - 1) / p.nt);
  p.rows = static_cast<int>((d.m + kSkinnyRows - 1) / kSkinnyRows);
  // K is cut as far as the CTAs still run in one round.
  const int ctas = p.nt == kSkinnyMmaCols ? kSkinnyMmaCtas : p.nt == kSkinnyMmaRowsCols ? kSkinnyMmaRowsCtas : skinny_ctas(p.nt, p.any);
  const int64_t slots = static_cast<int64_t>(ctas) * h->sm_count;
  const int64_t steps = (d.k + kSkinnyStep - 1) / kSkinnyStep;
  while (p.ranks < 8 && 2 * p.ranks <= steps && 2 * static_cast<int64_t>(p.rows) * p.items * p.ranks <= slots) p.ranks *= 2;
  p.k_per_rank = static_cast<int>((steps + p.ranks - 1) / p.ranks * kSkinnyStep);
  *out = p;
  return true;
}

template <typename T, bool K_MAJOR, bool ANY>
static const void* skinny_kernel_nt(int nt) {
  return nt == 1   ? reinterpret_cast<const void*>(&skinny_gemm_kernel<T, K_MAJOR, 1, ANY>)
         : nt == 2 ? reinterpret_cast<const void*>(&skinny_gemm_kernel<T, K_MAJOR, 2, ANY>)
                   : reinterpret_cast<const void*>(&skinny_gemm_kernel<T, K_MAJOR, 4, ANY>);
}

template <typename T>
static const void* skinny_kernel(bool k_major, bool any, int nt) {
  if (nt == kSkinnyMmaCols) return reinterpret_cast<const void*>(&skinny_mma_kernel<T>);
  if (nt == kSkinnyMmaRowsCols) return reinterpret_cast<const void*>(&skinny_mma_rows_kernel<T>);
  if (k_major) return any ? skinny_kernel_nt<T, true, true>(nt) : reinterpret_cast<const void*>(&skinny_gemm_kernel<T, true, 1, false>);
  return any ? skinny_kernel_nt<T, false, true>(nt) : skinny_kernel_nt<T, false, false>(nt);
}

static gk_status launch_skinny(const SkinnyPlan& sp, const gk_gemm_desc& d, const gk_fused_desc& fu, const gk_group_desc* gr,
                               const TcProblem& pr, const void* a, const void* b, const void* c, void* dd, cudaStream_t stream) {
  SkinnyParams p{};
  p.A = a; p.B = b; p.C = c; p.D = dd;
  p.M = static_cast<int32_t>(d.m); p.K = static_cast<int32_t>(d.k);
  p.lda = d.lda; p.ldc = d.ldc; p.ldd = d.ldd;
  p.b_sk = d.trans_b ? d.ldb : 1; p.b_sn = d.trans_b ? 1 : d.ldb;
  p.a_group = gr ? gr->stride_a : 0;
  p.alpha = static_cast<float>(d.alpha);
  p.beta = d.layout_c == GK_LAYOUT_DENSE ? static_cast<float>(d.beta) : 0.0f;
  p.bias = fu.bias; p.bias_axis = fu.bias_axis; p.act = fu.activation;
  p.dtype_d = fused_dtype(d.dtype_d);
  p.k_per_rank = sp.k_per_rank;
  p.f = pr.f;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sp.rows * sp.ranks), static_cast<unsigned>(sp.items));
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(sp.ranks); at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = sp.ranks > 1 ? 2 : 1;
  void* args[1] = {&p};
  const void* kernel = d.dtype_a == GK_F16 ? skinny_kernel<__half>(d.trans_a != 0, sp.any, sp.nt)
                                            : skinny_kernel<__nv_bfloat16>(d.trans_a != 0, sp.any, sp.nt);
  GK_CUDA_CHECK(cudaLaunchKernelExC(&cfg, kernel, args));
  return GK_OK;
}

// ------------------------------------------------------------------------------------------------
// activation gradient
// ------------------------------------------------------------------------------------------------
struct ActGradPlan { int rows = 0, strips = 0, strip = 0, per_group = 0; int64_t bytes = 0; };

static gk_status validate_actgrad(const gk_activation_gradient_desc* d) {
  if (!d) return set_error(GK_ERR_INVALID_ARGUMENT, "descriptor is NULL");
  if (d->struct_size != sizeof(gk_activation_gradient_desc))
    return set_error(GK_ERR_INVALID_ARGUMENT, "gk_activation_gradient_desc.struct_size is %u, this library expects %zu", d->struct_size,
                     sizeof(gk_activation_gradient_desc));
  if (d->m < 0 || d->n < 0) return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: negative extent (%lld, %lld)", (long long)d->m, (long long)d->n);
  if (d->m > INT32_MAX / 2 || d->n > INT32_MAX / 2) return set_error(GK_ERR_INVALID_CONFIG, "dimension too large");
  if (fused_dtype(d->dtype) < 0) return set_error(GK_ERR_UNSUPPORTED, "the activation gradient takes Float16, BFloat16 or Float32, not %s", dtype_name(d->dtype));
  if (d->activation < GK_ACT_NONE || d->activation > GK_ACT_SILU)
    return set_error(GK_ERR_UNSUPPORTED, "activation %d is not one of none/ReLU/GELU/SiLU", d->activation);
  const int64_t least = std::max<int64_t>(d->m, 1);
  if (d->ld_dd < least || (d->activation != GK_ACT_NONE && d->ld_z < least) || d->ld_dz < least || d->ld_db < least)
    return set_error(GK_ERR_DIMENSION_MISMATCH, "Dimensions do not match: a leading dimension is below M = %lld", (long long)d->m);
  if (d->groups < 1 || d->groups > GK_MAX_GROUPS)
    return set_error(GK_ERR_INVALID_CONFIG, "groups must be between 1 and %d, got %d", GK_MAX_GROUPS, d->groups);
  if (d->offsets) return check_offsets(d->groups, d->offsets_dtype, d->offsets);
  if (d->groups != 1) return set_error(GK_ERR_INVALID_ARGUMENT, "offsets is NULL but there are %d groups", d->groups);
  return GK_OK;
}

static ActGradPlan actgrad_plan(int sm_count, const gk_activation_gradient_desc& d, bool sums) {
  ActGradPlan p;
  p.rows = static_cast<int>((d.m + kActGradRows - 1) / kActGradRows);
  // Strips long enough to amortise their reduction, short enough for eight CTAs per SM.
  const int64_t want = (d.n * p.rows + 8 * sm_count - 1) / (8 * sm_count);
  int64_t strip = std::max<int64_t>(128, std::min<int64_t>(2048, (want + 127) / 128 * 128));
  // A short matrix is summed by one CTA per group and 64 rows: a second launch costs more than it spreads.
  p.per_group = sums && d.n <= 512 ? 1 : 0;
  const int64_t active = std::min<int64_t>(d.groups, d.n);
  int64_t strips = d.n / strip + active;
  while (strips > 65535) { strip *= 2; strips = d.n / strip + active; }
  p.strip = static_cast<int>(strip);
  p.strips = static_cast<int>(p.per_group ? d.groups : strips);
  if (sums && !p.per_group) p.bytes = static_cast<int64_t>(p.strips) * d.m * 4;
  return p;
}

template <typename T, int VEC>
static void (*actgrad_kernel(int act))(const ActGradParams) {
  switch (act) {
    case GK_ACT_RELU: return activation_gradient_kernel<T, VEC, FUSED_ACT_RELU>;
    case GK_ACT_GELU: return activation_gradient_kernel<T, VEC, FUSED_ACT_GELU>;
    case GK_ACT_SILU: return activation_gradient_kernel<T, VEC, FUSED_ACT_SILU>;
    default: return activation_gradient_kernel<T, VEC, FUSED_ACT_NONE>;
  }
}

}  // namespace gk

using namespace gk;

extern "C" {

gk_status gk_gemm_fused_query(gk_handle h, const gk_gemm_desc* desc, const gk_fused_desc* fused, const gk_group_desc* groups,
                              gk_gemm_plan* plan) {
  clear_error();
  if (!plan) return set_error(GK_ERR_INVALID_ARGUMENT, "plan is NULL");
  gk_status s = validate_fused(desc, fused, groups);
  if (s != GK_OK) return s;
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  std::memset(plan, 0, sizeof(*plan));
  if (desc->m == 0 || desc->n == 0) return GK_OK;
  SkinnyPlan sp;
  if (skinny_plan(h, *desc, groups, nullptr, nullptr, kSkinnyGroupBytes, &sp)) {
    plan->kernel = 6; plan->grid = sp.rows * sp.ranks * sp.items; plan->block = kSkinnyThreads; plan->cluster = sp.ranks;
    plan->tile_m = kSkinnyRows; plan->tile_n = sp.nt; plan->tile_k = kSkinnyStep; plan->stages = 1;
  }
  gk_epilogue_desc epi{sizeof(gk_epilogue_desc), fused->bias_axis, fused->bias, fused->activation, {0, 0, 0}};
  TcProblem pr;
  fused_problem(*desc, *fused, groups, &epi, nullptr, nullptr, nullptr, nullptr, &pr);
  const FusedFeed feed = fused_feed(*desc, groups, nullptr, nullptr);
  pr.generic = !feed.possible;
  TcLaunch L;
  if ((s = tc_plan(h, pr, false, &L)) != GK_OK) return s;
  if (plan->kernel == 0) {
    plan->kernel = 1; plan->grid = L.grid; plan->block = tc_threads(1); plan->cluster = L.cg;
    plan->smem_bytes = L.smem_bytes; plan->tmem_columns = static_cast<int32_t>(L.params.tmem_cols);
    plan->tile_m = kTcTileM * L.cg; plan->tile_n = L.params.bn * L.params.n_sub; plan->tile_k = L.params.bk * L.params.kps;
    plan->stages = L.params.stages;
    plan->workspace_bytes = feed.bytes() + (pr.form == kTcFused && pr.K > 0 ? tc_split_workspace_bytes(h, pr, L) : tc_depth_maps_bytes(L));
  }
  return GK_OK;
}

gk_status gk_gemm_fused(gk_handle h, const gk_gemm_desc* desc, const gk_fused_desc* fused, const gk_group_desc* groups,
                        const void* a, const void* b, const void* c, void* d, void* workspace, int64_t workspace_bytes,
                        gk_stream stream) {
  clear_error();
  gk_status s = validate_fused(desc, fused, groups);
  if (s != GK_OK) return s;
  if ((s = check_fused_pointers(*desc, *fused, groups, a, b, c, d)) != GK_OK) return s;
  if (workspace_bytes < 0 || (workspace_bytes > 0 && !workspace))
    return set_error(GK_ERR_INVALID_ARGUMENT, "workspace_bytes = %lld with a %s workspace", (long long)workspace_bytes, workspace ? "non-NULL" : "NULL");
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  if (desc->m == 0 || desc->n == 0) return GK_OK;
  if (!workspace) workspace_bytes = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  gk_epilogue_desc epi{sizeof(gk_epilogue_desc), fused->bias_axis, fused->bias, fused->activation, {0, 0, 0}};
  TcProblem pr;
  fused_problem(*desc, *fused, groups, &epi, a, b, desc->beta != 0.0 ? c : nullptr, d, &pr);
  SkinnyPlan sp;
  if (skinny_plan(h, *desc, groups, a, b, kSkinnyGroupBytes, &sp)) return launch_skinny(sp, *desc, *fused, groups, pr, a, b, c, d, st);
  const FusedFeed feed = fused_feed(*desc, groups, a, b);
  const int64_t copies = feed.bytes();
  // A ragged depth multiplies copies through tensor maps, which need their room behind them: decided before anything is enqueued.
  const int64_t maps = pr.form == kTcRaggedDepth ? static_cast<int64_t>(groups->groups) * kTcDepthMapsBytes : 0;
  pr.generic = !feed.possible || (copies > 0 && (workspace_bytes < copies + maps || (reinterpret_cast<uintptr_t>(workspace) & 255)));
  // Few columns of unaligned operands without room for their copies stream whatever their number per group (64 groups of
  // 2047 x 2049, 32 columns spread: 170 us, bounds-checked loads 2056; on one group 110 and 301).
  if (pr.generic && skinny_plan(h, *desc, groups, a, b, INT64_MAX, &sp)) return launch_skinny(sp, *desc, *fused, groups, pr, a, b, c, d, st);
  if (!pr.generic && copies > 0) {
    char* ws = static_cast<char*>(workspace);
    gk_gemm_desc e = *desc;
    gk_group_desc eg;
    if (groups) eg = *groups;
    if (feed.a.copy) {
      if ((s = launch_copy(h, feed.a, a, desc->lda, groups ? groups->stride_a : 0, ws, pr.f, feed.a.groups > 1, st)) != GK_OK) return s;
      a = ws; e.lda = feed.a.ld; eg.stride_a = feed.a.groups > 1 ? feed.a.group : 0;
    }
    if (feed.b.copy) {
      if ((s = launch_copy(h, feed.b, b, desc->ldb, 0, ws + feed.a.bytes, pr.f, false, st)) != GK_OK) return s;
      b = ws + feed.a.bytes; e.ldb = feed.b.ld;
    }
    workspace = ws + copies; workspace_bytes -= copies;
    fused_problem(e, *fused, groups ? &eg : nullptr, &epi, a, b, desc->beta != 0.0 ? c : nullptr, d, &pr);
  }
  TcLaunch L;
  if ((s = tc_plan(h, pr, true, &L)) != GK_OK) return s;
  if (pr.form == kTcFused) return pr.K > 0 ? tc_run(h, pr, L, workspace, workspace_bytes, st) : tc_launch(L, st);
  const int64_t need = tc_depth_maps_bytes(L);
  if (need > 0) {
    if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
      return set_error(GK_ERR_INVALID_ARGUMENT, "products with a ragged depth need a 256-byte aligned workspace of %lld bytes "
                       "(gk_gemm_fused_query reports it); got %lld bytes", (long long)need, (long long)workspace_bytes);
    if ((s = tc_write_depth_maps(&L, workspace, st)) != GK_OK) return s;
  }
  return tc_launch(L, st);
}

gk_status gk_activation_gradient_query(gk_handle h, const gk_activation_gradient_desc* desc, int64_t* workspace_bytes) {
  clear_error();
  if (!workspace_bytes) return set_error(GK_ERR_INVALID_ARGUMENT, "workspace_bytes is NULL");
  gk_status s = validate_actgrad(desc);
  if (s != GK_OK) return s;
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  *workspace_bytes = actgrad_plan(h->sm_count, *desc, true).bytes;
  return GK_OK;
}

gk_status gk_activation_gradient(gk_handle h, const gk_activation_gradient_desc* desc, const void* dd, const void* z, void* dz,
                                 float* db, void* workspace, int64_t workspace_bytes, gk_stream stream) {
  clear_error();
  gk_status s = validate_actgrad(desc);
  if (s != GK_OK) return s;
  if (!dz && !db) return set_error(GK_ERR_INVALID_ARGUMENT, "neither dZ nor the bias gradient is wanted");
  if (desc->n > 0 && desc->m > 0 && !dd) return set_error(GK_ERR_INVALID_ARGUMENT, "dD is NULL");
  if (desc->n > 0 && desc->m > 0 && desc->activation != GK_ACT_NONE && !z) return set_error(GK_ERR_INVALID_ARGUMENT, "Z is NULL");
  if (off_element(dd, desc->dtype) || off_element(z, desc->dtype) || off_element(dz, desc->dtype) || off_element(db, GK_F32))
    return set_error(GK_ERR_INVALID_ARGUMENT, "an array is not aligned to its element type");
  if (dz && ((dz == dd && desc->ld_dz != desc->ld_dd) || (dz == z && desc->ld_dz != desc->ld_z)))
    return set_error(GK_ERR_INVALID_ARGUMENT, "dZ in place of dD or Z must have its leading dimension");
  if (!h) return set_error(GK_ERR_INVALID_ARGUMENT, "handle is NULL");
  if (desc->m == 0 || (desc->n == 0 && !db)) return GK_OK;
  const ActGradPlan pl = actgrad_plan(h->sm_count, *desc, db != nullptr);
  if (workspace_bytes < pl.bytes || (pl.bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3))))
    return set_error(GK_ERR_INVALID_ARGUMENT, "the bias gradient needs a workspace of %lld bytes (gk_activation_gradient_query "
                     "reports it); got %lld bytes", (long long)pl.bytes, (long long)workspace_bytes);
  ActGradParams p{};
  p.dD = dd; p.Z = z; p.dZ = dz; p.db = db;
  p.partial = pl.bytes > 0 ? static_cast<float*>(workspace) : nullptr;
  p.M = static_cast<int32_t>(desc->m); p.act = desc->activation;
  p.ldd = desc->ld_dd; p.ldz = desc->ld_z; p.lddz = desc->ld_dz; p.lddb = desc->ld_db;
  p.strip = pl.strip; p.per_group = pl.per_group;
  p.f.offsets = desc->offsets; p.f.offsets64 = desc->offsets_dtype == GK_I64 ? 1 : 0;
  p.f.groups = desc->groups; p.f.total = static_cast<int32_t>(desc->n);
  const int es = dtype_size(desc->dtype), vec = 16 / es;
  auto ok = [&](const void* q, int64_t ld) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ld % vec == 0; };
  const bool wide = desc->m % vec == 0 && ok(dd, desc->ld_dd) && (desc->activation == GK_ACT_NONE || ok(z, desc->ld_z)) &&
                    (!dz || ok(dz, desc->ld_dz));
  void (*kernel)(const ActGradParams) =
      desc->dtype == GK_F16    ? (wide ? actgrad_kernel<__half, 8>(p.act) : actgrad_kernel<__half, 1>(p.act))
      : desc->dtype == GK_BF16 ? (wide ? actgrad_kernel<__nv_bfloat16, 8>(p.act) : actgrad_kernel<__nv_bfloat16, 1>(p.act))
                               : (wide ? actgrad_kernel<float, 4>(p.act) : actgrad_kernel<float, 1>(p.act));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pl.strips > 0)
    GK_CUDA_CHECK(launch_dependent(kernel, dim3(pl.rows, pl.strips), dim3(kActGradThreads), 0, st, p));
  if (db && !pl.per_group)
    GK_CUDA_CHECK(launch_dependent(&bias_gradient_sum_kernel, dim3((p.M + kActGradThreads - 1) / kActGradThreads, p.f.groups),
                                   dim3(kActGradThreads), 0, st, p));
  return GK_OK;
}

}  // extern "C"
