// The epilogues of the layer-level products (gk_gemm_fused), shared by the tensor-core kernel, the split-K
// reduction and the streaming kernel for a few columns, and the column groups of ragged products.
//
//   x = alpha * (op(A) op(B))(m, n) + bias            (+ beta * C(m, n) in the STANDARD and GRADIENT forms)
//   STANDARD   Z = x (kept on request)    D = act(x)
//   RESIDUAL   Z = x (kept on request)    D = act(x) + beta * C
//   GRADIENT   Z is read                  D = x * act'(Z)
//
// x, act and act' are FP32; D and Z are rounded once, when they are stored (act sees the unrounded x).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace gk {

enum FusedForm : int32_t { FUSED_STANDARD = 0, FUSED_RESIDUAL = 1, FUSED_GRADIENT = 2 };
enum FusedAct : int32_t { FUSED_ACT_NONE = 0, FUSED_ACT_RELU = 1, FUSED_ACT_GELU = 2, FUSED_ACT_SILU = 3 };

// What the fused forms of a kernel need beside C, D, alpha, beta, bias and act of the plain ones.
struct FusedParams {
  int32_t form;
  int32_t dtype_z;
  void* Z;                 // written (STANDARD, RESIDUAL; NULL: not kept) or read (GRADIENT)
  int64_t z_sn;            // elements between the columns of Z
  // column groups (ragged products): group g holds the columns offsets[g] .. offsets[g + 1] - 1
  const void* offsets;     // device, groups + 1 values; NULL: one group of all `total` columns
  int32_t offsets64;       // 0: 32-bit values, 1: 64-bit values
  int32_t groups;
  int32_t total;           // columns there are: offsets are clamped to [0, total]
  int64_t bias_group;      // elements between the biases of consecutive groups
};

// A NaN passes through all activations; at minus infinity GELU and SiLU have their limit 0 (the factor that multiplies what
// has run out to zero is clamped), as their derivatives have 0 and 1.
__device__ __forceinline__ float fused_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fused_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fused_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fused_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 fused_2(float x) { return make_float2(x, x); }

// The normal distribution's tail, Phi(-a) = e * R(a) with e = exp(-a^2 / 2), for a = min(|x|, 16) (beyond it both are zero
// in FP32); returns S * R(a).  (1 + erf(x / sqrt(2)) instead would cancel for x below -1.)  R is a polynomial without constant
// term in t = 1 / (1 + c a) - the form of Hastings' approximations of the error function, but fitted here (least squares
// with Lawson's weights, over 0 <= a <= 14.5) for the relative error.  Two elements at a time, for the packed FP32
// instructions; GELU' needs the exponential as well.
//   results of 16 bits   degree 7, 8.0e-7; in FP32, where a^2 / 2 is rounded before the exponential, 1.7e-6 up to a = 5 and
//                        6.9e-6 up to 13 - far below half a step of 16 bits (2.4e-4)
//   WIDE, of 32 bits     degree 9, 1.4e-8; the exponent's roundings are carried along, so that the FP32 arithmetic leaves
//                        4.2e-7 everywhere (4096 x 2048 x 2048 with GELU: 46.5 us with erff, 54.4 with erfcf)
template <bool WIDE, int S>
__device__ __forceinline__ float2 fused_tail(float2 a, float2& e) {
  const float kLog = -0.72134752044448170f;                // -log2(e) / 2
  const float2 a2 = __fmul2_rn(a, a), s = __fmul2_rn(a2, fused_2(kLog));
  e = make_float2(fused_exp2(s.x), fused_exp2(s.y));
  if constexpr (WIDE) {
    const float2 lo = __ffma2_rn(a, a, make_float2(-a2.x, -a2.y));      // what a^2 and the product with kLog, and kLog itself, lost
    float2 d = __ffma2_rn(a2, fused_2(kLog), make_float2(-s.x, -s.y));
    d = __ffma2_rn(lo, fused_2(kLog), d);
    d = __ffma2_rn(a2, fused_2(static_cast<float>(-0.72134752044448170368 - static_cast<double>(kLog))), d);
    e = __ffma2_rn(__fmul2_rn(e, fused_2(0.69314718055994531f)), d, e);
    const float2 q = __ffma2_rn(a, fused_2(0.265f), fused_2(1.0f));
    const float2 t = make_float2(fused_rcp(q.x), fused_rcp(q.y));
    float2 r = __ffma2_rn(t, fused_2(S * 0.03062436632f), fused_2(S * -0.14330013024f));
    r = __ffma2_rn(r, t, fused_2(S * 0.21594934599f));
    r = __ffma2_rn(r, t, fused_2(S * -0.11428526510f));
    r = __ffma2_rn(r, t, fused_2(S * 0.13655412860f));
    r = __ffma2_rn(r, t, fused_2(S * 0.06089536025f));
    r = __ffma2_rn(r, t, fused_2(S * 0.10255500375f));
    r = __ffma2_rn(r, t, fused_2(S * 0.10526679036f));
    r = __ffma2_rn(r, t, fused_2(S * 0.10574039670f));
    return __fmul2_rn(r, t);
  }
  const float2 d = __ffma2_rn(a, fused_2(0.363f), fused_2(1.0f));
  const float2 t = make_float2(fused_rcp(d.x), fused_rcp(d.y));
  float2 r = __ffma2_rn(t, fused_2(S * 0.04808691645f), fused_2(S * -0.17913879823f));
  r = __ffma2_rn(r, t, fused_2(S * 0.17315124342f));
  r = __ffma2_rn(r, t, fused_2(S * 0.03082215889f));
  r = __ffma2_rn(r, t, fused_2(S * 0.13898195055f));
  r = __ffma2_rn(r, t, fused_2(S * 0.14320129268f));
  r = __ffma2_rn(r, t, fused_2(S * 0.14489563390f));
  return __fmul2_rn(r, t);
}

template <bool WIDE>
__device__ __forceinline__ float2 fused_gelu2(float2 x) {      // x Phi(x) = max(x, 0) - |x| Phi(-|x|)
  float2 e;
  const float2 a = make_float2(fused_min_nan(fabsf(x.x), 16.0f), fused_min_nan(fabsf(x.y), 16.0f));
  const float2 r = __fmul2_rn(a, fused_tail<WIDE, -1>(a, e));
  return __ffma2_rn(r, e, make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}

template <bool WIDE>
__device__ __forceinline__ float2 fused_gelu_gradient2(float2 z) {
  float2 e;
  const float2 a = make_float2(fused_min_nan(fabsf(z.x), 16.0f), fused_min_nan(fabsf(z.y), 16.0f));
  // w = Phi(-a) - a phi(a) is the derivative at -a, and 1 - w the one at a
  const float2 w = __fmul2_rn(__ffma2_rn(a, fused_2(-0.3989422804014327f), fused_tail<WIDE, 1>(a, e)), e);
  const float2 r = __ffma2_rn(w, fused_2(-1.0f), fused_2(1.0f));
  return make_float2(z.x > 0.0f ? r.x : w.x, z.y > 0.0f ? r.y : w.y);
}

// Activations for results of 32 bits, one element.
__device__ __forceinline__ float fused_act(float x, int32_t act) {
  if (act == FUSED_ACT_RELU) return fused_max_nan(x, 0.0f);
  if (act == FUSED_ACT_GELU) return fused_gelu2<true>(fused_2(x)).x;
  if (act == FUSED_ACT_SILU) return fused_max_nan(x, -128.0f) / (1.0f + expf(-x));
  return x;
}

// act'(z), with ReLU'(0) = 0.  Where z multiplies something that has run out to zero it is clamped first, so
// that an infinite z (a 16-bit pre-activation that overflowed) gives the limit, 0 or 1, instead of inf * 0.
__device__ __forceinline__ float fused_act_gradient(float z, int32_t act) {
  if (act == FUSED_ACT_RELU) return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
  if (act == FUSED_ACT_GELU) return fused_gelu_gradient2<true>(fused_2(z)).x;
  if (act == FUSED_ACT_SILU) {
    const float c = fminf(fmaxf(z, -80.0f), 80.0f);
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + c * (1.0f - s));
  }
  return 1.0f;
}

// Two elements at a time.  For results of 16 bits, whose half step (2^-12 relative at best) is far above the 2^-21 of the
// hardware exponential and reciprocal, SiLU takes those too.
__device__ __forceinline__ float2 fused_sigmoid2(float2 x) {
  const float2 s = __fmul2_rn(x, fused_2(-1.4426950408889634f));
  const float2 d = __fadd2_rn(make_float2(fused_exp2(s.x), fused_exp2(s.y)), fused_2(1.0f));
  return make_float2(fused_rcp(d.x), fused_rcp(d.y));
}

template <int ACT, bool WIDE = false>
__device__ __forceinline__ float2 fused_act2(float2 x) {
  if constexpr (ACT == FUSED_ACT_RELU) return make_float2(fused_max_nan(x.x, 0.0f), fused_max_nan(x.y, 0.0f));
  if constexpr (ACT == FUSED_ACT_GELU) return fused_gelu2<WIDE>(x);
  if constexpr (ACT == FUSED_ACT_SILU && WIDE) return make_float2(fused_act(x.x, ACT), fused_act(x.y, ACT));
  if constexpr (ACT == FUSED_ACT_SILU)
    return __fmul2_rn(make_float2(fused_max_nan(x.x, -128.0f), fused_max_nan(x.y, -128.0f)), fused_sigmoid2(x));
  return x;
}

template <int ACT, bool WIDE = false>
__device__ __forceinline__ float2 fused_act_gradient2(float2 z) {
  if constexpr (ACT == FUSED_ACT_RELU || (ACT == FUSED_ACT_SILU && WIDE))
    return make_float2(fused_act_gradient(z.x, ACT), fused_act_gradient(z.y, ACT));
  if constexpr (ACT == FUSED_ACT_GELU) return fused_gelu_gradient2<WIDE>(z);
  if constexpr (ACT == FUSED_ACT_SILU) {
    const float2 s = fused_sigmoid2(z);
    const float2 c = make_float2(fminf(fmaxf(z.x, -80.0f), 80.0f), fminf(fmaxf(z.y, -80.0f), 80.0f));
    const float2 w = __ffma2_rn(c, __ffma2_rn(s, fused_2(-1.0f), fused_2(1.0f)), fused_2(1.0f));
    return __fmul2_rn(s, w);
  }
  return fused_2(1.0f);
}

__device__ __forceinline__ float fused_load(const void* p, int64_t i, int dt) {   // dt: 0 F16, 1 BF16, 2 F32
  if (dt == 2) return static_cast<const float*>(p)[i];
  if (dt == 0) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void fused_put(void* p, int64_t i, int dt, float v) {
  if (dt == 2) static_cast<float*>(p)[i] = v;
  else if (dt == 0) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// One element (m, n) for the kernels that finish element by element: x = alpha * sum + bias; keeps or reads Z and
// returns D's value.  C is at element ci.
__device__ __forceinline__ float fused_finish(const FusedParams& f, float x, float beta, const void* C, int64_t ci, int dtype_c,
                                              int act, int m, int64_t n) {
  const float c = beta != 0.0f ? beta * fused_load(C, ci, dtype_c) : 0.0f;
  const int64_t zi = m + n * f.z_sn;
  if (f.form != FUSED_RESIDUAL && beta != 0.0f) x += c;
  if (f.form == FUSED_GRADIENT) return x * fused_act_gradient(fused_load(f.Z, zi, f.dtype_z), act);
  if (f.Z != nullptr) fused_put(f.Z, zi, f.dtype_z, x);
  x = fused_act(x, act);
  return f.form == FUSED_RESIDUAL && beta != 0.0f ? x + c : x;
}

// Column group boundaries as a warp reads them: lane l of a chunk of 32 groups gets [lo, hi) of group
// base + l.  Whatever the array holds, every value is clamped to [0, total] and the running maximum is
// taken, so groups never overlap, never run backwards and never leave the matrix.  `carry` starts as
// fused_first_offset() and is handed from chunk to chunk; all 32 lanes call.
__device__ __forceinline__ int fused_offset(const FusedParams& f, int i) {
  const long long v = f.offsets64 ? static_cast<const long long*>(f.offsets)[i]
                                  : static_cast<long long>(static_cast<const int32_t*>(f.offsets)[i]);
  return static_cast<int>(v < 0 ? 0 : (v > f.total ? f.total : v));
}

__device__ __forceinline__ int fused_first_offset(const FusedParams& f) { return f.offsets ? fused_offset(f, 0) : 0; }

__device__ __forceinline__ void fused_group_chunk(const FusedParams& f, int base, int lane, int& carry, int& lo, int& hi) {
  const int g = base + lane;
  int v = g < f.groups ? (f.offsets ? fused_offset(f, g + 1) : f.total) : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v = max(v, o);
  }
  hi = max(v, carry);
  lo = __shfl_up_sync(0xffffffffu, hi, 1);
  if (lane == 0) lo = carry;
  carry = __shfl_sync(0xffffffffu, hi, 31);
}

// Inclusive sum over the lanes of a warp.
__device__ __forceinline__ int fused_warp_scan(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// The block's work item in a list that deals every group out in chunks of at most `per` columns:
// item -> group g, first column c0, columns n (n == 0: the list is shorter than `item`).  Called by one
// whole warp; all lanes get the answer.
__device__ __forceinline__ void fused_find_item(const FusedParams& f, int item, int per, int lane, int& g, int& c0, int& n) {
  g = 0; c0 = 0; n = 0;
  int carry = fused_first_offset(f);
  int first = 0;   // items before this chunk of groups
  for (int base = 0; base < f.groups; base += 32) {
    int lo, hi;
    fused_group_chunk(f, base, lane, carry, lo, hi);
    const int items = (hi - lo + per - 1) / per;
    const int incl = fused_warp_scan(items, lane);
    const int before = first + incl - items;
    const unsigned hit = __ballot_sync(0xffffffffu, item >= before && item < before + items);
    if (hit) {
      const int src = __ffs(hit) - 1;
      g = base + src;
      const int k = item - __shfl_sync(0xffffffffu, before, src);
      c0 = __shfl_sync(0xffffffffu, lo, src) + k * per;
      n = min(per, __shfl_sync(0xffffffffu, hi, src) - c0);
      return;
    }
    first += __shfl_sync(0xffffffffu, incl, 31);
  }
}

}  // namespace gk
