// Instances of the tcgen05 kernel for the layer-level forms: 16-bit operands, one plane; one CTA per tile, CTA pairs, or
// one CTA fed by bounds-checked loads; one per kind of epilogue.  Included by one translation unit per form.
#pragma once
#include "tc_gemm.cuh"

namespace gk {

template <int FORM, int EPI>
static const void* tc_form_instance(int cg, bool generic) {
  if (generic) return reinterpret_cast<const void*>(&tc_gemm_kernel<1, 1, false, false, true, false, FORM, EPI>);
  return cg == 2 ? reinterpret_cast<const void*>(&tc_gemm_kernel<2, 1, false, false, false, false, FORM, EPI>)
                 : reinterpret_cast<const void*>(&tc_gemm_kernel<1, 1, false, false, false, false, FORM, EPI>);
}

template <int FORM>
const void* tc_kernel_form(int epi, int cg, bool generic) {
  if (epi == kTcWords) return tc_form_instance<FORM, kTcWords>(cg, generic);
  if (epi == kTcFloats) return tc_form_instance<FORM, kTcFloats>(cg, generic);
  return tc_form_instance<FORM, kTcElements>(cg, generic);
}

}  // namespace gk
