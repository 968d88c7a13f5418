// tcgen05 GEMM instances of the layer-level forms (fused epilogues, ragged columns, ragged depth): 16-bit operands,
// one plane; one CTA per tile, CTA pairs, or one CTA fed by bounds-checked loads.
#include "tc_gemm.cuh"

namespace gk {

template <int FORM>
static const void* pick(int cg, bool generic) {
  if (generic) return reinterpret_cast<const void*>(&tc_gemm_kernel<1, 1, false, false, true, false, FORM>);
  return cg == 2 ? reinterpret_cast<const void*>(&tc_gemm_kernel<2, 1, false, false, false, false, FORM>)
                 : reinterpret_cast<const void*>(&tc_gemm_kernel<1, 1, false, false, false, false, FORM>);
}

const void* tc_kernel_fused(int form, int cg, bool generic) {
  if (form == kTcFused) return pick<kTcFused>(cg, generic);
  if (form == kTcRaggedCols) return pick<kTcRaggedCols>(cg, generic);
  return pick<kTcRaggedDepth>(cg, generic);
}

}  // namespace gk
