// tcgen05 GEMM instances: ragged depth.
#include "tc_kernels_form.cuh"

namespace gk {
template const void* tc_kernel_form<kTcRaggedDepth>(int epi, int cg, bool generic);
}
