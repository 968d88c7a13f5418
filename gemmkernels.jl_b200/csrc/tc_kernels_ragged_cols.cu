// tcgen05 GEMM instances: ragged columns.
#include "tc_kernels_form.cuh"

namespace gk {
template const void* tc_kernel_form<kTcRaggedCols>(int epi, int cg, bool generic);
}
