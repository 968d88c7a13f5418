// tcgen05 GEMM instances: fused epilogues.
#include "tc_kernels_form.cuh"

namespace gk {
template const void* tc_kernel_form<kTcFused>(int epi, int cg, bool generic);
}
