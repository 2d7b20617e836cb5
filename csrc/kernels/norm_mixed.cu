// Norms and residual joins: types float, bf16 (along the residual connection, inside a block)
#include "norm_kernels.cuh"

bool rownorm::run_mixed(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st) { return run<float, bf16>(p, backward, vec, st); }
