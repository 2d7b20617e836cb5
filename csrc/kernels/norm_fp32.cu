// Norms and residual joins: types float, float (along the residual connection, inside a block)
#include "norm_kernels.cuh"

bool rownorm::run_fp32(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st) { return run<float, float>(p, backward, vec, st); }
