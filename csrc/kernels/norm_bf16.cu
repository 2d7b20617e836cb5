// Norms and residual joins: types bf16, bf16 (along the residual connection, inside a block)
#include "norm_kernels.cuh"

bool rownorm::run_bf16(const GeepsResidual& p, bool backward, bool vec, cudaStream_t st) { return run<bf16, bf16>(p, backward, vec, st); }
