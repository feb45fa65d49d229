/* spmm_bf16.cu -- CUDA-core kernels of the block-vector product, bf16. */
#include "spmm_cores.cuh"

template struct dia::Cores<__nv_bfloat16>;
