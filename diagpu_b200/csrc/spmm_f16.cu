/* spmm_f16.cu -- CUDA-core kernels of the block-vector product, fp16. */
#include "spmm_cores.cuh"

template struct dia::Cores<__half>;
