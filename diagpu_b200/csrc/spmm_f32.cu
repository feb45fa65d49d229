/* spmm_f32.cu -- CUDA-core kernels of the block-vector product, fp32. */
#include "spmm_cores.cuh"

template struct dia::Cores<float>;
