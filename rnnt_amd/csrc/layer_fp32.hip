// The Dense layer's matrix products in fp32 (kernels: layer_gemm.h).
#include "layer_gemm_launch.h"

int layer_gemm_fp32(int product, int block, bool, const void* args, hipStream_t st) {
  return launch_product<Fp32, false>(product, block, *static_cast<const GemmArgs*>(args), st);
}

int layer_grads_fp32(bool, const void* dx, const void* dk, hipStream_t st) {
  return launch_grads<Fp32, false>(*static_cast<const GemmArgs*>(dx), *static_cast<const GemmArgs*>(dk), st);
}
