// The Dense layer's matrix products in bf16 (kernels: layer_gemm.h).
#include "layer_gemm_launch.h"

int layer_gemm_bf16(int product, int block, bool direct, const void* args, hipStream_t st) {
  const GemmArgs& g = *static_cast<const GemmArgs*>(args);
  return direct ? launch_product<Bf16, true>(product, block, g, st) : launch_product<Bf16, false>(product, block, g, st);
}
