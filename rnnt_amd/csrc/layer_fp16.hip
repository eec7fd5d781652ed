// The Dense layer's matrix products in fp16 (kernels: layer_gemm.h).
#include "layer_gemm_launch.h"

int layer_gemm_fp16(int product, int block, bool direct, const void* args, hipStream_t st) {
  const GemmArgs& g = *static_cast<const GemmArgs*>(args);
  return direct ? launch_product<Fp16, true>(product, block, g, st) : launch_product<Fp16, false>(product, block, g, st);
}
