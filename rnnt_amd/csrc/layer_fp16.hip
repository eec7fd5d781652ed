// The Dense layer's matrix products in fp16 (kernels: layer_gemm.h).
#include "layer_gemm_launch.h"

int layer_gemm_fp16(int product, int block, bool direct, const void* args, hipStream_t st) {
  const GemmArgs& g = *static_cast<const GemmArgs*>(args);
  return direct ? launch_product<Fp16, true>(product, block, g, st) : launch_product<Fp16, false>(product, block, g, st);
}

int layer_grads_fp16(bool direct, const void* dx, const void* dk, hipStream_t st) {
  const GemmArgs &a = *static_cast<const GemmArgs*>(dx), &b = *static_cast<const GemmArgs*>(dk);
  return direct ? launch_grads<Fp16, true>(a, b, st) : launch_grads<Fp16, false>(a, b, st);
}
