// The Dense layer's matrix products in bf16 (kernels: layer_gemm.h).
#include "layer_gemm_launch.h"

int layer_gemm_bf16(int product, int block, bool direct, const void* args, hipStream_t st) {
  const GemmArgs& g = *static_cast<const GemmArgs*>(args);
  return direct ? launch_product<Bf16, true>(product, block, g, st) : launch_product<Bf16, false>(product, block, g, st);
}

int layer_grads_bf16(bool direct, const void* dx, const void* dk, hipStream_t st) {
  const GemmArgs &a = *static_cast<const GemmArgs*>(dx), &b = *static_cast<const GemmArgs*>(dk);
  return direct ? launch_grads<Bf16, true>(a, b, st) : launch_grads<Bf16, false>(a, b, st);
}
