// Instances of k_layer_gemm for one element type.
#pragma once
#include "layer_gemm.h"
#include "layer_plan.h"

namespace {

unsigned blocks_of(const GemmArgs& g) { return (unsigned)(g.whole + (g.tiles_m * g.tiles_n - g.whole) * g.splits); }

template <class T, int PRODUCT, int BM, int BN, int BK, int WM, int WN, bool DIRECT, int GROUPS = 1>
int launch_gemm(const GemmArgs& g, hipStream_t st) {
  constexpr bool kASlow = PRODUCT == kKernelGrad, kBSlow = PRODUCT != kInputGrad;
  const unsigned grid = blocks_of(g), block = (BM / WM) * (BN / WN) * 64 * GROUPS;
  if constexpr (DIRECT) k_layer_gemm_ring<T, kASlow, kBSlow, BM, BN, WM, WN, GROUPS><<<grid, block, 0, st>>>(g);
  else k_layer_gemm<T, kASlow, kBSlow, BM, BN, BK, WM, WN, GROUPS><<<grid, block, 0, st>>>(g);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}

template <class T, int PRODUCT, bool DIRECT>
int launch_block(int block, const GemmArgs& g, hipStream_t st) {
  constexpr int BK = kPlanes<T> == 3 ? 32 : 64;
  switch (block) {
    case kBlock32:
      if constexpr (PRODUCT != kKernelGrad) return launch_gemm<T, PRODUCT, 32, DIRECT ? 64 : 128, 64, 32, 32, DIRECT>(g, st);
      break;
    case kBlock64x64: return launch_gemm<T, PRODUCT, 64, 64, BK, 32, 32, DIRECT>(g, st);
    case kBlock32Groups:
      if constexpr (PRODUCT != kKernelGrad) return launch_gemm<T, PRODUCT, 32, 64, 32, 32, 32, DIRECT, 4>(g, st);
      break;
    case kBlock64Groups:
      if constexpr (PRODUCT != kKernelGrad) return launch_gemm<T, PRODUCT, 64, 64, BK, 32, 32, DIRECT, 4>(g, st);
      break;
    case kBlock64Thin:
      if constexpr (PRODUCT == kForward && DIRECT) return launch_gemm<T, PRODUCT, 64, 32, 32, 32, 32, DIRECT, 4>(g, st);
      break;
    case kBlock128x128: return launch_gemm<T, PRODUCT, 128, 128, BK, 64, 64, DIRECT>(g, st);
    case kBlock256x256:
      if constexpr (DIRECT) return launch_gemm<T, PRODUCT, 256, 256, 64, 128, 64, DIRECT>(g, st);
      break;
  }
  return RNNT_MI355X_INVALID_VALUE;
}

template <class T, bool DIRECT>
int launch_product(int product, int block, const GemmArgs& g, hipStream_t st) {
  switch (product) {
    case kForward: return launch_block<T, kForward, DIRECT>(block, g, st);
    case kInputGrad: return launch_block<T, kInputGrad, DIRECT>(block, g, st);
  }
  return launch_block<T, kKernelGrad, DIRECT>(block, g, st);
}

template <class T, bool DIRECT>
int launch_grads(const GemmArgs& dx, const GemmArgs& dk, hipStream_t st) {
  const unsigned first = blocks_of(dx), all = first + blocks_of(dk);
  if constexpr (DIRECT) k_layer_grads_ring<T><<<all, 256, 0, st>>>(dx, dk, first);
  else k_layer_grads<T><<<all, 256, 0, st>>>(dx, dk, first);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}

}  // namespace
