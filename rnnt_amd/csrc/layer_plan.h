// How a Dense layer's products are cut into blocks, shared by the host code (layer.hip) and the kernels of each type.
#pragma once
#include <hip/hip_runtime.h>

// the three products of a layer: which operand is strided along k
enum LayerProduct { kForward = 0 /* x k-fast, W k-slow */, kInputGrad = 1 /* dz, W k-fast */, kKernelGrad = 2 /* x, dz k-slow */ };
// block of the result
enum LayerBlock { kBlock32 = 0 /* 32 x 64 from aligned 16-bit operands, else 32 x 128 */, kBlock64x64 = 1, kBlock128x128 = 2, kBlock256x256 = 3, kBlock32Groups = 5, kBlock64Groups = 6 /* 32 x 64, 64 x 64, four groups share k */, kBlock64Thin = 7 /* 64 x 32, four groups, aligned 16-bit operands, forward */, kBlockRows = 4 /* up to 8 rows, forward: layer.hip */ };

// launch one product, or both gradients' in 128 x 128 blocks; `args` is a GemmArgs (layer_gemm.h), every translation unit has its own copy of that type
#define RNNT_HIDDEN __attribute__((visibility("hidden")))
RNNT_HIDDEN int layer_gemm_fp32(int product, int block, bool direct, const void* args, hipStream_t st);
RNNT_HIDDEN int layer_gemm_bf16(int product, int block, bool direct, const void* args, hipStream_t st);
RNNT_HIDDEN int layer_gemm_fp16(int product, int block, bool direct, const void* args, hipStream_t st);
RNNT_HIDDEN int layer_grads_fp32(bool direct, const void* dx, const void* dk, hipStream_t st);
RNNT_HIDDEN int layer_grads_bf16(bool direct, const void* dx, const void* dk, hipStream_t st);
RNNT_HIDDEN int layer_grads_fp16(bool direct, const void* dx, const void* dk, hipStream_t st);
