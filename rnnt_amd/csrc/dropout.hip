// Dropout whose mask is never stored (gfx950): y = x * m / keep, with m drawn from Philox4x32-10 at a counter made of the
// element's row, its column and the caller's offset (op_util.h).  The backward pass is the same call on the upstream
// gradient.
#include "op_util.h"

namespace {

#ifdef RNNT_BUILD_STAMP
__attribute__((used)) const char kBuildStamp[] = RNNT_BUILD_STAMP;  // the flags all sources were compiled with: build.py looks for it
#endif

constexpr int kThreads = 256;
constexpr int kGroups = 4;  // groups of eight elements per thread, all loaded before the first draw

// One pass, read once and written once: 4 bytes an element in 16 bits, and ten Philox rounds per eight elements.  Bound by
// memory: 262144 x 1024 bfloat16 187 us = 5.7 TB/s (a large copy: 5.3 TB/s).
template <class T>
__global__ __launch_bounds__(kThreads) void k_dropout(const typename T::elem* x, typename T::elem* y,
                                                      uint32_t rows, int cols, uint32_t groups, uint32_t magic,
                                                      long long x_stride, DropArgs a) {
  load_offset(a);
  const uint64_t start = (uint64_t)blockIdx.x * (kThreads * kGroups);
  // uniform over the block: the row its first group lies in
  const uint32_t row0 = (uint32_t)(start / groups), g0 = (uint32_t)(start - (uint64_t)row0 * groups);
  uint32_t row[kGroups], g[kGroups];
  Raw8<T> raw[kGroups];
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    const uint32_t v = g0 + j * kThreads + threadIdx.x;
    // v / groups: exact while v * groups < 2^32 (magic = ceil(2^32 / groups)); longer rows end at most once in a block
    const uint32_t q = magic ? __umulhi(v, magic) : (v >= groups ? 1u : 0u);
    row[j] = groups == 1 ? row0 + v : row0 + q;
    g[j] = groups == 1 ? 0 : v - q * groups;
    if (row[j] < rows && 8 * g[j] + 8 <= (uint32_t)cols) raw[j] = load8_raw<T>(x + (long long)row[j] * x_stride + 8 * g[j]);
  }
#pragma unroll
  for (int j = 0; j < kGroups; ++j) {
    if (row[j] >= rows) continue;
    const int left = cols - (int)(8 * g[j]);
    typename T::elem* out = y + (long long)row[j] * cols + 8 * g[j];
    float v[8];
    if (left >= 8) {
      unpack8<T>(raw[j], v);
      drop8(a, row[j], g[j], v);
      store8<T>(out, v);
    } else {
      load_some<T>(x + (long long)row[j] * x_stride + 8 * g[j], left, v);
      drop8(a, row[j], g[j], v);
      store_some<T>(out, left, v);
    }
  }
}

template <class T>
int launch(const void* x, void* y, long long rows, int cols, long long x_stride, const DropArgs& a, hipStream_t st) {
  const uint32_t groups = (uint32_t)(((long long)cols + 7) / 8);
  const uint64_t total = (uint64_t)rows * groups, per = kThreads * kGroups;
  if ((total + per - 1) / per > 0x7fffffffull) return RNNT_MI355X_UNSUPPORTED_SIZE;
  // the block's first group is below `groups`, so v < groups + 1024
  const bool small = (uint64_t)groups * (groups + per) < (1ull << 32);
  const uint32_t magic = small && groups > 1 ? (uint32_t)(((1ull << 32) + groups - 1) / groups) : 0;
  k_dropout<T><<<(unsigned)((total + per - 1) / per), kThreads, 0, st>>>(
      static_cast<const typename T::elem*>(x), static_cast<typename T::elem*>(y), (uint32_t)rows, cols, groups, magic, x_stride, a);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}

}  // namespace

extern "C" int rnnt_mi355x_dropout(const void* x, long long x_stride, void* y, long long rows, int cols, int dtype, int drop16,
                                   uint64_t seed, uint64_t offset, const uint64_t* offset_dev, void* hip_stream) {
  if (!x || !y || rows < 1 || cols < 1 || x_stride < cols || drop16 < 0 || drop16 > 65535) return RNNT_MI355X_INVALID_VALUE;
  if (x == y && x_stride != cols) return RNNT_MI355X_INVALID_VALUE;
  if (rows > 0x7fffffffll) return RNNT_MI355X_UNSUPPORTED_SIZE;
  const DropArgs a = drop_args(drop16, seed, offset, offset_dev);
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case RNNT_MI355X_FP32: return launch<Fp32>(x, y, rows, cols, x_stride, a, st);
    case RNNT_MI355X_BF16: return launch<Bf16>(x, y, rows, cols, x_stride, a, st);
    case RNNT_MI355X_FP16: return launch<Fp16>(x, y, rows, cols, x_stride, a, st);
  }
  return RNNT_MI355X_INVALID_VALUE;
}
