// Dense layer with its epilogue for MI355X (gfx950):
//     z = x W + b,   y = residual + dropout(act(z))
// and its backward pass
//     dz = dropout'(dy) act'(z),   dx = dz W^T,   dW = x^T dz,   db = sum over rows of dz,   d residual = dy
// -- the TimeDistributed(Dense) and Dropout layers of get_fc (reference rnnt/keras_model.py:83-104), Keras kernel layout
// [in, out], at any width.  Products: layer_gemm.h.  Here: how they are cut, dz, and the sums of partial results.
#include "layer_gemm.h"
#include "layer_plan.h"

namespace {

// ---- dz and the column sums that become db -------------------------------------------------------------------------------
enum Saved { kNothing = 0, kPreActivation = 1, kOutput = 2 };
constexpr int kDzGroups = 32, kDzLanes = 8;  // a block: 32 groups of eight columns, 8 rows at a time

struct DzArgs {
  const void *dy, *saved;
  void* dz;         // nullable: dz is dy (linear, no dropout) and only the sums are wanted
  float* partial;   // nullable [row blocks][N]
  long long dy_ld, dz_ld;
  int M, N, rows;   // rows of a block
  int across;       // blocks that a row takes
  unsigned blocks;  // of this pass; copies follow
  int act, from;
  DropArgs drop;
};

// dz / dropout' of eight elements: act' from what the forward pass left.
template <class T>
__device__ __forceinline__ void slopes8(const DzArgs& a, long long m, int n0, int n, float (&v)[8]) {
  float s[8];
  if (a.from == kPreActivation) {
    using A = typename AuxOf<T>::type;
    const typename A::elem* p = static_cast<const typename A::elem*>(a.saved) + m * a.N + n0;
    if (n >= 8) unpack8<A>(load8_raw<A>(p), s);
    else load_some<A>(p, n, s);
    switch (a.act) {
      case kTanh:
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= slope_of(s[i], kTanh);
        break;
      case kRelu:
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= slope_of(s[i], kRelu);
        break;
      case kGelu:
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= slope_of(s[i], kGelu);
        break;
      case kSilu:
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= slope_of(s[i], kSilu);
        break;
    }
  } else {  // y = act(z) * scale (0 where dropped: dy is dropped there as well)
    const typename T::elem* p = static_cast<const typename T::elem*>(a.saved) + m * a.N + n0;
    if (n >= 8) unpack8<T>(load8_raw<T>(p), s);
    else load_some<T>(p, n, s);
    const float keep = a.drop.drop ? __builtin_amdgcn_rcpf(a.drop.scale) : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = s[i] * keep;
      v[i] *= a.act == kRelu ? (s[i] > 0.f ? 1.f : 0.f) : fmaf(-t, t, 1.f);
    }
  }
}

// ---- rows that do not lie on 16-byte boundaries --------------------------------------------------------------------------
// A 16-bit matrix copied to rows of whole 16-byte pieces, zeros behind the last column: with it the products take the
// ring kernel.
struct PackArgs {
  const uint16_t* src;
  uint16_t* dst;
  long long src_ld, dst_ld, rows;
  int cols;
  unsigned blocks;  // 0: nothing to copy
};
__device__ __forceinline__ void pack_block(const PackArgs& p, unsigned block) {
  const int pieces = (p.cols + 7) / 8;
  const long long id = (long long)block * 256 + threadIdx.x, row = id / pieces;
  if (row >= p.rows) return;
  const int c = (int)(id - row * pieces) * 8;
  const Raw8<Bf16> r = load_group<Bf16>(p.src + row * p.src_ld + c, p.cols - c);
  *reinterpret_cast<u4*>(p.dst + row * p.dst_ld + c) = r.q[0];
}
__global__ __launch_bounds__(256) void k_layer_pack(PackArgs a, PackArgs b) {
  if (blockIdx.x < a.blocks) pack_block(a, blockIdx.x);
  else pack_block(b, blockIdx.x - a.blocks);
}

// dz, its column sums, and the copies of the operands that lie badly: what the gradient's products begin with.  In 16-bit layers
// dz is rounded to the type, as the matrix instruction takes it: a rounding next to the result's own, so that the gradients'
// relative error (2-norm, against float64) is 2.9e-4 instead of 2.1e-4 in float16 and 2.3e-3 instead of 1.7e-3 in bfloat16.  dz in two parts
// would keep it and double both products.  The column sums take it unrounded.  Bound by
// memory, dy and the saved tensor read once and dz written once (49200 x 250 float32, tanh and dropout: 28 us = 5.3 TB/s), or by
// the slope and the generator where elements are small (32768 x 4096 bfloat16, gelu and dropout: 185 us = 4.3 TB/s).
template <class T>
__global__ __launch_bounds__(kDzGroups * kDzLanes) void k_layer_dz(DzArgs a, PackArgs p, PackArgs q) {
  static_assert(kDzGroups * kDzLanes == 256, "pack_block's size");
  __shared__ float sums[kDzLanes][kDzGroups * 8 + 4];
  if (blockIdx.x >= a.blocks) {
    const unsigned i = blockIdx.x - a.blocks;
    if (i < p.blocks) pack_block(p, i);
    else pack_block(q, i - p.blocks);
    return;
  }
  load_offset(a.drop);
  const int bx = blockIdx.x % (unsigned)a.across, by = blockIdx.x / (unsigned)a.across;
  const int gx = threadIdx.x % kDzGroups, ty = threadIdx.x / kDzGroups;
  const int n0 = (bx * kDzGroups + gx) * 8, left = a.N - n0;
  const int m0 = by * a.rows, m1 = min(a.M, m0 + a.rows);
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (left > 0) {
#pragma unroll 2
    for (int m = m0 + ty; m < m1; m += kDzLanes) {
      float v[8];
      const typename T::elem* p = static_cast<const typename T::elem*>(a.dy) + (long long)m * a.dy_ld + n0;
      if (left >= 8) unpack8<T>(load8_raw<T>(p), v);
      else load_some<T>(p, left, v);
      if (a.act != kLinear) slopes8<T>(a, m, n0, left, v);
      if (a.drop.drop) drop8(a.drop, (uint32_t)m, (uint32_t)n0 >> 3, v);
      if (a.dz) {
        typename T::elem* q = static_cast<typename T::elem*>(a.dz) + m * a.dz_ld + n0;
        store8<T>(q, v);  // whole pieces: what lies behind the last column is zero
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += v[i];
    }
  }
  if (!a.partial) return;  // uniform
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[ty][gx * 8 + i] = sum[i];
  __syncthreads();
  const int n = bx * kDzGroups * 8 + threadIdx.x;
  if (n < a.N) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kDzLanes; ++i) s += sums[i][threadIdx.x];
    a.partial[(long long)by * a.N + n] = s;
  }
}

// ---- joining the splits of a product, and db from its partial sums -------------------------------------------------------
struct DbArgs {
  const float* partial;  // [blocks][N]
  void* db;              // null: none
  int blocks, N;
};
// 16 columns, 16 row blocks at a time; the order is fixed
template <class T>
__device__ __forceinline__ void db_block(const DbArgs& d, unsigned block, float* sums) {
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, n = block * 16 + c;
  float s = 0.f;
  if (n < d.N) {
#pragma unroll 16
    for (int i = r; i < d.blocks; i += 16) s += d.partial[(long long)i * d.N + n];
  }
  sums[r * 17 + c] = s;
  __syncthreads();
  if (r == 0 && n < d.N) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i * 17 + c];
    static_cast<typename T::elem*>(d.db)[n] = from_float<T>(s);
  }
}

// The cut tiles of a product: 256 / lanes groups of eight columns of one tile's rows a block; `lanes` threads share a group's
// splits.  The order is fixed.
struct JoinArgs {
  GemmArgs g;
  int bm, bn, lanes;
  unsigned blocks;
};
template <class T>
__device__ __forceinline__ void join_block(const JoinArgs& j, unsigned block, float* sums) {
  const GemmArgs& g = j.g;
  const int here = 256 / j.lanes, c = threadIdx.x % here, s0 = threadIdx.x / here, groups = j.bn / 8, per_tile = j.bm * groups / here;
  const int tile = block / per_tile, group = (block - tile * per_tile) * here + c;
  int tm, tn;
  place_of(g, g.whole + tile, tm, tn);
  const long long m = (long long)tm * j.bm + group / groups;
  const int n = tn * j.bn + 8 * (group % groups), left = g.N - n;
  const bool in = m < g.M && left > 0;
  float v[1][8] = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
  if (in) {
    const long long piece = (long long)j.bm * j.bn;
    const float* p = g.partial + tile * g.splits * piece + 8 * group;
#pragma unroll 4
    for (int s = s0; s < g.splits; s += j.lanes) {
      float w[8];
      unpack8<Fp32>(load8_raw<Fp32>(p + s * piece), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[0][i] += w[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[threadIdx.x * 9 + i] = v[0][i];
  __syncthreads();
  if (s0 != 0 || !in) return;
  for (int s = 1; s < j.lanes; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0][i] += sums[(s * here + c) * 9 + i];
  DropArgs drop = g.e.drop;
  if (drop.drop) load_offset(drop);
  finish<T, 1>(g.e, drop, {m}, g.M, n, left, v);
}
// What is left after the products of a call, in one launch.
template <class T>
__global__ __launch_bounds__(256) void k_layer_join(JoinArgs a, JoinArgs b, DbArgs db) {
  __shared__ float sums[256 * 9];
  const unsigned id = blockIdx.x;
  if (id < a.blocks) join_block<T>(a, id, sums);
  else if (id < a.blocks + b.blocks) join_block<T>(b, id - a.blocks, sums);
  else db_block<T>(db, id - a.blocks - b.blocks, sums);
}

// ---- a decoder's few rows ------------------------------------------------------------------------------------------------
constexpr int kRowsMost = 8, kRowsSlices = 16, kRowsChunk = 1024;
template <class T>
constexpr int kRowsVec = T::code == RNNT_MI355X_FP32 ? 1 : 2;  // columns a lane: a wavefront reads 256 bytes of a row of W

// x W for at most 8 rows: bound by the read of W, or by a launch and a few memory latencies for a small one, where the
// matrix cores' tiles of 32 rows would be mostly empty.  A block has 64 or 128 columns; its 16 wavefronts share k, each reads
// its rows of W straight into registers, 16 at a time, and takes x from LDS.  The sums of the wavefronts meet in LDS.
// 8 x 250 x 62 float32: 6.0 us of the GPU, the matrix cores' block of 32 rows 13.6.
template <class T, int MR>
__global__ __launch_bounds__(64 * kRowsSlices) void k_layer_rows(GemmArgs g) {
  using E = typename T::elem;
  constexpr int VEC = kRowsVec<T>, BN = 64 * VEC, kRed = kRowsSlices * MR * BN, kX = MR * kRowsChunk;
  __shared__ __attribute__((aligned(16))) float lds[kRed > kX ? kRed : kX];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % g.tiles_n, split = blockIdx.x / g.tiles_n;
  const int n0 = tile * BN, n = n0 + VEC * lane, left = g.N - n;
  const int k_begin = split * g.k_each, k_end = min(g.K, k_begin + g.k_each);
  const E *x = static_cast<const E*>(g.a), *w = static_cast<const E*>(g.b);
  float acc[MR][VEC];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[m][v] = 0.f;

  for (int k0 = k_begin; k0 < k_end; k0 += kRowsChunk) {
    const int len = min(kRowsChunk, k_end - k0), each = ((len + kRowsSlices - 1) / kRowsSlices + 3) & ~3;
    __syncthreads();
    for (int i = threadIdx.x; i < kX; i += 64 * kRowsSlices) {
      const int m = i / kRowsChunk, k = i % kRowsChunk;
      lds[i] = m < g.M && k < len ? to_float<T>(x[m * g.a_ld + k0 + k]) : 0.f;
    }
    __syncthreads();
    const int first = wave * each, last = min(len, first + each);
#pragma unroll 1
    for (int k = first; k < last; k += 16) {
      E q[16][VEC];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const E* p = w + (long long)(k0 + k + j) * g.b_ld + n;
#pragma unroll
        for (int v = 0; v < VEC; ++v) q[j][v] = 0;
        if (k + j < last) {
          if (left >= VEC) __builtin_memcpy(q[j], p, sizeof(q[j]));
          else if (left > 0) q[j][0] = p[0];
        }
      }
#pragma unroll
      for (int j = 0; j < 16; j += 4)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          const f4 a = *reinterpret_cast<const f4*>(lds + m * kRowsChunk + min(k + j, kRowsChunk - 4));
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              // past the wavefront's last k the row of W was not read: nothing is added, also where x is no number
              const float add = k + j + i < last ? a[i] : 0.f;
              acc[m][v] = fmaf(add, to_float<T>(q[j + i][v]), acc[m][v]);
            }
        }
    }
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int v = 0; v < VEC; ++v) lds[(wave * MR + m) * BN + VEC * lane + v] = acc[m][v];
  __syncthreads();
  for (int i = threadIdx.x; i < MR * BN; i += 64 * kRowsSlices) {
    float s = lds[i];
#pragma unroll
    for (int j = 1; j < kRowsSlices; ++j) s += lds[j * MR * BN + i];
    lds[i] = s;  // this thread's own
  }
  __syncthreads();
  constexpr int kGroups = BN / 8;
  const int m = threadIdx.x / kGroups, c = 8 * (threadIdx.x % kGroups);
  if (m >= MR || m >= g.M || n0 + c >= g.N) return;
  float v[1][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[0][i] = lds[m * BN + c + i];
  if (g.whole == 0) {
    store8<Fp32>(g.partial + ((long long)tile * g.splits + split) * (kRowsMost * BN) + m * BN + c, v[0]);
  } else {
    DropArgs drop = g.e.drop;
    if (drop.drop) load_offset(drop);
    finish<T, 1>(g.e, drop, {m}, g.M, n0 + c, g.N - n0 - c, v);
  }
}

template <class T>
int launch_rows(const GemmArgs& g, hipStream_t st) {
  const unsigned grid = (unsigned)(g.tiles_n * g.splits), block = 64 * kRowsSlices;
  if (g.M == 1) k_layer_rows<T, 1><<<grid, block, 0, st>>>(g);
  else if (g.M == 2) k_layer_rows<T, 2><<<grid, block, 0, st>>>(g);
  else if (g.M <= 4) k_layer_rows<T, 4><<<grid, block, 0, st>>>(g);
  else k_layer_rows<T, 8><<<grid, block, 0, st>>>(g);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}

// ---- host ----------------------------------------------------------------------------------------------------------------
struct Plan {
  int block, bm, bn, tiles_m, tiles_n, whole, splits, k_each;
  bool direct;
  size_t partial_bytes;
};

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

constexpr int kCUs = 256;

// Which block, and which tiles are cut along k.
Plan plan_product(int product, int dtype, int M, int N, int K, bool direct) {
  Plan p;
  p.direct = direct;
  p.bm = p.bn = 128;
  p.block = kBlock128x128;
  const int steps = ceil_div(K, 32);
  if (product == kForward && M <= kRowsMost) {
    // 256 blocks of 16 wavefronts if k allows pieces of 512 or more
    p.block = kBlockRows;
    p.bm = kRowsMost;
    p.bn = dtype == RNNT_MI355X_FP32 ? 64 : 128;
    p.tiles_m = 1;
    p.tiles_n = ceil_div(N, p.bn);
    p.splits = kCUs / p.tiles_n < K / 512 ? kCUs / p.tiles_n : K / 512;
    if (p.splits < 2) p.splits = 1;
    p.k_each = ceil_div(ceil_div(K, p.splits), 64) * 64;
    p.splits = ceil_div(K, p.k_each);
    p.whole = p.splits == 1 ? p.tiles_n : 0;
    p.partial_bytes = p.whole ? 0 : (size_t)p.tiles_n * p.splits * p.bm * p.bn * sizeof(float);
    return p;
  }
  if (product != kKernelGrad && M <= 64 && ceil_div(N, 64) >= 32) {
    // Few rows of a wide layer: a block for every CU at most, in which four groups share k; pieces of k only where blocks are
    // fewer, of 1024 or more.  Against blocks of one group and more pieces: 64 x 2048 x 8192 bfloat16 14.7 us (16.1), float32
    // 27 (33), 64 x 4096 x 16384 float32 82 (124), 32 x 512 x 4096 float32 9.0 (11.5); with fewer columns the pieces win.
    p.block = M <= 32 ? kBlock32Groups : kBlock64Groups;
    p.bm = M <= 32 ? 32 : 64;
    p.bn = 64;
    p.tiles_m = 1;
    if (product == kForward && direct && M > 32 && K <= 2048 && ceil_div(N, 32) <= kCUs) {
      // Columns halved instead of k cut, while every block reading all of x costs less than a join.  Thin against wide, us a call:
      // 64 rows in bfloat16, weights that come from memory: 2048 x 8192 17.2 (17.2), 2560 x 8192 21.2 (19.7), 3584 x 8192 26.1 (23.0);
      // 2560 x 4096 16.6 (18.4), 3584 x 4096 19.3 (18.4), 4096 x 4096 21.4 (17.6); 48 rows in float16 1024 x 8192 10.1 (11.5).  Weights that
      // the caches hold: 2048 x 8192 12.6 (14.1), 512 x 4096 6.6 (7.3), 256 x 8192 6.0 (6.7).  16 rows 1024 x 4096 7.9 (7.7).
      p.block = kBlock64Thin;
      p.bn = 32;
    }
    p.tiles_n = ceil_div(N, p.bn);
    p.splits = kCUs / p.tiles_n < K / 1024 ? kCUs / p.tiles_n : K / 1024;
    if (p.splits < 1) p.splits = 1;
    p.k_each = ceil_div(ceil_div(K, p.splits), 64) * 64;
    p.splits = ceil_div(K, p.k_each);
    p.whole = p.splits == 1 ? p.tiles_n : 0;
    p.partial_bytes = (size_t)(p.tiles_n - p.whole) * p.splits * p.bm * p.bn * sizeof(float);
    return p;
  }
  if (product != kKernelGrad && M <= 32) {
    p.block = kBlock32;
    p.bm = 32;
    p.bn = direct ? 64 : 128;
  } else if (M <= 64 || N <= 64) {
    p.block = kBlock64x64;
    p.bm = p.bn = 64;
  } else if (direct && (long long)ceil_div(M, 256) * ceil_div(N, 256) * (product == kKernelGrad ? ceil_div(K, 4096) : 1) >= 192) {
    p.block = kBlock256x256;
    p.bm = p.bn = 256;
  }
  p.tiles_m = ceil_div(M, p.bm);
  p.tiles_n = ceil_div(N, p.bn);
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  // Rounds of one tile a CU are done whole.  The rest would leave CUs idle for a round: it may be cut along k until there are
  // two pieces for every CU (one of the largest block), of two steps of 32 k at least in float32 and four in 16 bits.
  const int want = p.block == kBlock256x256 ? kCUs : 2 * kCUs;
  const int others = (int)(tiles % kCUs), least = dtype == RNNT_MI355X_FP32 ? 2 : 4;
  p.splits = others == 0 ? 1 : want / others;
  if (p.splits > steps / least) p.splits = steps / least;
  if (p.splits < 2) p.splits = 1;
  if (p.splits > 1) {
    // What that saves against what joining the pieces costs, in us.  A CU multiplies at 4.3 TFLOP/s in 16 bits (1.1 PFLOP/s of
    // the card) and at a sixth of it in float32; a block alone on its CU, with nobody to fill its waits, takes a quarter
    // more and 0.4 a step.  Joining is a launch, and the pieces written and read at 4 TB/s.  Measured, whole against cut:
    // float32 1200x250x250 24 : 14 us, 6151x1032x520 87 : 69, 6151x520x1032 56 : 66; bfloat16 64x2048x8192 19 : 15, 4096x512x512 10 : 24.
    double step = 2.0 * p.bm * p.bn * 32 / 4.3e6 * (dtype == RNNT_MI355X_FP32 ? 6 : 1);
    if (tiles < kCUs) step = 0.4 + 1.25 * step;
    const double saves = steps * step * (1.0 - 1.0 / p.splits), costs = 5.0 + 2.0 * others * p.splits * p.bm * p.bn * 4 / 4e6;
    if (saves < costs) p.splits = 1;
  }
  const int whole_k = p.block == kBlock32 || dtype != RNNT_MI355X_FP32 ? 64 : 32;  // what the steps of a piece divide
  p.k_each = ceil_div(ceil_div(K, p.splits), whole_k) * whole_k;
  p.splits = ceil_div(K, p.k_each);
  p.whole = (int)(p.splits == 1 ? tiles : tiles - others);
  p.partial_bytes = (size_t)(tiles - p.whole) * p.splits * p.bm * p.bn * sizeof(float);
  return p;
}

// Rows of whole 16-byte pieces on 16-byte boundaries, in a tile whose byte offsets fit 31 bits.
bool can_go_direct(const void* p, long long ld, int cols, int dtype) {
  return dtype != RNNT_MI355X_FP32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && cols % 8 == 0 && ld < (1 << 21);
}

size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

template <class T>
int gemm_of(int product, int block, bool direct, const GemmArgs& g, hipStream_t st) {
  if constexpr (T::code == RNNT_MI355X_FP32) return layer_gemm_fp32(product, block, direct, &g, st);
  else if constexpr (T::code == RNNT_MI355X_BF16) return layer_gemm_bf16(product, block, direct, &g, st);
  else return layer_gemm_fp16(product, block, direct, &g, st);
}

template <class T>
int grads_of(bool direct, const GemmArgs& dx, const GemmArgs& dk, hipStream_t st) {
  if constexpr (T::code == RNNT_MI355X_FP32) return layer_grads_fp32(direct, &dx, &dk, st);
  else if constexpr (T::code == RNNT_MI355X_BF16) return layer_grads_bf16(direct, &dx, &dk, st);
  else return layer_grads_fp16(direct, &dx, &dk, st);
}

GemmArgs product_args(const Plan& p, const void* a, long long a_ld, const void* b, long long b_ld, int M, int N, int K, const Epilogue& e, void* partial) {
  GemmArgs g;
  g.a = a;
  g.b = b;
  g.a_ld = a_ld;
  g.b_ld = b_ld;
  g.M = M;
  g.N = N;
  g.K = K;
  g.tiles_m = p.tiles_m;
  g.tiles_n = p.tiles_n;
  g.whole = p.whole;
  g.splits = p.splits;
  g.k_each = p.k_each;
  g.partial = static_cast<float*>(partial);
  g.e = e;
  return g;
}

JoinArgs join_args(const Plan& p, const GemmArgs& g) {
  JoinArgs j{g, p.bm, p.bn, p.splits >= 8 ? 8 : p.splits >= 4 ? 4 : 2, 0u};
  if (p.bm * p.bn / 8 < 256 / j.lanes) j.lanes = 8;
  j.blocks = (unsigned)(p.tiles_m * p.tiles_n - p.whole) * (unsigned)(p.bm * p.bn / 8 / (256 / j.lanes));
  return j;
}
JoinArgs no_join() {
  JoinArgs j{};
  j.lanes = 1;
  return j;
}

template <class T>
int run_join(const JoinArgs& a, const JoinArgs& b, const DbArgs& db, hipStream_t st) {
  const unsigned blocks = a.blocks + b.blocks + (db.db ? (unsigned)ceil_div(db.N, 16) : 0u);
  if (blocks == 0) return RNNT_MI355X_OK;
  k_layer_join<T><<<blocks, 256, 0, st>>>(a, b, db);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}

template <class T>
int run_product(int product, const Plan& p, const GemmArgs& g, hipStream_t st) {
  return p.block == kBlockRows ? launch_rows<T>(g, st) : gemm_of<T>(product, p.block, p.direct, g, st);
}

Epilogue plain_output(void* out, long long ld) {
  Epilogue e;
  e.out = out;
  e.bias = e.residual = nullptr;
  e.aux = nullptr;
  e.out_ld = ld;
  e.residual_ld = 0;
  e.act = kLinear;
  e.drop = drop_args(0, 0, 0, nullptr);
  return e;
}

int check_layer(const rnnt_mi355x_layer* l) {
  if (!l || l->rows < 1 || l->in < 1 || l->out < 1 || l->dtype < 0 || l->dtype > RNNT_MI355X_FP16 || l->act < kLinear || l->act > kSilu ||
      l->drop16 < 0 || l->drop16 > 65535 || l->x_stride < l->in || l->kernel_stride < l->out)
    return RNNT_MI355X_INVALID_VALUE;
  // 32-bit indexes inside an operand's rows and of its tiles; a launch has fewer than 2^32 threads: 2^24 tiles of 64 rows
  if (l->rows > (1ll << 30) - 64 || l->in > (1 << 24) || l->out > (1 << 24) || ((l->rows + 63) / 64) * ((l->in + 63) / 64) > 0x7fffffffll ||
      ((l->rows + 63) / 64) * ((l->out + 63) / 64) > 0x7fffffffll || (long long)((l->in + 63) / 64) * ((l->out + 63) / 64) > 0x7fffffffll)
    return RNNT_MI355X_UNSUPPORTED_SIZE;
  return RNNT_MI355X_OK;
}

int saved_by(const rnnt_mi355x_layer* l) {
  if (l->act == kLinear) return kNothing;
  if (l->aux) return kPreActivation;
  const bool from_y = !l->residual && (l->act == kRelu || (l->act == kTanh && l->dtype == RNNT_MI355X_FP32));
  return from_y && l->y ? kOutput : -1;
}

// Rows in the workspace: whole 16-byte pieces, and no multiple of 4 KiB apart, which puts the same piece of all rows of a
// tile into the same few memory channels: 32768 x 4096 x 1024 in bfloat16 ran 300 us with such rows of x and 257 us with
// rows 128 bytes longer.
long long workspace_stride(int cols, int dtype) {
  const long long e = dtype == RNNT_MI355X_FP32 ? 4 : 2, ld = ((long long)cols + 7) & ~7ll;
  return ld * e % 4096 == 0 ? ld + 128 / e : ld;
}

// An operand as its product reads it: where it is, or copied to `at` of the workspace.
struct Operand {
  const void* p;
  long long ld, rows;
  int cols;
  bool pack;
  size_t at, bytes;
};
// Copying costs a read and a write of the operand; the product reads it at twice the speed or better.  6151 x 515 x 1030 in
// float16, forward: 46 us from the rows as they are, 21 us copies included.  Operands that few rows use stay where they are, and those of 2^33 elements.
Operand operand(const void* p, long long ld, long long rows, int cols, int dtype, bool often) {
  Operand o{p, ld, rows, cols, false, 0, 0};
  if (dtype != RNNT_MI355X_FP32 && often && !can_go_direct(p, ld, cols, dtype) && cols < (1 << 20) && rows * ((cols + 7) / 8) < 1ll << 30) {
    o.pack = true;
    o.ld = workspace_stride(cols, dtype);
    o.bytes = align_up((size_t)rows * o.ld * 2);
  }
  return o;
}
bool direct(const Operand& o, int dtype) { return o.pack || can_go_direct(o.p, o.ld, o.cols, dtype); }
// What copies an operand; afterwards it is its copy.
PackArgs pack_of(Operand& o, long long src_ld, char* ws) {
  PackArgs p{static_cast<const uint16_t*>(o.p), reinterpret_cast<uint16_t*>(ws + o.at), src_ld, o.ld, o.rows, o.cols, 0u};
  if (!o.pack) return p;
  p.blocks = (unsigned)((o.rows * ((o.cols + 7) / 8) + 255) / 256);
  o.p = ws + o.at;
  return p;
}

constexpr int kOften = 512;  // rows that share the kernel

struct ForwardPlan {
  Operand x, kernel;
  Plan y;
  size_t partial_at, bytes;
};
ForwardPlan plan_forward(const rnnt_mi355x_layer* l) {
  ForwardPlan f;
  const bool often = l->rows >= kOften;
  // x is read once for every 256 columns or fewer: worth a copy from a few blocks on
  f.x = operand(l->x, l->x_stride, l->rows, l->in, l->dtype, often);
  f.kernel = operand(l->kernel, l->kernel_stride, l->in, l->out, l->dtype, often);
  f.kernel.at = f.x.at + f.x.bytes;
  f.partial_at = f.kernel.at + f.kernel.bytes;
  f.y = plan_product(kForward, l->dtype, (int)l->rows, l->out, l->in, direct(f.x, l->dtype) && direct(f.kernel, l->dtype));
  f.bytes = f.partial_at + f.y.partial_bytes;
  return f;
}

struct BackwardPlan {
  bool need_dz;  // else dz is dy
  Operand x, kernel, dz;
  size_t sums_at, partial_at, bytes;
  int dz_rows, dz_blocks, dz_across;  // the dz pass: rows of a block, blocks down and across
  Plan dx, dk;
};
BackwardPlan plan_backward(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride) {
  BackwardPlan b;
  const int M = (int)l->rows, dtype = l->dtype;
  const size_t e = dtype == RNNT_MI355X_FP32 ? 4 : 2;
  const bool often = M >= kOften;
  // the pass that makes dz also puts a dy whose rows lie badly on boundaries
  b.need_dz = l->act != kLinear || l->drop16 != 0 || (often && dtype != RNNT_MI355X_FP32 && !can_go_direct(dy, dy_stride, l->out, dtype));
  b.dz = Operand{dy, dy_stride, M, l->out, false, 0, 0};
  if (b.need_dz) {
    b.dz.ld = workspace_stride(l->out, dtype);
    b.dz.pack = dtype != RNNT_MI355X_FP32 && b.dz.ld < (1 << 21);
    b.dz.bytes = align_up((size_t)M * b.dz.ld * e);
  }
  b.x = operand(l->x, l->x_stride, M, l->in, dtype, often);
  b.kernel = operand(l->kernel, l->kernel_stride, l->in, l->out, dtype, often);
  b.x.at = b.dz.bytes;
  b.kernel.at = b.x.at + b.x.bytes;
  b.sums_at = b.kernel.at + b.kernel.bytes;
  // about 8192 blocks, in rows of 8, and at most 2048 partial sums a column
  b.dz_across = ceil_div(l->out, kDzGroups * 8);
  const long long most = ((long long)M / 2048 + 7) / 8 * 8;
  long long rows = ((long long)M * b.dz_across / 8192 + 7) / 8 * 8;
  if (rows < most) rows = most;
  b.dz_rows = (int)(rows < 8 ? 8 : rows);
  b.dz_blocks = ceil_div(M, b.dz_rows);
  b.partial_at = b.sums_at + align_up((size_t)b.dz_blocks * l->out * sizeof(float));
  b.dx = plan_product(kInputGrad, dtype, M, l->in, l->out, direct(b.dz, dtype) && direct(b.kernel, dtype));
  b.dk = plan_product(kKernelGrad, dtype, l->in, l->out, M, direct(b.dz, dtype) && direct(b.x, dtype));
  b.bytes = b.partial_at + align_up(b.dx.partial_bytes) + b.dk.partial_bytes;
  return b;
}

template <class T>
int forward(const rnnt_mi355x_layer* l, ForwardPlan f, void* workspace, hipStream_t st) {
  Epilogue e = plain_output(l->y, l->out);
  e.bias = l->bias;
  e.residual = l->residual;
  e.residual_ld = l->residual_stride;
  e.aux = l->act == kLinear ? nullptr : l->aux;
  e.act = l->act;
  e.drop = drop_args(l->drop16, l->seed, l->offset, l->offset_dev);
  char* ws = static_cast<char*>(workspace);
  const PackArgs px = pack_of(f.x, l->x_stride, ws), pk = pack_of(f.kernel, l->kernel_stride, ws);
  if (px.blocks + pk.blocks) {
    k_layer_pack<<<px.blocks + pk.blocks, 256, 0, st>>>(px, pk);
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
  }
  const GemmArgs g = product_args(f.y, f.x.p, f.x.ld, f.kernel.p, f.kernel.ld, (int)l->rows, l->out, l->in, e, ws + f.partial_at);
  const int rc = run_product<T>(kForward, f.y, g, st);
  return rc == RNNT_MI355X_OK ? run_join<T>(join_args(f.y, g), no_join(), DbArgs{}, st) : rc;
}

template <class T>
int backward(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride, void* dx, void* dkernel, void* dbias, void* workspace, int from,
             hipStream_t st) {
  BackwardPlan b = plan_backward(l, dy, dy_stride);
  const int M = (int)l->rows;
  char* ws = static_cast<char*>(workspace);
  if (b.need_dz) b.dz.p = ws + b.dz.at;
  float* sums = reinterpret_cast<float*>(ws + b.sums_at);
  if (!dx) b.kernel.pack = false;
  if (!dkernel) b.x.pack = false;
  const PackArgs px = pack_of(b.x, l->x_stride, ws), pk = pack_of(b.kernel, l->kernel_stride, ws);
  DzArgs a;
  a.dy = dy;
  a.saved = from == kPreActivation ? l->aux : l->y;
  a.dz = b.need_dz ? ws + b.dz.at : nullptr;
  a.partial = dbias ? sums : nullptr;
  a.dy_ld = dy_stride;
  a.dz_ld = b.dz.ld;
  a.M = M;
  a.N = l->out;
  a.rows = b.dz_rows;
  a.across = b.dz_across;
  a.blocks = b.need_dz || dbias ? (unsigned)b.dz_across * (unsigned)b.dz_blocks : 0u;
  a.act = l->act;
  a.from = from;
  a.drop = drop_args(l->drop16, l->seed, l->offset, l->offset_dev);
  if (a.blocks + px.blocks + pk.blocks) {
    k_layer_dz<T><<<a.blocks + px.blocks + pk.blocks, kDzGroups * kDzLanes, 0, st>>>(a, px, pk);
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
  }
  const GemmArgs gx = product_args(b.dx, b.dz.p, b.dz.ld, b.kernel.p, b.kernel.ld, M, l->in, l->out, plain_output(dx, l->in), ws + b.partial_at);
  const GemmArgs gk = product_args(b.dk, b.x.p, b.x.ld, b.dz.p, b.dz.ld, l->in, l->out, M, plain_output(dkernel, l->out), ws + b.partial_at + align_up(b.dx.partial_bytes));
  int rc = RNNT_MI355X_OK;
  if (dx && dkernel && b.dx.block == kBlock128x128 && b.dk.block == kBlock128x128 && b.dx.direct == b.dk.direct) {
    rc = grads_of<T>(b.dx.direct, gx, gk, st);
  } else {
    if (dx) rc = run_product<T>(kInputGrad, b.dx, gx, st);
    if (rc == RNNT_MI355X_OK && dkernel) rc = run_product<T>(kKernelGrad, b.dk, gk, st);
  }
  if (rc == RNNT_MI355X_OK)
    rc = run_join<T>(dx ? join_args(b.dx, gx) : no_join(), dkernel ? join_args(b.dk, gk) : no_join(), DbArgs{sums, dbias, b.dz_blocks, l->out}, st);
  return rc;
}

}  // namespace

extern "C" int rnnt_mi355x_layer_workspace_bytes(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride, size_t* forward_bytes,
                                                 size_t* backward_bytes) {
  const int rc = check_layer(l);
  if (rc != RNNT_MI355X_OK) return rc;
  if (backward_bytes && dy_stride < l->out) return RNNT_MI355X_INVALID_VALUE;
  if (forward_bytes) *forward_bytes = plan_forward(l).bytes;
  if (backward_bytes) *backward_bytes = plan_backward(l, dy, dy_stride).bytes;
  return RNNT_MI355X_OK;
}

extern "C" int rnnt_mi355x_layer_forward(const rnnt_mi355x_layer* l, void* workspace, void* hip_stream) {
  const int rc = check_layer(l);
  if (rc != RNNT_MI355X_OK) return rc;
  if (!l->x || !l->kernel || !l->y || (l->residual && l->residual_stride < l->out)) return RNNT_MI355X_INVALID_VALUE;
  const ForwardPlan f = plan_forward(l);
  if (!workspace && f.bytes) return RNNT_MI355X_INVALID_VALUE;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (l->dtype) {
    case RNNT_MI355X_FP32: return forward<Fp32>(l, f, workspace, st);
    case RNNT_MI355X_BF16: return forward<Bf16>(l, f, workspace, st);
  }
  return forward<Fp16>(l, f, workspace, st);
}

extern "C" int rnnt_mi355x_layer_backward(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride, void* dx, void* dkernel,
                                          void* dbias, void* workspace, void* hip_stream) {
  const int rc = check_layer(l);
  if (rc != RNNT_MI355X_OK) return rc;
  const int from = saved_by(l);
  if (!l->x || !l->kernel || !dy || dy_stride < l->out || !workspace || from < 0) return RNNT_MI355X_INVALID_VALUE;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (l->dtype) {
    case RNNT_MI355X_FP32: return backward<Fp32>(l, dy, dy_stride, dx, dkernel, dbias, workspace, from, st);
    case RNNT_MI355X_BF16: return backward<Bf16>(l, dy, dy_stride, dx, dkernel, dbias, workspace, from, st);
  }
  return backward<Fp16>(l, dy, dy_stride, dx, dkernel, dbias, workspace, from, st);
}
