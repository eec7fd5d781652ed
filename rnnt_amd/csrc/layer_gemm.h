// Matrix product of the Dense layer (layer.hip): D[m][n] = sum_k A(m,k) B(k,n) on the matrix cores, for the three products
// of a layer -- forward (x W), input gradient (dz W^T), kernel gradient (x^T dz) -- from the operands as they lie in
// memory.
//
// An operand is "k-fast" (k contiguous: x and dz in the first two, W in the second) or "k-slow" (k strided: W in the
// first, both in the third).  Both are staged in LDS as they are, 16 bytes of consecutive elements at a time; the matrix
// instruction wants eight consecutive k of a row per lane, which a k-fast tile gives with one 16-byte LDS read and a
// k-slow tile with two transposing 8-byte reads (ds_read_b64_tr_b16: a group of 16 lanes reads 4 k x 16 columns and each
// lane receives the 4 k of one column).  16-byte pieces are XOR-permuted inside a row so that the lanes served together
// fall into different banks.
//
// float32: the matrix cores do 256 float32 operations a cycle and CU, but 4096 in 16 bits.  A float32 is split into three
// bfloat16 (8 + 8 + 8 bits of significand: x = h + m + l up to 2^-25 of x), and the product is the six partial products
// above 2^-24: hh + hm + mh + hl + lh + mm, each exact in float32 and accumulated there.  What is left out (ml, lm, ll) is
// below 2^-24 of |a||b|, half a rounding of the float32 product itself.  Parts below 2^-126 may count as zero, so operands
// below 2^-102 lose their last bits.
#pragma once
#include "op_util.h"

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v lds_s4;

template <class T>
constexpr int kPlanes = T::code == RNNT_MI355X_FP32 ? 3 : 1;

// What a product's result goes through; `act` and the pointers are the same for every element.
struct Epilogue {
  void* out;             // [M, N] of the layer's type, or float32 when `partial`
  const void* bias;      // nullable [N]
  const void* residual;  // nullable, rows residual_ld apart
  void* aux;             // nullable [M, N]: the pre-activation, for the backward pass
  long long out_ld, residual_ld;
  int act;
  DropArgs drop;
};

enum Act { kLinear = 0, kTanh = 1, kRelu = 2, kGelu = 3, kSilu = 4 };

__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// tanh z = 1 - 2 / (e^2z + 1); exact limits at +-inf, absolute error below 2^-22
__device__ __forceinline__ float tanh_of(float z) { return 1.f - 2.f * __builtin_amdgcn_rcpf(exp_fast(2.f * z) + 1.f); }
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-z)); }
// Phi(z), the normal distribution's function, and e = exp(-z^2/2): erfc(t) = (a1 p + ... + a5 p^5) exp(-t^2),
// p = 1 / (1 + 0.3275911 t), t >= 0, to 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26)
__device__ __forceinline__ float normal_of(float z, float& e) {
  const float t = fabsf(z) * 0.70710678118654752f;
  e = exp_fast(-t * t);
  const float p = __builtin_amdgcn_rcpf(fmaf(0.3275911f, t, 1.f));
  const float q = p * fmaf(p, fmaf(p, fmaf(p, fmaf(p, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  const float tail = 0.5f * q * e;  // 1 - Phi(|z|)
  return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case kTanh: return tanh_of(z);
    case kRelu: return z < 0.f ? 0.f : z;  // NaN stays
    case kGelu: {
      float e;
      const float p = normal_of(z, e);
      return z == -INFINITY ? 0.f : z * p;
    }
    case kSilu: return z == -INFINITY ? 0.f : z * sigmoid_of(z);
  }
  return z;
}
// act'(z)
__device__ __forceinline__ float slope_of(float z, int act) {
  switch (act) {
    case kTanh: {
      // 1 - tanh^2 = 4 q / (1 + q)^2 with q = e^-2|z|: no cancellation far out
      const float q = exp_fast(-2.f * fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + q);
      return 4.f * q * r * r;
    }
    case kRelu: return z > 0.f ? 1.f : 0.f;
    case kGelu: {
      float e;
      const float p = normal_of(z, e);
      return fabsf(z) > 20.f ? p : fmaf(z * 0.3989422804014327f, e, p);
    }
    case kSilu: {
      const float p = sigmoid_of(z);
      return fabsf(z) > 100.f ? (z > 0.f ? 1.f : 0.f) : p * fmaf(z, 1.f - p, 1.f);
    }
  }
  return 1.f;
}

// The pre-activation that the backward pass reads: float32 for float32 and float16 layers, float16 for bfloat16 ones.
// bfloat16 would put a rounding of 2^-9 into act'(z) on top of dz's own; float16 has 2^-12, at the same size.  Its range is
// 2^-24 .. 65504: beyond it act' is at its limits, and below it only the sign of z counts.
template <class T>
struct AuxOf { using type = Fp32; };
template <>
struct AuxOf<Bf16> { using type = Fp16; };
template <class T>
__device__ __forceinline__ float aux_value(float z) {
  if constexpr (T::code != RNNT_MI355X_BF16) return z;
  // fminf / fmaxf drop NaN, which has to stay
  const float c = z != z ? z : fminf(fmaxf(z, -65504.f), 65504.f);
  return fabsf(c) < 5.9604645e-8f && c != 0.f ? copysignf(5.9604645e-8f, c) : c;
}

// Eight consecutive results of a row, n of them inside it.
template <class T>
__device__ __forceinline__ void finish8(const Epilogue& e, const DropArgs& drop, long long m, int n0, int n, float (&v)[8]) {
  using E = typename T::elem;
  const bool full = n >= 8;
  if (e.bias) {
    float b[8];
    const E* p = static_cast<const E*>(e.bias) + n0;
    if (full) unpack8<T>(load8_raw<T>(p), b);
    else load_some<T>(p, n, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
  }
  if (e.aux) {
    using A = typename AuxOf<T>::type;
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = aux_value<T>(v[i]);
    typename A::elem* p = static_cast<typename A::elem*>(e.aux) + m * e.out_ld + n0;
    if (full) store8<A>(p, z);
    else store_some<A>(p, n, z);
  }
  if (e.act != kLinear) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_of(v[i], e.act);
  }
  if (drop.drop) drop8(drop, (uint32_t)m, (uint32_t)n0 >> 3, v);
  if (e.residual) {
    float r[8];
    const E* p = static_cast<const E*>(e.residual) + m * e.residual_ld + n0;
    if (full) unpack8<T>(load8_raw<T>(p), r);
    else load_some<T>(p, n, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  E* p = static_cast<E*>(e.out) + m * e.out_ld + n0;
  if (full) store8<T>(p, v);
  else store_some<T>(p, n, v);
}

// ---- staging ------------------------------------------------------------------------------------------------------------
// Three bfloat16 whose sum is x up to 2^-25 |x|.  x past bfloat16's range, or no number, gives infinities and NaN among
// the parts; their products are NaN and the result is computed again (fix_nan).
__device__ __forceinline__ void split8(const float (&v)[8], u4 (&q)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t ha = float_to_bf16_bits(a), hb = float_to_bf16_bits(b), w = ha | (hb << 16);
      q[p][i] = w;
      a -= __uint_as_float(w << 16);
      b -= __uint_as_float(w & 0xffff0000u);
    }
  }
}

// A tile of an operand: R rows (of the result's m or n) by BK.  In LDS it is a sequence of 16-byte pieces of eight
// elements: k-fast row by row (BK / 8 pieces), k-slow k by k (R / 8 pieces); float32 has three such planes.
template <class T, bool KS, int R, int BK, int THREADS>
struct Tile {
  using E = typename T::elem;
  static constexpr int kPieces = R * BK / 8, kEach = kPieces / THREADS, kRow = KS ? R / 8 : BK / 8;
  static constexpr int kPlaneBytes = R * BK * 2, kBytes = kPlaneBytes * kPlanes<T>;
  static_assert(kPieces % THREADS == 0 && (!KS || R >= 64) && (BK == 32 || BK == 64), "tile shape");

  // place p holds row p / kRow and piece (p % kRow) ^ permute(row): k-fast reads take one piece of 8 consecutive rows
  // together, k-slow reads 32 bytes of 4 consecutive k
  static __device__ __forceinline__ int permute(int row) { return KS ? (row & 3) << 1 : kRow == 8 ? row & 7 : (row >> 1) & 3; }

  // Registers: a thread's pieces of the tile at row r0 (of r_end) and k0 (of k_end); zeros past both ends.
  static __device__ __forceinline__ void load(Raw8<T> (&raw)[kEach], const E* base, long long ld, int r0, int r_end, int k0, int k_end) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = j * THREADS + threadIdx.x, row = p / kRow, piece = (p % kRow) ^ permute(row);
      // outer: the strided index, inner: the contiguous one
      const int outer = KS ? k0 + row : r0 + row, inner = KS ? r0 + 8 * piece : k0 + 8 * piece;
      const int outer_end = KS ? k_end : r_end, inner_end = KS ? r_end : k_end;
      const E* at = base + (long long)outer * ld + inner;
      if (outer < outer_end && inner + 8 <= inner_end) {
        raw[j] = load8_raw<T>(at);
      } else {
        E some[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) some[i] = 0;
        if (outer < outer_end) {
#pragma unroll
          for (int i = 0; i < 7; ++i)
            if (inner + i < inner_end) some[i] = at[i];
        }
        __builtin_memcpy(&raw[j], some, sizeof(some));
      }
    }
  }
  static __device__ __forceinline__ void store(const Raw8<T> (&raw)[kEach], char* lds) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = j * THREADS + threadIdx.x;
      if constexpr (kPlanes<T> == 3) {
        float v[8];
        u4 q[3];
        unpack8<T>(raw[j], v);
        split8(v, q);
#pragma unroll
        for (int s = 0; s < 3; ++s) *reinterpret_cast<u4*>(lds + s * kPlaneBytes + p * 16) = q[s];
      } else {
        *reinterpret_cast<u4*>(lds + p * 16) = raw[j].q[0];
      }
    }
  }

  // Straight into LDS (16-bit types, rows on 16-byte boundaries): a wavefront writes 1 KiB of consecutive places.  A piece
  // that is not there gets an address past the buffer's end, for which the hardware's bounds check delivers zeros.
  static __device__ __forceinline__ void load_direct(char* lds, const E* base, long long ld, int r0, int r_end, int k0, int k_end) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const E* corner = base + (KS ? (long long)k0 * ld + r0 : (long long)r0 * ld + k0);
    // bytes from the corner that any piece inside the operand can reach
    const long long rows = KS ? k_end - k0 : r_end - r0, last = KS ? r_end - r0 : k_end - k0;
    const long long span = ((rows - 1) * ld + last) * 2;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(corner), 0, (int)(span < 0x7ffffff0ll ? span : 0x7ffffff0ll), 0x00020000);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = j * THREADS + threadIdx.x, row = p / kRow, piece = (p % kRow) ^ permute(row);
      const bool in = KS ? k0 + row < k_end && r0 + 8 * piece < r_end : r0 + row < r_end && k0 + 8 * piece < k_end;
      const int offset = in ? (row * (int)ld + 8 * piece) * 2 : 0x7ffffff0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + (j * THREADS + wave * 64) * 16), 16, offset, 0, 0, 0);
    }
  }

  // The eight k of rows r .. r+31 (one a lane, twice) that step s of 16 k takes: lanes 32.. have the second eight.
  static __device__ __forceinline__ u4 frag(const char* lds, int r, int s, int lane) {
    if constexpr (!KS) {
      const int row = r + (lane & 31), piece = (2 * s + (lane >> 5)) ^ permute(row);
      return *reinterpret_cast<const u4*>(lds + (row * kRow + piece) * 16);
    } else {
      union {
        u4 q;
        s4v h[2];
      } f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 16 * s + 8 * (lane >> 5) + 4 * j + ((lane & 15) >> 2), c = r + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        f.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(lds + (k * kRow + ((c >> 3) ^ permute(k))) * 16 + (c & 7) * 2));
      }
      return f.q;
    }
  }
};

template <class T>
__device__ __forceinline__ f16v mfma(const u4& a, const u4& b, const f16v& c) {
  if constexpr (T::code == RNNT_MI355X_FP16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

struct GemmArgs {
  const void *a, *b;
  long long a_ld, b_ld;
  int M, N, K;
  int tiles_m, tiles_n, splits, k_each;  // k_each: multiple of BK, the k that one of the splits takes
  float* partial;                        // splits > 1: [splits][M][N]
  Epilogue e;
};

// A float32 result that is NaN may owe it to the split of an infinite or overflowing operand: it is computed again in
// float32.  Nothing of a finite product comes here.
template <bool A_KS, bool B_KS>
__device__ __attribute__((noinline)) float product_again(const float* a, const float* b, long long a_ld, long long b_ld, long long m, int n, int k0, int k1) {
  float s = 0.f;
  for (int k = k0; k < k1; ++k)
    s = fmaf(A_KS ? a[(long long)k * a_ld + m] : a[m * a_ld + k], B_KS ? b[(long long)k * b_ld + n] : b[(long long)n * b_ld + k], s);
  return s;
}

// Blocks are dealt to the 8 XCDs in turn; consecutive work of one XCD shares operands in its L2, so tiles are numbered
// XCD by XCD, and inside that in columns of 8 tile rows.
__device__ __forceinline__ void tile_of(const GemmArgs& g, int& tm, int& tn, int& split) {
  const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.splits, id = blockIdx.x;
  const int xcd = id & 7, each = total >> 3, rest = total & 7;
  const int w = xcd * each + min(xcd, rest) + (id >> 3);
  split = w / tiles;
  const int t = w - split * tiles, band = 8 * g.tiles_n, band_id = t / band, in = t - band_id * band;
  const int rows = min(8, g.tiles_m - 8 * band_id);
  tm = 8 * band_id + in % rows;
  tn = in / rows;
}

// WM x WN of the result per wavefront in 32 x 32 blocks; two LDS buffers, the next tile on its way while one is used.
template <class T, bool A_KS, bool B_KS, int BM, int BN, int BK, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void k_layer_gemm(GemmArgs g) {
  constexpr int kThreads = (BM / WM) * (BN / WN) * 64, IM = WM / 32, IN = WN / 32;
  using TA = Tile<T, A_KS, BM, BK, kThreads>;
  using TB = Tile<T, B_KS, BN, BK, kThreads>;
  using E = typename T::elem;
  constexpr int kStage = TA::kBytes + TB::kBytes, kOut = (kThreads / 64) * 32 * WN * 4;
  // two objects, so that the compiler sees that a tile on its way does not touch the one being read
  __shared__ __attribute__((aligned(16))) char buf0[kStage > kOut ? kStage : kOut];
  __shared__ __attribute__((aligned(16))) char buf1[kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  int tm, tn, split;
  tile_of(g, tm, tn, split);
  const int m0 = tm * BM, n0 = tn * BN, k0 = split * g.k_each, k1 = min(g.K, k0 + g.k_each);
  const E *a = static_cast<const E*>(g.a), *b = static_cast<const E*>(g.b);

  f16v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  Raw8<T> ra[DIRECT ? 1 : TA::kEach], rb[DIRECT ? 1 : TB::kEach];
  auto fetch = [&](char* buf, int k) {
    if constexpr (DIRECT) {
      TA::load_direct(buf, a, g.a_ld, m0, g.M, k, k1);
      TB::load_direct(buf + TA::kBytes, b, g.b_ld, n0, g.N, k, k1);
    } else {
      TA::load(ra, a, g.a_ld, m0, g.M, k, k1);
      TB::load(rb, b, g.b_ld, n0, g.N, k, k1);
    }
  };
  auto put = [&](char* buf) {
    if constexpr (!DIRECT) {
      TA::store(ra, buf);
      TB::store(rb, buf + TA::kBytes);
    }
  };
  auto multiply = [&](const char* buf) {
#pragma unroll
    for (int s = 0; s < BK / 16; ++s) {
      u4 fa[kPlanes<T>][IM], fb[kPlanes<T>][IN];
#pragma unroll
      for (int p = 0; p < kPlanes<T>; ++p) {
#pragma unroll
        for (int i = 0; i < IM; ++i) fa[p][i] = TA::frag(buf + p * TA::kPlaneBytes, wm + 32 * i, s, lane);
#pragma unroll
        for (int j = 0; j < IN; ++j) fb[p][j] = TB::frag(buf + TA::kBytes + p * TB::kPlaneBytes, wn + 32 * j, s, lane);
      }
      // the kernel's side is the instruction's first operand: a lane then holds four consecutive n of one m
#pragma unroll
      for (int pa = 0; pa < kPlanes<T>; ++pa)
#pragma unroll
        for (int pb = 0; pb + pa < kPlanes<T>; ++pb)
#pragma unroll
          for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j) acc[i][j] = mfma<T>(fb[pb][j], fa[pa][i], acc[i][j]);
    }
  };
  auto step = [&](char* now, char* next, int k) {
    const bool more = k + BK < k1;
    if (more) fetch(next, k + BK);
    multiply(now);
    if (more) put(next);
    __syncthreads();
  };
  fetch(buf0, k0);
  put(buf0);
  __syncthreads();
  for (int k = k0; k < k1; k += 2 * BK) {
    step(buf0, buf1, k);
    if (k + BK < k1) step(buf1, buf0, k + BK);
  }

  // Through LDS into rows: eight consecutive n a lane, 32 rows of this wavefront at a time.  Pieces of four are permuted
  // by the row, as lanes write one column of 32 rows.
  constexpr int kQuads = WN / 4, kPerRow = WN / 8, kRows = 64 / kPerRow;
  float* mine = reinterpret_cast<float*>(buf0) + wave * 32 * WN;
  const int quad_mask = kQuads < 16 ? kQuads - 1 : 15;
  DropArgs drop = g.e.drop;
  if (drop.drop) load_offset(drop);
#pragma unroll
  for (int i = 0; i < IM; ++i) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = lane & 31, quad = (8 * j + 2 * q + (lane >> 5)) ^ (row & quad_mask);
        *reinterpret_cast<f4*>(mine + row * WN + 4 * quad) = f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 32 / kRows; ++r) {
      const int row = r * kRows + lane / kPerRow, c = lane % kPerRow;
      const f4 lo = *reinterpret_cast<const f4*>(mine + row * WN + 4 * ((2 * c) ^ (row & quad_mask)));
      const f4 hi = *reinterpret_cast<const f4*>(mine + row * WN + 4 * ((2 * c + 1) ^ (row & quad_mask)));
      float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const long long m = m0 + wm + 32 * i + row;
      const int n = n0 + wn + 8 * c, left = g.N - n;
      if (m < g.M && left > 0) {
        if constexpr (kPlanes<T> == 3) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (v[x] != v[x] && x < left) v[x] = product_again<A_KS, B_KS>(a, b, g.a_ld, g.b_ld, m, n + x, k0, k1);
        }
        if (g.splits > 1) {
          float* p = g.partial + ((long long)split * g.M + m) * g.N + n;
          if (left >= 8) store8<Fp32>(p, v);
          else store_some<Fp32>(p, left, v);
        } else {
          finish8<T>(g.e, drop, m, n, left, v);
        }
      }
    }
  }
}

}  // namespace
