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

// tanh z = 1 - 2 / (e^2z + 1), exact limits at +-inf; below 0.3, where that difference cancels, the series to z^9 (the next
// term is 2^-24 of the sum there).  Relative error below 2^-20 everywhere.
__device__ __forceinline__ float tanh_of(float z) {
  const float q = z * z, far = 1.f - 2.f * __builtin_amdgcn_rcpf(exp_fast(2.f * z) + 1.f);
  const float near = fmaf(fmaf(fmaf(fmaf(62.f / 2835.f, q, -17.f / 315.f), q, 2.f / 15.f), q, -1.f / 3.f) * q, z, z);
  return fabsf(z) < 0.3f ? near : far;
}
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.f + exp_fast(-z)); }
// Phi(z), the normal distribution's function, and e = exp(-z^2/2).  1 - Phi(a) = e R(a) with R smooth and positive: a polynomial
// in p = 1 / (1 + 0.3 a), fitted here by least squares with weights driven to equal relative errors, 1.2e-7 over 0 <= a <= 13.2.
// The tail keeps its digits that way: e's argument adds 1.25 a^2 2^-24, 2e-6 at z = -5 and 1e-5 at -12.
__device__ __forceinline__ float normal_of(float z, float& e) {
  const float a = fabsf(z);
  e = exp_fast(-0.5f * (a * a));
  const float p = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
  float q = fmaf(p, 0.03608877f, -0.15893343f);
  q = fmaf(p, q, 0.20934585f);
  q = fmaf(p, q, -0.05644957f);
  q = fmaf(p, q, 0.13003232f);
  q = fmaf(p, q, 0.09946515f);
  q = fmaf(p, q, 0.1208263f);
  q = fmaf(p, q, 0.11962454f);
  const float tail = p * q * e;  // 1 - Phi(|z|)
  return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float floor_of(float z, float least) { return __builtin_elementwise_maximum(z, least); }  // NaN stays
// z Phi(z) for results of 16 bits: max(z, 0) - a T with a = |z| and T = 1 - Phi(a) = 2^P(a).  P, of degree 8, is fitted to log2 T with
// weights for the relative error of T: 2e-6 up to a = 1, 1.1e-4 < 2^-13 up to 5.9, below which a float16 result is zero, 1e-3 < 2^-9.9
// down to bfloat16's smallest normal numbers; below 2^-122, where T is subnormal, the result is zero.  12 instructions, exp2
// among them, where the form above takes 21 with exp2 and a reciprocal, in an epilogue that is bound by them (32768 x 1024 x 4096
// in bfloat16).
__device__ __forceinline__ float gelu_16(float z) {
  const float a = fminf(fabsf(z), 16.f);  // P(16) = -189
  float p = fmaf(a, 4.4102764e-8f, -2.5647158e-6f);
  p = fmaf(a, p, 6.4033525e-5f);
  p = fmaf(a, p, -9.1116347e-4f);
  p = fmaf(a, p, 8.3481059e-3f);
  p = fmaf(a, p, -5.3563926e-2f);
  p = fmaf(a, p, -4.5882209e-1f);
  p = fmaf(a, p, -1.1511463f);
  p = fmaf(a, p, -1.f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), floor_of(z, 0.f));
}
__device__ __forceinline__ float act_of(float z, int act) {
  switch (act) {
    case kTanh: return tanh_of(z);
    case kRelu: return z < 0.f ? 0.f : z;  // NaN stays
    case kGelu: {
      float e;
      const float p = normal_of(z, e);
      return floor_of(z, -64.f) * p;  // p = 0 there, and 0 times -inf would be NaN
    }
    case kSilu: return floor_of(z, -256.f) * sigmoid_of(z);
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
// bfloat16 would put a rounding of 2^-8 into act'(z) on top of dz's own; float16 has 2^-11, at the same size.  Past its
// range it is infinite, where act' is at its limits; below it only relu's slope asks for more than z = 0 says, and relu
// keeps its slope in the place of z.
template <class T>
struct AuxOf { using type = Fp32; };
template <>
struct AuxOf<Bf16> { using type = Fp16; };

// act(z) of eight values; the choice is the same for all lanes and made once.
template <class T>
__device__ __forceinline__ void act8(int act, float (&v)[8]) {
  switch (act) {
    case kTanh:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_of(v[i], kTanh);
      break;
    case kRelu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_of(v[i], kRelu);
      break;
    case kGelu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = T::code == RNNT_MI355X_FP32 ? act_of(v[i], kGelu) : gelu_16(v[i]);
      break;
    case kSilu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_of(v[i], kSilu);
      break;
  }
}

template <class T>
__device__ __forceinline__ Raw8<T> load_group(const typename T::elem* p, int n) {
  if (n >= 8) return load8_raw<T>(p);
  typename T::elem some[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) some[i] = i < n ? p[i] : 0;
  Raw8<T> r;
  __builtin_memcpy(&r, some, sizeof(some));
  return r;
}
template <class T>
__device__ __forceinline__ void store_group(typename T::elem* p, int n, const float (&v)[8]) {
  if (n >= 8) store8<T>(p, v);
  else store_some<T>(p, n, v);
}

// G times eight consecutive results, of rows m[g] and the same columns n0 .., n of them inside the row.  Stage by stage over
// all G: a group's chain of the generator or of an activation is long, several of them fill each other's waits.  An epilogue
// with gelu, a saved pre-activation and dropout is bound by its vector instructions (about 190 cycles for 64 results), which
// a block alone on its CU cannot hide behind matrix instructions: bfloat16 32768 x 1024 x 4096 310 us without, 400 with.
template <class T, int G>
__device__ __forceinline__ void finish(const Epilogue& e, const DropArgs& drop, const long long (&m)[G], int M, int n0, int n, float (&v)[G][8]) {
  using E = typename T::elem;
  Raw8<T> res[G];
  if (e.residual) {
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (m[g] < M) res[g] = load_group<T>(static_cast<const E*>(e.residual) + m[g] * e.residual_ld + n0, n);
  }
  if (e.bias) {
    float b[8];
    unpack8<T>(load_group<T>(static_cast<const E*>(e.bias) + n0, n), b);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] += b[i];
  }
  if (e.aux) {
    using A = typename AuxOf<T>::type;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = v[g][i];
      if (e.act == kRelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = z[i] > 0.f ? 1.f : z[i];
      }
      if (m[g] < M) store_group<A>(static_cast<typename A::elem*>(e.aux) + m[g] * e.out_ld + n0, n, z);
    }
  }
  if (e.act != kLinear) {
#pragma unroll
    for (int g = 0; g < G; ++g) act8<T>(e.act, v[g]);
  }
  if (drop.drop) {
#pragma unroll
    for (int g = 0; g < G; ++g) drop8(drop, (uint32_t)m[g], (uint32_t)n0 >> 3, v[g]);
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (m[g] >= M) continue;
    if (e.residual) {
      float r[8];
      unpack8<T>(res[g], r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] += r[i];
    }
    store_group<T>(static_cast<E*>(e.out) + m[g] * e.out_ld + n0, n, v[g]);
  }
}

// ---- staging ------------------------------------------------------------------------------------------------------------
// Three bfloat16 whose sum is x up to 2^-25 |x|.  x past bfloat16's range, or no number, gives infinities and NaN among
// the parts; their products are NaN and the result is computed again (product_again).
__device__ __forceinline__ void split8(const float (&v)[8], u4 (&q)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const uint32_t w = pack_bf16(a, b);
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
  static_assert(kPieces % THREADS == 0 && (!KS || R >= 32) && (BK == 32 || BK == 64), "tile shape");

  static_assert((THREADS & (THREADS - 1)) == 0, "");
  static __device__ __forceinline__ int tid() { return threadIdx.x & (THREADS - 1); }  // of the wavefronts that share this tile

  // place p holds row p / kRow and piece (p % kRow) ^ permute(row).  64 banks serve 256 bytes a cycle: k-fast reads take one
  // piece of 16 rows together, k-slow reads 64 bytes of 4 consecutive k.
  static __device__ __forceinline__ int permute(int row) {
    if constexpr (KS) return kRow == 4 ? 0 : kRow == 8 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
    else return kRow == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
  }

  // Registers: a thread's pieces of the tile at row r0 (of r_end) and k0 (of k_end); zeros past both ends.
  static __device__ __forceinline__ void load(Raw8<T> (&raw)[kEach], const E* base, long long ld, int r0, int r_end, int k0, int k_end) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int p = j * THREADS + tid(), row = p / kRow, piece = (p % kRow) ^ permute(row);
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
      const int p = j * THREADS + tid();
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
  // that is not there gets an address past the buffer's end, for which the hardware's bounds check delivers zeros.  One tile
  // after the other, each BK further along k.  Past the end the pieces are zeros.
  struct Source {
    const E* corner;
    long long span, step;  // bytes left from the corner; bytes a tile further
    int left;              // k left
    int offset[kEach], k[kEach];
    __device__ __forceinline__ void init(const E* base, long long ld, int r0, int r_end, int k0, int k_end) {
      corner = base + (KS ? (long long)k0 * ld + r0 : (long long)r0 * ld + k0);
      // rows are whole pieces long: a piece that begins inside is there to its end
      const long long rows = KS ? k_end - k0 : r_end - r0, last = ((KS ? r_end - r0 : k_end - k0) + 7) & ~7;
      span = ((rows - 1) * ld + last) * 2;
      step = (KS ? BK * ld : BK) * 2;
      left = k_end - k0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int p = j * THREADS + tid(), row = p / kRow, piece = (p % kRow) ^ permute(row);
        k[j] = KS ? row : 8 * piece;
        offset[j] = (KS ? r0 + 8 * piece < r_end : r0 + row < r_end) ? (row * (int)ld + 8 * piece) * 2 : 0x7ffffff0;
      }
    }
    __device__ __forceinline__ void next(char* lds) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass has no type for the buffer descriptor and would drop the kernel's launch stub
      const int wave = __builtin_amdgcn_readfirstlane(tid() >> 6);
      auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(corner), 0, (int)(span < 0 ? 0 : span < 0x7ffffff0ll ? span : 0x7ffffff0ll), 0x00020000);
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + (j * THREADS + wave * 64) * 16), 16,
                                                 k[j] < left ? offset[j] : 0x7ffffff0, 0, 0, 0);
      corner = left > BK ? corner + step / 2 : corner;  // past the end nothing is read: the address stays inside
      span -= step;
      left -= BK;
#endif
    }
  };

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
  // `whole` tiles of the result are done by one block each; the others are cut along k into `splits` pieces of k_each (a
  // multiple of BK), whose float32 results go to partial: [other tile][split][BM][BN]
  int tiles_m, tiles_n, whole, splits, k_each;
  float* partial;
  Epilogue e;
};

// A float32 result that is NaN may owe it to the split of an infinite or overflowing operand: it is computed again in
// float32.  Nothing of a finite product comes here.
template <bool A_KS, bool B_KS>
__device__ __forceinline__ float product_again(const float* a, const float* b, long long a_ld, long long b_ld, long long m, int n, int k0, int k1) {
  float s = 0.f;
  for (int k = k0; k < k1 && s == s; ++k)  // once no number, always none
    s = fmaf(A_KS ? a[(long long)k * a_ld + m] : a[m * a_ld + k], B_KS ? b[(long long)k * b_ld + n] : b[(long long)n * b_ld + k], s);
  return s;
}

// What a wavefront's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// All but this wavefront's last N loads into LDS have landed, its LDS reads are done, and every wavefront is here.
template <int N>
__device__ __forceinline__ void landed() {
  static_assert(N < 64, "");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (0 << 8));  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The i-th tile of the result: columns of 8 tile rows, so that tiles in work at the same time share operands.
__device__ __forceinline__ void place_of(const GemmArgs& g, int i, int& tm, int& tn) {
  const int band = 8 * g.tiles_n, band_id = i / band, in = i - band_id * band, rows = min(8, g.tiles_m - 8 * band_id);
  tm = 8 * band_id + in % rows;
  tn = in / rows;
}

// The i-th of n pieces of work for this block.  Blocks are dealt to the 8 XCDs in turn; each XCD gets a consecutive run, as
// it has an L2 of its own.
__device__ __forceinline__ int dealt(int id, int n) {
  const int xcd = id & 7, each = n >> 3, rest = n & 7;
  return xcd * each + min(xcd, rest) + (id >> 3);
}

struct Work {
  int tm, tn, k0, k1;
  float* partial;  // null: the tile is whole
};
template <int BM, int BN>
__device__ __forceinline__ Work work_of(const GemmArgs& g, int id) {
  Work w;
  if (id < g.whole) {
    place_of(g, dealt(id, g.whole), w.tm, w.tn);
    w.k0 = 0;
    w.k1 = g.K;
    w.partial = nullptr;
  } else {
    // split by split: neighbouring tiles of the same k share operands, the splits of a tile share nothing
    const int others = g.tiles_m * g.tiles_n - g.whole, i = dealt(id - g.whole, others * g.splits), split = i / others, tile = i - split * others;
    place_of(g, g.whole + tile, w.tm, w.tn);
    w.k0 = split * g.k_each;
    w.k1 = min(g.K, w.k0 + g.k_each);
    w.partial = g.partial + ((long long)tile * g.splits + split) * (BM * BN);
  }
  return w;
}

// Steps of BK that each of the groups takes.
template <int BK, int GROUPS>
__device__ __forceinline__ int steps_of(const Work& w) {
  return (w.k1 - w.k0 + GROUPS * BK - 1) / (GROUPS * BK);
}
// The groups' sums join in the first group's accumulators, in the groups' order.  place[o]: kSums bytes of LDS for group o > 0,
// not in use for anything else.
template <int IM, int IN, int THREADS>
constexpr int kSums = IM * IN * 16 * THREADS * 4;
template <int IM, int IN, int GROUPS, int THREADS>
__device__ __forceinline__ void join_groups(f16v (&acc)[IM][IN], char* const (&place)[GROUPS], int group) {
  const int tid = threadIdx.x & (THREADS - 1);
#pragma unroll
  for (int o = 1; o < GROUPS; ++o) {
    if (group != o) continue;
    f4* mine = reinterpret_cast<f4*>(place[o]);
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int j = 0; j < IN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f16v& r = acc[i][j];
          mine[((i * IN + j) * 4 + q) * THREADS + tid] = f4{r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]};
        }
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int o = 1; o < GROUPS; ++o) {
    const f4* other = reinterpret_cast<const f4*>(place[o]);
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int j = 0; j < IN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f4 v = other[((i * IN + j) * 4 + q) * THREADS + tid];
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][j][4 * q + x] += v[x];
        }
  }
}

// A wavefront's 32 IM x 32 IN block of the result, through LDS into rows: eight consecutive n a lane, 32 rows by (up to) 64
// columns at a time.  Pieces of four are permuted by the row, as lanes write one column of 32 rows.  lds: kWayOut bytes of
// this wavefront, not in use for anything else.
template <int IN>
constexpr int kWayOut = 32 * 32 * (IN < 2 ? IN : 2) * 4;
template <class T, bool A_KS, bool B_KS, int BN, int IM, int IN>
__device__ __forceinline__ void write_result(const GemmArgs& g, f16v (&acc)[IM][IN], char* lds, int m0, int n0, const Work& w, int wm, int wn) {
  // w.partial: [BM][BN], of which this wavefront's block begins at wm, wn
  constexpr int JN = IN < 2 ? IN : 2, WN = 32 * JN, kQuads = WN / 4, kPerRow = WN / 8, kRows = 64 / kPerRow;
  static_assert(IN % JN == 0, "");
  using E = typename T::elem;
  const E *a = static_cast<const E*>(g.a), *b = static_cast<const E*>(g.b);
  const int lane = threadIdx.x & 63;
  float* mine = reinterpret_cast<float*>(lds);
  const int quad_mask = kQuads < 16 ? kQuads - 1 : 15;
  DropArgs drop = g.e.drop;
  if (drop.drop) load_offset(drop);
#pragma unroll
  for (int i = 0; i < IM; ++i) {
#pragma unroll
    for (int j0 = 0; j0 < IN; j0 += JN) {
      wave_fence();
#pragma unroll
      for (int j = 0; j < JN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = lane & 31, quad = (8 * j + 2 * q + (lane >> 5)) ^ (row & quad_mask);
          const f16v& r = acc[i][j0 + j];
          *reinterpret_cast<f4*>(mine + row * WN + 4 * quad) = f4{r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]};
        }
      wave_fence();
      const int c = lane % kPerRow, n = n0 + 32 * j0 + 8 * c, left = g.N - n;
      if (left <= 0) continue;
      constexpr int G = 2;  // rows a lane has in hand at a time: what registers the accumulators leave
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += G * kRows) {
        float v[G][8];
        long long m[G];
        auto place = [&](int r, int half) {  // of four values of this lane
          const int row = r0 + r * kRows + lane / kPerRow;
          return mine + row * WN + 4 * ((2 * c + half) ^ (row & quad_mask));
        };
        auto take = [&] {
#pragma unroll
          for (int r = 0; r < G; ++r) {
            const f4 lo = *reinterpret_cast<const f4*>(place(r, 0)), hi = *reinterpret_cast<const f4*>(place(r, 1));
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              v[r][x] = lo[x];
              v[r][4 + x] = hi[x];
            }
            m[r] = m0 + 32 * i + r0 + r * kRows + lane / kPerRow;
          }
        };
        take();
        if constexpr (kPlanes<T> == 3) {
          bool bad = false;
#pragma unroll
          for (int r = 0; r < G; ++r)
#pragma unroll
            for (int x = 0; x < 8; ++x) bad |= v[r][x] != v[r][x];
          if (__any(bad)) {
#pragma unroll 1
            for (int t = 0; t < G * 8; ++t) {
              const int r = t >> 3, x = t & 7;
              const long long row = m0 + 32 * i + r0 + r * kRows + lane / kPerRow;
              float* p = place(r, x >> 2) + (x & 3);
              if (*p != *p && x < left && row < g.M) *p = product_again<A_KS, B_KS>(a, b, g.a_ld, g.b_ld, row, n + x, w.k0, w.k1);
            }
            take();
          }
        }
        if (w.partial) {
#pragma unroll
          for (int r = 0; r < G; ++r) store8<Fp32>(w.partial + (wm + m[r] - m0) * BN + wn + n - n0, v[r]);
        } else {
          finish<T, G>(g.e, drop, m, g.M, n, left, v);
        }
      }
    }
  }
}

// Any alignment and type: tiles come through registers, where float32 is split.  WM x WN of the result per wavefront.
// The next tile is on its way while one is multiplied, and other blocks of the CU multiply while this one splits and stores:
// 128 x 128 blocks are held to 168 registers, three on a CU.  Bound by the matrix cores at the clock that they leave: float32
// 8192 x 4096 x 4096 1.36 ms = 202 TFLOP/s, matrix cores busy 65 % of the cycles at 1.54 GHz (the library's float32 product:
// 152 TFLOP/s); two LDS buffers with the splitting between the matrix instructions, one block of 256 x 128 a CU: 203 TFLOP/s.
// GROUPS > 1: as many groups of wavefronts share k, each with a tile of its own (few rows: a block then reads its part of W with
// all its wavefronts and joins their sums in LDS, where pieces of k on several blocks would go through memory).
template <class T, int BM, int BN, int BK, int WM, int WN, int GROUPS>
constexpr int registers_lds() {
  constexpr int kThreads = (BM / WM) * (BN / WN) * 64, kStage = (BM + BN) * BK * 2 * kPlanes<T>, kOut = (kThreads / 64) * kWayOut<WN / 32>;
  constexpr int kOwn = GROUPS == 1 ? kOut : kSums<WM / 32, WN / 32, kThreads>;
  return GROUPS * (kStage > kOwn ? kStage : kOwn);
}
template <class T, bool A_KS, bool B_KS, int BM, int BN, int BK, int WM, int WN, int GROUPS>  // 1 or 4
__device__ __forceinline__ void gemm_registers(const GemmArgs& g, int id, char* lds) {
  constexpr int kThreads = (BM / WM) * (BN / WN) * 64, IM = WM / 32, IN = WN / 32;
  using TA = Tile<T, A_KS, BM, BK, kThreads>;
  using TB = Tile<T, B_KS, BN, BK, kThreads>;
  using E = typename T::elem;
  constexpr int kBuffer = registers_lds<T, BM, BN, BK, WM, WN, GROUPS>();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x & (kThreads - 1)) >> 6);
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  char* buf = lds + group * (kBuffer / GROUPS);
  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  const Work w = work_of<BM, BN>(g, id);
  const int m0 = w.tm * BM, n0 = w.tn * BN, steps = steps_of<BK, GROUPS>(w);
  int k0 = w.k0 + group * steps * BK;
  const int k1 = min(w.k1, k0 + steps * BK);
  const E *a = static_cast<const E*>(g.a), *b = static_cast<const E*>(g.b);

  f16v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  Raw8<T> ra[TA::kEach], rb[TB::kEach];
  auto fetch = [&](int k) {
    TA::load(ra, a, g.a_ld, m0, g.M, k, k1);
    TB::load(rb, b, g.b_ld, n0, g.N, k, k1);
  };
  auto put = [&](char* buf) {
    TA::store(ra, buf);
    TB::store(rb, buf + TA::kBytes);
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
  fetch(k0);
  for (int left = steps; left > 0; --left) {
    put(buf);
    __syncthreads();
    k0 += BK;
    if (left > 1) fetch(k0);  // past k1: zeros
    multiply(buf);
    __syncthreads();
  }
  if constexpr (GROUPS > 1) {
    char* const place[GROUPS] = {lds, lds + kBuffer / GROUPS, lds + kBuffer / GROUPS * 2, lds + kBuffer / GROUPS * 3};
    join_groups<IM, IN, GROUPS, kThreads>(acc, place, group);
    if (group != 0) return;
  }
  write_result<T, A_KS, B_KS, BN, IM, IN>(g, acc, lds + wave * kWayOut<IN>, m0 + wm, n0 + wn, w, wm, wn);
}

// Operands of 16-bit types whose rows are whole 16-byte pieces on 16-byte boundaries (with zeros in the last piece behind the
// last k, where k runs along the row): tiles of 32 k go straight from memory into a ring of four LDS buffers, with one
// barrier a step: it tells that a tile has landed for every wavefront (each waits for its own part) and that nobody reads
// the oldest one any more, whose buffer is then filled again.
// While step t is multiplied, tiles t+2 and t+3 are on their way and t+1 is there, so that its first fragments are read before
// the barrier that ends the step.
// 256 x 256 blocks, bfloat16 32768 x 4096 x 1024: 250 us = 1.10 PFLOP/s, matrix cores busy 63 % of the cycles at 1.73 GHz (the
// library's product: 248 us, 63 % at 1.82 GHz); 128 x 128 blocks 365 us, 128 x 256 in three buffers with two blocks a CU 294 us:
// both read the operands from L2 more often.
// GROUPS, 1 or 4: as above.
template <class T, bool A_KS, bool B_KS, int BM, int BN, int WM, int WN, int GROUPS>
__device__ __forceinline__ void gemm_ring(const GemmArgs& g, int id, char* lds0, char* lds1, char* lds2, char* lds3) {
  constexpr int kThreads = (BM / WM) * (BN / WN) * 64, IM = WM / 32, IN = WN / 32, BK = 32;
  using TA = Tile<T, A_KS, BM, BK, kThreads>;
  using TB = Tile<T, B_KS, BN, BK, kThreads>;
  using E = typename T::elem;
  constexpr int kStage = TA::kBytes + TB::kBytes, kLoads = TA::kEach + TB::kEach, kHalf = kThreads / 128;
  static_assert(kHalf * kWayOut<IN> <= kStage, "half of the wavefronts have their way out in the first buffer, half in the second");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x & (kThreads - 1)) >> 6);
  const int group = GROUPS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  char *buf0 = lds0 + group * kStage, *buf1 = lds1 + group * kStage, *buf2 = lds2 + group * kStage, *buf3 = lds3 + group * kStage;
  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  const Work w = work_of<BM, BN>(g, id);
  const int m0 = w.tm * BM, n0 = w.tn * BN, steps = steps_of<BK, GROUPS>(w), k0 = w.k0 + group * steps * BK, k1 = min(w.k1, k0 + steps * BK);
  typename TA::Source sa;
  typename TB::Source sb;
  sa.init(static_cast<const E*>(g.a), g.a_ld, m0, g.M, k0, k1);
  sb.init(static_cast<const E*>(g.b), g.b_ld, n0, g.N, k0, k1);

  f16v acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  auto fetch = [&](char* buf) {
    sa.next(buf);
    sb.next(buf + TA::kBytes);
  };
  u4 fa[2][IM], fb[2][IN];
  auto read = [&](int set, const char* buf, int s) {
#pragma unroll
    for (int j = 0; j < IN; ++j) fb[set][j] = TB::frag(buf + TA::kBytes, wn + 32 * j, s, lane);
#pragma unroll
    for (int i = 0; i < IM; ++i) fa[set][i] = TA::frag(buf, wm + 32 * i, s, lane);
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int j = 0; j < IN; ++j) acc[i][j] = mfma<T>(fb[set][j], fa[set][i], acc[i][j]);
  };
  auto step = [&](const char* now, const char* next, char* free) {
    fetch(free);
    read(1, now, 1);
    multiply(0);
    read(0, next, 0);
    multiply(1);
    landed<kLoads>();
  };
  fetch(buf0);
  fetch(buf1);
  fetch(buf2);
  landed<kLoads>();
  read(0, buf0, 0);
  for (int left = steps;;) {
    step(buf0, buf1, buf3);
    if (--left == 0) break;
    step(buf1, buf2, buf0);
    if (--left == 0) break;
    step(buf2, buf3, buf1);
    if (--left == 0) break;
    step(buf3, buf0, buf2);
    if (--left == 0) break;
  }
  landed<0>();  // also the tiles past the end, which were still on their way
  if constexpr (GROUPS > 1) {
    static_assert(kSums<IM, IN, kThreads> <= kStage * GROUPS && kThreads / 64 * kWayOut<IN> <= kStage * GROUPS, "");
    char* const place[GROUPS] = {lds0, lds1, lds2, lds3};
    join_groups<IM, IN, GROUPS, kThreads>(acc, place, group);
    if (group != 0) return;
    write_result<T, A_KS, B_KS, BN, IM, IN>(g, acc, lds0 + wave * kWayOut<IN>, m0 + wm, n0 + wn, w, wm, wn);
    return;
  }
  write_result<T, A_KS, B_KS, BN, IM, IN>(g, acc, (wave < kHalf ? buf0 : buf1) + (wave % kHalf) * kWayOut<IN>, m0 + wm, n0 + wn, w, wm, wn);
}

// One product.
template <class T, bool A_KS, bool B_KS, int BM, int BN, int BK, int WM, int WN, int GROUPS>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64 * GROUPS, BM == 128 ? 3 : 1) void k_layer_gemm(GemmArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[registers_lds<T, BM, BN, BK, WM, WN, GROUPS>()];
  gemm_registers<T, A_KS, B_KS, BM, BN, BK, WM, WN, GROUPS>(g, blockIdx.x, lds);
}
// LDS buffers are objects of their own, so that the compiler sees that a tile on its way does not touch the ones being read.
template <class T, bool A_KS, bool B_KS, int BM, int BN, int WM, int WN, int GROUPS>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64 * GROUPS) void k_layer_gemm_ring(GemmArgs g) {
  constexpr int kStage = (BM + BN) * 32 * 2 * GROUPS;
  __shared__ __attribute__((aligned(16))) char lds0[kStage], lds1[kStage], lds2[kStage], lds3[kStage];
  gemm_ring<T, A_KS, B_KS, BM, BN, WM, WN, GROUPS>(g, blockIdx.x, lds0, lds1, lds2, lds3);
}

// Both gradients of a layer in one launch, 128 x 128 blocks: they need nothing of one another, and the blocks of the second
// fill what the last round of the first leaves idle.  49200 x 250 x 250 in float32: 101 us, one after the other 109.
template <class T>
__global__ __launch_bounds__(256, 3) void k_layer_grads(GemmArgs dx, GemmArgs dk, unsigned dx_blocks) {
  __shared__ __attribute__((aligned(16))) char lds[registers_lds<T, 128, 128, 32 * (kPlanes<T> == 1 ? 2 : 1), 64, 64, 1>()];
  constexpr int BK = kPlanes<T> == 1 ? 64 : 32;
  if (blockIdx.x < dx_blocks) gemm_registers<T, false, false, 128, 128, BK, 64, 64, 1>(dx, blockIdx.x, lds);
  else gemm_registers<T, true, true, 128, 128, BK, 64, 64, 1>(dk, blockIdx.x - dx_blocks, lds);
}
template <class T>
__global__ __launch_bounds__(256) void k_layer_grads_ring(GemmArgs dx, GemmArgs dk, unsigned dx_blocks) {
  constexpr int kStage = (128 + 128) * 32 * 2;
  __shared__ __attribute__((aligned(16))) char lds0[kStage], lds1[kStage], lds2[kStage], lds3[kStage];
  if (blockIdx.x < dx_blocks) gemm_ring<T, false, false, 128, 128, 64, 64, 1>(dx, blockIdx.x, lds0, lds1, lds2, lds3);
  else gemm_ring<T, true, true, 128, 128, 64, 64, 1>(dk, blockIdx.x - dx_blocks, lds0, lds1, lds2, lds3);
}

}  // namespace
