// Shared by the Dense, dropout and beam operators: element types, loads of eight elements at any alignment, the
// counter-based generator.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/rnnt_mi355x.h"

namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// The same vectors at the alignment of their elements: rows of 250 floats or 515 halves start anywhere, and global
// memory takes wide accesses at any address.
typedef u4 u4_any __attribute__((aligned(1)));

struct Fp32 { using elem = float; static constexpr int code = RNNT_MI355X_FP32; };
struct Bf16 { using elem = uint16_t; static constexpr int code = RNNT_MI355X_BF16; };
struct Fp16 { using elem = uint16_t; static constexpr int code = RNNT_MI355X_FP16; };

__device__ __forceinline__ float half_bits_to_float(uint32_t h) {
  const uint16_t b = (uint16_t)h;
  _Float16 f;
  __builtin_memcpy(&f, &b, 2);
  return (float)f;
}
__device__ __forceinline__ uint32_t float_to_half_bits(float v) {
  const _Float16 f = (_Float16)v;
  uint16_t b;
  __builtin_memcpy(&b, &f, 2);
  return b;
}
// round to nearest even, NaN stays NaN
__device__ __forceinline__ uint32_t float_to_bf16_bits(float v) {
  const __bf16 f = (__bf16)v;
  uint16_t b;
  __builtin_memcpy(&b, &f, 2);
  return b;
}

// two at a time: one instruction
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), bf2));
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), hf2));
}

template <class T>
__device__ __forceinline__ float to_float(typename T::elem v) {
  if constexpr (T::code == RNNT_MI355X_FP32) return v;
  else if constexpr (T::code == RNNT_MI355X_BF16) return __uint_as_float((uint32_t)v << 16);
  else return half_bits_to_float(v);
}
template <class T>
__device__ __forceinline__ typename T::elem from_float(float v) {
  if constexpr (T::code == RNNT_MI355X_FP32) return v;
  else if constexpr (T::code == RNNT_MI355X_BF16) return (uint16_t)float_to_bf16_bits(v);
  else return (uint16_t)float_to_half_bits(v);
}

// Eight consecutive elements as they lie in memory: 32 or 16 bytes.
template <class T>
struct Raw8 {
  u4 q[T::code == RNNT_MI355X_FP32 ? 2 : 1];
};
template <class T>
__device__ __forceinline__ Raw8<T> load8_raw(const typename T::elem* p) {
  Raw8<T> r;
  const u4_any* v = reinterpret_cast<const u4_any*>(p);
  r.q[0] = v[0];
  if constexpr (T::code == RNNT_MI355X_FP32) r.q[1] = v[1];
  return r;
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (T::code == RNNT_MI355X_FP32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.q[i >> 2][i & 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r.q[0][i];
      if constexpr (T::code == RNNT_MI355X_BF16) {
        v[2 * i] = __uint_as_float(w << 16);
        v[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
      } else {
        v[2 * i] = half_bits_to_float(w & 0xffffu);
        v[2 * i + 1] = half_bits_to_float(w >> 16);
      }
    }
  }
}
template <class T>
__device__ __forceinline__ void store8(typename T::elem* p, const float (&v)[8]) {
  u4_any* d = reinterpret_cast<u4_any*>(p);
  if constexpr (T::code == RNNT_MI355X_FP32) {
    d[0] = u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    d[1] = u4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
  } else {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T::code == RNNT_MI355X_BF16) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      else w[i] = pack_half(v[2 * i], v[2 * i + 1]);
    }
    d[0] = w;
  }
}
// The first n < 8 elements of a group (the end of a row whose length is no multiple of eight).
template <class T>
__device__ __forceinline__ void load_some(const typename T::elem* p, int n, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.f;
}
template <class T>
__device__ __forceinline__ void store_some(typename T::elem* p, int n, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_float<T>(v[i]);
}

// What a dropout mask is made from.  The offset may live in device memory, so that a captured graph draws another mask
// on every replay.
struct DropArgs {
  uint32_t drop;  // an element is dropped with probability drop / 65536; 0: no dropout
  uint32_t key0, key1, off0, off1;
  const uint64_t* offset;  // nullable: replaces off0, off1
  float scale;             // 65536 / (65536 - drop)
};

__host__ inline DropArgs drop_args(int drop16, uint64_t seed, uint64_t offset, const uint64_t* offset_dev) {
  DropArgs a;
  a.drop = (uint32_t)drop16;
  a.key0 = (uint32_t)seed;
  a.key1 = (uint32_t)(seed >> 32);
  a.off0 = (uint32_t)offset;
  a.off1 = (uint32_t)(offset >> 32);
  a.offset = offset_dev;
  a.scale = (float)(65536.0 / (65536.0 - drop16));
  return a;
}

__device__ __forceinline__ void load_offset(DropArgs& a) {
  if (a.offset) {
    const uint64_t o = *a.offset;
    a.off0 = (uint32_t)o;
    a.off1 = (uint32_t)(o >> 32);
  }
}

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);  // one instruction for the truth table of a ^ b ^ c
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds of two
// 32x32-bit products over a counter of four words, of which every value gives 128 independent bits.  Eight columns of a
// row share a counter and take 16 bits each: with 32 bits the generator (20 wide products, ~60 cycles an element-quad on
// a wavefront) would bound 16-bit tensors instead of memory.  The price is a drop probability in steps of 2^-16.
__device__ __forceinline__ u4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((uint32_t)(q >> 32), c1, k0);
    c1 = (uint32_t)q;
    c2 = xor3((uint32_t)(p >> 32), c3, k1);
    c3 = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u4{c0, c1, c2, c3};
}

// v[i] *= 1/keep or 0 for columns 8*group + i of a row.  A dropped infinity or NaN becomes 0, as a dropped value is not
// there.
__device__ __forceinline__ void drop8(const DropArgs& a, uint32_t row, uint32_t group, float (&v)[8]) {
  const u4 w = philox(group, row, a.off0, a.off1, a.key0, a.key1);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = (w[i] & 0xffffu) >= a.drop ? v[2 * i] * a.scale : 0.f;
    v[2 * i + 1] = (w[i] >> 16) >= a.drop ? v[2 * i + 1] * a.scale : 0.f;
  }
}

}  // namespace
