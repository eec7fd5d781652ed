// One step of a beam search for MI355X (gfx950): selection over beams x vocabulary, and the hypotheses' states in their
// new order.  Where the reference's decoder scores one hypothesis at a time in numpy (reference
// rnnt/rnnt_decoder.py:156-158, 200-202) and sorts them on the host, here
//     x[b,k,v]     = logits[b,k,v] (+ enc[b,v], rounded to float32)
//     total[b,k,v] = scores[b,k] + x[b,k,v] - log sum_v' exp x[b,k,v'],      v' over the allowed symbols
// and the `width` largest totals of an utterance, ties to the lowest k * V + v.
//
// A wavefront takes a piece of a row into registers, at most 32 values a lane.  Inside a row the order of the totals is
// the order of x, so a piece needs only its own `width` largest x (exact float32 comparisons) and its share of the
// softmax sum; the totals themselves are formed in float64, because candidates of different beams lie arbitrarily close
// and a float32 sum would order them by its rounding.
//   - the lanes' maxima are sorted across the wavefront; the width-th of them is a lower bound T of the width-th largest
//     value, and the few values >= T are compacted and sorted (a bitonic network over the lanes);
//   - sorted lists are joined by the first step of a bitonic merge: of two sorted lists a, b the values
//     max(a[i], b[P-1-i]) are the P largest, and log2 P exchanges sort them.
// Rows of up to 2048 symbols take one launch, a block per utterance; longer ones a launch over pieces of 2048 and one that
// joins the pieces' lists.  Measured, 32 utterances x 16 beams x 32003 symbols in bfloat16 with a mask: pieces 19.6 us (34 MB;
// more than half of it are the 30 instructions a symbol, four of them in float64), join 7.8 us; 4 x 32 x 65536 in float16 without one: 12.1 and
// 11 us; 64 x 8 x 1024 in float32: 7.9 us.  The joins, and the short rows, are chains of latencies: sorting networks over a wavefront, LDS, memory.
#include "op_util.h"

namespace {

constexpr double kLog2e64 = 1.4426950408889634;
constexpr float kScoreLimit = 1073741824.f;  // 2^30: a score beyond it marks an empty beam (or is no score at all)
constexpr int kMaxBeams = 64, kMaxWidth = 64;
constexpr int kPiece = 2048;  // symbols of a row that one wavefront takes

// ---- exchanges between lanes --------------------------------------------------------------------------------------------
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);        // quad_perm 1,0,3,2
  else if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);   // quad_perm 2,3,0,1
  else if constexpr (M == 3) return __builtin_amdgcn_update_dpp(0, v, 0x1B, 0xf, 0xf, true);   // quad_perm 3,2,1,0
  else if constexpr (M == 7) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);  // row_half_mirror
  else if constexpr (M == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);  // row_ror:8
  else if constexpr (M == 15) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true); // row_mirror
  else if constexpr (M == 4) return lane_xor<7>(lane_xor<3>(v));
  else if constexpr (M == 16) {  // the first result has rows 0, 0, 2, 2 of 16 lanes, the second 1, 1, 3, 3
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  } else if constexpr (M == 31) return lane_xor<16>(lane_xor<15>(v));
  else {
    static_assert(M == 63, "");
    return lane_xor<32>(lane_xor<16>(lane_xor<15>(v)));
  }
}

// Candidates: larger is better, all of them different; zero stands for none.
struct RowKey {  // value of a row, then the lower symbol
  uint32_t hi, lo;
  __device__ __forceinline__ bool operator>(const RowKey& o) const {
    return (((uint64_t)hi << 32) | lo) > (((uint64_t)o.hi << 32) | o.lo);
  }
};
struct TotalKey {  // total in float64, then the lower place in beams x vocabulary
  uint64_t hi;
  uint32_t lo;
  __device__ __forceinline__ bool operator>(const TotalKey& o) const { return (hi > o.hi) | ((hi == o.hi) & (lo > o.lo)); }  // no branch
};
template <int M>
__device__ __forceinline__ RowKey lane_xor(const RowKey& k) {
  return {lane_xor<M>(k.hi), lane_xor<M>(k.lo)};
}
template <int M>
__device__ __forceinline__ TotalKey lane_xor(const TotalKey& k) {
  return {((uint64_t)lane_xor<M>((uint32_t)(k.hi >> 32)) << 32) | lane_xor<M>((uint32_t)k.hi), lane_xor<M>(k.lo)};
}
// order-preserving integers of floating values (no NaN comes here; every finite or infinite value gives more than zero)
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((int32_t)b >> 31 | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered(uint64_t k) {
  return __builtin_bit_cast(double, k >> 63 ? k ^ 0x8000000000000000ull : ~k);
}

// The lane whose index has bit log2(D) clear keeps the larger key.
template <int M, int D, class K>
__device__ __forceinline__ void exchange(K& k, int lane) {
  const K o = lane_xor<M>(k);
  if ((o > k) == !(lane & D)) k = o;
}
// In each list of P lanes a bitonic sequence becomes a descending one.
template <int P, class K>
__device__ __forceinline__ void clean(K& k, int lane) {
  if constexpr (P >= 64) exchange<32, 32>(k, lane);
  if constexpr (P >= 32) exchange<16, 16>(k, lane);
  if constexpr (P >= 16) exchange<8, 8>(k, lane);
  if constexpr (P >= 8) exchange<4, 4>(k, lane);
  if constexpr (P >= 4) exchange<2, 2>(k, lane);
  if constexpr (P >= 2) exchange<1, 1>(k, lane);
}
// 64 keys in descending order over the lanes: at every stage two sorted runs are joined by their mirrored exchange.
template <class K>
__device__ __forceinline__ void sort64(K& k, int lane) {
  exchange<1, 1>(k, lane);
  exchange<3, 2>(k, lane);  clean<2>(k, lane);
  exchange<7, 4>(k, lane);  clean<4>(k, lane);
  exchange<15, 8>(k, lane); clean<8>(k, lane);
  exchange<31, 16>(k, lane); clean<16>(k, lane);
  exchange<63, 32>(k, lane); clean<32>(k, lane);
}
// acc and a list that comes in reverse order, P lanes a list: acc becomes the P largest of both.
template <int P, class K>
__device__ __forceinline__ void join(K& acc, const K& reversed, int lane) {
  if (reversed > acc) acc = reversed;
  clean<P>(acc, lane);
}

template <int M>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<M>(__float_as_uint(v)));
}
template <int M>
__device__ __forceinline__ double lane_xor(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, ((uint64_t)lane_xor<M>((uint32_t)(b >> 32)) << 32) | lane_xor<M>((uint32_t)b));
}
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // NaN stays
__device__ __forceinline__ float wave_max(float v) {
  v = largest(v, lane_xor<1>(v));
  v = largest(v, lane_xor<2>(v));
  v = largest(v, lane_xor<7>(v));
  v = largest(v, lane_xor<15>(v));
  v = largest(v, lane_xor<16>(v));
  return largest(v, lane_xor<32>(v));
}
// the same order of additions in every wavefront: equal rows get equal sums
__device__ __forceinline__ double wave_sum(double v) {
  v += lane_xor<1>(v);
  v += lane_xor<2>(v);
  v += lane_xor<7>(v);
  v += lane_xor<15>(v);
  v += lane_xor<16>(v);
  return v + lane_xor<32>(v);
}

// What a wavefront's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct BeamArgs {
  const void* logits;
  const void* enc;         // nullable
  const float* scores;     // [B, K]
  const uint8_t* allowed;  // nullable
  const uint8_t* finished; // nullable, [B, K]
  long long logits_b, logits_k, enc_b, allowed_b;  // strides in elements
  int B, K, V, width, end, pieces;
  float* out_scores;
  int32_t *out_parent, *out_token;
};

// The piece [v0, v0 + 64 * E) of a row in registers: element j*64*W + lane*W + i of it, W = 4 or 8 consecutive ones.
// Symbols past V and forbidden ones are -inf whatever the memory holds.
template <class T, int E>
__device__ __forceinline__ void load_piece(const BeamArgs& a, int b, int k, int v0, int lane, float (&x)[E]) {
  const typename T::elem* row = static_cast<const typename T::elem*>(a.logits) + b * a.logits_b + k * a.logits_k;
  const typename T::elem* enc = a.enc ? static_cast<const typename T::elem*>(a.enc) + b * a.enc_b : nullptr;
  const uint8_t* allowed = a.allowed ? a.allowed + b * a.allowed_b : nullptr;
  constexpr int G = E / 8;
  Raw8<T> r[G], e[G];
  u2 m[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int v = v0 + j * 512 + lane * 8;
    if (v + 8 <= a.V) {
      r[j] = load8_raw<T>(row + v);
      if (enc) e[j] = load8_raw<T>(enc + v);
      if (allowed) __builtin_memcpy(&m[j], allowed + v, 8);
    }
  }
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const int v = v0 + j * 512 + lane * 8;
    float y[8];
    if (v + 8 <= a.V) {
      unpack8<T>(r[j], y);
      if (enc) {
        float z[8];
        unpack8<T>(e[j], z);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += z[i];
      }
      if (allowed) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (m[j][i >> 2] >> (8 * (i & 3))) & 0xffu ? y[i] : -INFINITY;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = -INFINITY;
        if (v + i < a.V) {
          const float t = to_float<T>(row[v + i]) + (enc ? to_float<T>(enc[v + i]) : 0.f);
          if (!allowed || allowed[v + i]) y[i] = t;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[8 * j + i] = y[i];
  }
}

// 64 values in descending order over the lanes, without what they belong to.
template <int M, int D>
__device__ __forceinline__ void exchange_value(uint32_t& v, int lane) {
  const uint32_t o = lane_xor<M>(v);
  v = lane & D ? min(v, o) : max(v, o);
}
__device__ __forceinline__ void sort64_values(uint32_t& v, int lane) {
  exchange_value<1, 1>(v, lane);
  exchange_value<3, 2>(v, lane);
  exchange_value<1, 1>(v, lane);
  exchange_value<7, 4>(v, lane);
  exchange_value<2, 2>(v, lane);
  exchange_value<1, 1>(v, lane);
  exchange_value<15, 8>(v, lane);
  exchange_value<4, 4>(v, lane);
  exchange_value<2, 2>(v, lane);
  exchange_value<1, 1>(v, lane);
  exchange_value<31, 16>(v, lane);
  exchange_value<8, 8>(v, lane);
  exchange_value<4, 4>(v, lane);
  exchange_value<2, 2>(v, lane);
  exchange_value<1, 1>(v, lane);
  exchange_value<63, 32>(v, lane);
  exchange_value<16, 16>(v, lane);
  exchange_value<8, 8>(v, lane);
  exchange_value<4, 4>(v, lane);
  exchange_value<2, 2>(v, lane);
  exchange_value<1, 1>(v, lane);
}

// The larger of a lane's key and its partner's.
template <int M>
__device__ __forceinline__ RowKey larger(const RowKey& k) {
  const RowKey o = lane_xor<M>(k);
  return o > k ? o : k;
}

// Softmax share and the 64 best candidates of a piece: *m the largest value, *s = sum exp(x - m) (NaN when a value is NaN
// or +inf), and in lane i the i-th candidate, of which the first `width` are right.  buf: 64 keys of LDS of this wavefront.
template <int E>
__device__ __forceinline__ RowKey best_of_piece(const float (&x)[E], int v0, int width, int lane, RowKey* buf, float* m, double* s) {
  float top = x[0];
#pragma unroll
  for (int e = 1; e < E; ++e) top = largest(top, x[e]);
  const float mx = wave_max(top);
  const bool number = mx < INFINITY;
  // exp(x - mx) = 2^(n + f): the argument in float64 (in float32 its rounding alone would cost 2^-21 of a term ten below the
  // largest, the same way for all symbols of equal value), as a fixed-point number with 32 bits of fraction by adding 1.5 x 2^20, f
  // rounded to 23 bits as the significand of 1 + f, and n added to the result's exponent.  A term is off by 2^-24 (1.43 for exp2,
  // measured over all its arguments, and ln 2 for f); at x = mx it is exact, so that a row of one symbol sums to 1.  Terms
  // below 2^-120 become that.  Eight terms are added pairwise in float32, another 3 x 2^-24 where their bits differ, then in
  // float64: the sum decides between candidates of different beams.  The same with the argument in float32 and a first-order
  // correction for what it leaves out: 32 x 16 x 32003 in bfloat16 31.0 us a step (29.7 this way, 27.6 without any).
  const double base = mx == -INFINITY || !number ? 0.0 : (double)mx;
  constexpr double kFixed = 1572864.0 + 0x1p-24, kLeast = kFixed - 120.0;
  double sum = 0.0;
#pragma unroll
  for (int e = 0; e < E; e += 8) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t h = __builtin_bit_cast(uint64_t, fmax(fma((double)x[e + i] - base, kLog2e64, kFixed), kLeast));
      const float f = __uint_as_float(__builtin_amdgcn_alignbit(0x7fu, (uint32_t)h, 9));  // 1 <= f < 2: terms are doubled
      uint32_t n = (uint32_t)(h >> 32);
      asm("" : "+v"(n));  // else three instructions take the place of the shift and add that the next line is
      t[i] = __uint_as_float(__float_as_uint(__builtin_amdgcn_exp2f(f)) + (n << 23));
    }
    sum += (double)(((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7])));
  }
  sum = wave_sum(sum);
  *m = number ? mx : 0.f;
  *s = !number ? NAN : mx == -INFINITY ? 0.0 : 0.5 * sum;

  // `width` lanes have a value of floor_x or more
  uint32_t tops = top > -INFINITY ? ordered(top + 0.f) : 0u;
  sort64_values(tops, lane);
  const uint32_t floor_key = (uint32_t)__shfl((int)tops, width - 1, 64);
  const float floor_x = floor_key ? unordered(floor_key) : -__FLT_MAX__;  // -inf is never a candidate
  auto place = [&](int e) { return (uint32_t)(v0 + (e >> 3) * 512 + lane * 8 + (e & 7)); };
  int fill = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = x[e] >= floor_x;
    const uint64_t who = __ballot(in);
    if (who) {  // uniform
      const int at = fill + __popcll(who & ((1ull << lane) - 1));
      if (in && at < 64) buf[at] = RowKey{__float_as_uint(x[e]), place(e)};
      fill += __popcll(who);
    }
  }
  RowKey acc = {0u, 0u};
  if (fill <= 64) {  // uniform, and nearly always so
    wave_sync();
    if (lane < fill) acc = RowKey{ordered(__uint_as_float(buf[lane].hi) + 0.f), ~buf[lane].lo};  // -0 and +0 tie
    sort64(acc, lane);
    return acc;
  }
  // Many values of one size, or many of the best in one lane: the next best key of all, `width` times over.
  RowKey last = {~0u, ~0u};
#pragma unroll 1
  for (int i = 0; i < width; ++i) {
    RowKey best = {0u, 0u};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const RowKey k = {x[e] >= floor_x ? ordered(x[e] + 0.f) : 0u, ~place(e)};
      if (last > k && k > best) best = k;
    }
    if (best.hi == 0u) best.lo = 0u;
    best = larger<1>(best);
    best = larger<2>(best);
    best = larger<7>(best);
    best = larger<15>(best);
    best = larger<16>(best);
    best = larger<32>(best);
    if (lane == i) acc = best;
    last = best;
  }
  return acc;
}

__device__ __forceinline__ bool live_score(float s) { return fabsf(s) <= kScoreLimit; }

// A row's softmax: the largest value and log sum exp(x - m).
struct RowSum {
  double m, log_s;
};

// The candidate c of beam k, or the one of a finished beam, in the order of the utterance.
__device__ __forceinline__ TotalKey total_key(const BeamArgs& a, int k, bool done, float score, const RowSum& row, const RowKey& c) {
  TotalKey t = {0ull, 0u};
  if (done) {
    t.hi = ordered((double)score + 0.0);
    t.lo = ~(uint32_t)(k * a.V + a.end);
  } else if (c.hi) {
    t.hi = ordered((double)score + (((double)unordered(c.hi) - row.m) - row.log_s) + 0.0);
    t.lo = ~(uint32_t)(k * a.V + (int)~c.lo);
  }
  return t;
}

__device__ __forceinline__ void write_out(const BeamArgs& a, int b, int lane, const TotalKey& k) {
  if (lane < a.width) {
    const long long o = (long long)b * a.width + lane;
    const uint32_t flat = ~k.lo;
    a.out_scores[o] = k.hi ? (float)unordered(k.hi) : -INFINITY;
    a.out_parent[o] = k.hi ? (int32_t)(flat / (uint32_t)a.V) : -1;
    a.out_token[o] = k.hi ? (int32_t)(flat % (uint32_t)a.V) : -1;
  }
}

// The wavefronts' lists, P lanes each and 64 / P to a wavefront: all joined in wavefront 0.
template <int P>
__device__ __forceinline__ void join_block(TotalKey& acc, TotalKey (*lds)[64], int wave, int waves, int lane) {
  if constexpr (P <= 8) join<P>(acc, lane_xor<15>(acc), lane);
  if constexpr (P <= 16) join<P>(acc, lane_xor<31>(acc), lane);
  if constexpr (P <= 32) join<P>(acc, lane_xor<63>(acc), lane);
  for (int half = waves >> 1; half >= 1; half >>= 1) {  // waves: a power of two
    if (wave >= half && wave < 2 * half) lds[wave][lane] = acc;
    __syncthreads();
    if (wave < half) join<P>(acc, lds[wave + half][(lane & ~(P - 1)) | (P - 1 - (lane & (P - 1)))], lane);
    __syncthreads();
  }
}

// One launch for short rows: a block per utterance, its wavefronts share the beams.
// More than 8 values a lane, with what they are loaded into, do not fit the 128 registers of 16 wavefronts: such blocks have 8.
template <class T, int E, int P>
__global__ __launch_bounds__(E > 8 ? 512 : 1024) void k_beam_rows(BeamArgs a) {
  __shared__ RowKey lists[kMaxBeams][P];
  __shared__ RowSum rows[kMaxBeams];
  __shared__ TotalKey tree[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, b = blockIdx.x;
  RowKey* buf = reinterpret_cast<RowKey*>(tree[wave]);  // 64 keys; the lists are joined there after the barrier
  for (int k = wave; k < a.K; k += waves) {
    const float score = a.scores[(long long)b * a.K + k];
    const bool done = a.finished && a.finished[(long long)b * a.K + k];
    RowKey best = {0u, 0u};
    RowSum row = {0.0, 0.0};
    if (live_score(score) && !done) {  // uniform
      float x[E], m;
      double s;
      load_piece<T, E>(a, b, k, 0, lane, x);
      best = best_of_piece<E>(x, 0, a.width, lane, buf, &m, &s);
      row = RowSum{(double)m, log(s)};
      if (!(s > 0.0)) best = RowKey{0u, 0u};  // nothing allowed, or a NaN or +inf among the values
    }
    if (lane < P) lists[k][lane] = lane < a.width ? best : RowKey{0u, 0u};
    if (lane == 0) rows[k] = row;
  }
  __syncthreads();
  TotalKey acc = {0ull, 0u};
  constexpr int G = 64 / P;
  const int i = lane & (P - 1);
  for (int k0 = wave * G; k0 < a.K; k0 += waves * G) {
    const int k = k0 + lane / P;
    TotalKey t = {0ull, 0u};
    if (k < a.K) {
      const float score = a.scores[(long long)b * a.K + k];
      const bool done = a.finished && a.finished[(long long)b * a.K + k];
      const int r = P - 1 - i;
      if (live_score(score) && (!done || r == 0)) t = total_key(a, k, done, score, rows[k], lists[k][r]);
    }
    join<P>(acc, t, lane);
  }
  int active = 1;  // wavefronts that took beams, up to a power of two
  while (active * G < a.K && active < waves) active <<= 1;
  join_block<P>(acc, tree, wave, active, lane);
  if (wave == 0) write_out(a, b, lane, acc);
}

// The block's keys whose lanes say `in`, into LDS in any order; *n counts them, and past 64 they are not kept.
__device__ __forceinline__ void gather(const TotalKey& k, bool in, int lane, TotalKey* buf, int* n) {
  const uint64_t who = __ballot(in);
  if (!who) return;  // uniform
  int at = 0;
  if (lane == 0) at = atomicAdd(n, __popcll(who));
  at = __builtin_amdgcn_readfirstlane(at) + __popcll(who & ((1ull << lane) - 1));
  if (in && at < 64) buf[at] = k;
}

// Long rows, first launch: a wavefront per piece.  Workspace: the pieces' sums, then their lists of P keys.
struct PieceSum {
  double s;
  float m;        // the value of the list's first entry, -inf where there is none
  uint32_t best;  // its `lo`
};
__device__ __forceinline__ RowKey head_of(const PieceSum& q) { return q.m > -INFINITY ? RowKey{ordered(q.m + 0.f), q.best} : RowKey{0u, 0u}; }
template <class T, int P>
__global__ __launch_bounds__(256) void k_beam_pieces(BeamArgs a, PieceSum* sums, RowKey* lists) {
  __shared__ RowKey buf[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned id = blockIdx.x * 4u + (unsigned)__builtin_amdgcn_readfirstlane(wave);  // B * K * pieces < 2^31
  if (id >= (unsigned)a.B * (unsigned)a.K * (unsigned)a.pieces) return;
  const unsigned row = id / (unsigned)a.pieces;
  const int piece = (int)(id - row * (unsigned)a.pieces);
  if (!live_score(a.scores[row]) || (a.finished && a.finished[row])) return;  // nothing of it is read
  float x[kPiece / 64], m;
  double s;
  load_piece<T, kPiece / 64>(a, (int)(row / (unsigned)a.K), (int)(row % (unsigned)a.K), piece * kPiece, lane, x);
  const RowKey best = best_of_piece<kPiece / 64>(x, piece * kPiece, a.width, lane, buf[wave], &m, &s);
  if (lane < P) lists[(long long)id * P + lane] = lane < a.width ? best : RowKey{0u, 0u};
  if (lane == 0) sums[id] = PieceSum{s, m, best.lo};
}

// Second launch: a block per utterance joins the pieces.  Only the `width` lists with the best first entries can hold
// anything that is kept: the first entries alone choose them, and only those lists are read on.
template <int P>
__global__ __launch_bounds__(1024) void k_beam_join(BeamArgs a, const PieceSum* sums, const RowKey* lists) {
  __shared__ RowSum rows[kMaxBeams];
  __shared__ float live[kMaxBeams];  // the score of a beam that has candidates, else NaN
  __shared__ bool over[kMaxBeams];   // finished: its score is its one candidate
  __shared__ TotalKey tree[16][64];
  __shared__ TotalKey best[kMaxWidth];
  __shared__ uint32_t most[kMaxBeams];  // the largest value of a beam's row
  __shared__ double terms[64][kMaxBeams];
  __shared__ uint32_t tops[64];
  __shared__ TotalKey few[64];
  __shared__ int found[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, b = blockIdx.x;
  const int lists_here = a.K * a.pieces;
  lists += (long long)b * lists_here * P;
  if (threadIdx.x < 2) found[threadIdx.x] = 0;
  if (threadIdx.x < 64) tops[threadIdx.x] = 0u;
  const int first = wave * 64 + lane;
  sums += (long long)b * lists_here;
  PieceSum q = {0.0, -INFINITY, 0u};
  if (first < lists_here) q = sums[first];
  auto piece = [&](int l) { return l == first ? q : sums[l]; };
  // a piece without an allowed symbol has m = -inf and s = 0; a NaN sum stays one
  auto term = [](const PieceSum& q, float m) { return q.m == -INFINITY ? q.s : q.s * exp((double)q.m - (double)m); };
  auto note = [&](int k, float score, bool done, float m, double s) {
    if (!live_score(score) || (!done && !(s > 0.0))) score = NAN;
    rows[k] = RowSum{(double)m, log(s)};
    live[k] = score;
    over[k] = done;
  };
  if (a.pieces <= 64) {
    // A thread per piece, then one per beam: a double's exp and log are some hundred instructions, which a wavefront per beam
    // goes through beam after beam (the join of 32 x 16 x 32003: 10.0 us that way, 8.0 this way).  Longer rows fill wavefronts.
    auto read = [&](int k) {  // a beam whose pieces were made
      const long long row = (long long)b * a.K + k;
      return live_score(a.scores[row]) && !(a.finished && a.finished[row]);
    };
    const bool mine = first < lists_here && read(first / a.pieces);
    float score = NAN;
    bool done = false;
    if ((int)threadIdx.x < a.K) {
      const long long row = (long long)b * a.K + threadIdx.x;
      score = a.scores[row];
      done = a.finished && a.finished[row];
    }
    if ((int)threadIdx.x < kMaxBeams) most[threadIdx.x] = 0u;
    __syncthreads();
    for (int l = first; l < lists_here; l += waves * 64) {
      const int k = l / a.pieces;
      if (l == first ? mine : read(k)) atomicMax(&most[k], ordered(piece(l).m));
    }
    __syncthreads();
    for (int l = first; l < lists_here; l += waves * 64) {
      const int k = l / a.pieces;
      if (l == first ? mine : read(k)) terms[l - k * a.pieces][k] = term(piece(l), unordered(most[k]));
    }
    __syncthreads();
    if ((int)threadIdx.x < a.K) {
      const int k = threadIdx.x;
      double s = 0.0;
      if (most[k]) {
#pragma unroll 8
        for (int p = 0; p < a.pieces; ++p) s += terms[p][k];
      }
      note(k, score, done, unordered(most[k]), s);
    }
  } else {
    for (int k = wave; k < a.K; k += waves) {
      const long long row = (long long)b * a.K + k;
      const PieceSum* mine = sums + k * a.pieces;
      const float score = a.scores[row];
      const bool done = a.finished && a.finished[row];
      float m = -INFINITY;
      double s = 0.0;
      if (live_score(score) && !done) {  // uniform
        for (int p = lane; p < a.pieces; p += 64) m = fmaxf(m, mine[p].m);
        m = wave_max(m);
        for (int p = lane; p < a.pieces; p += 64) s += term(mine[p], m);
        s = wave_sum(s);
      }
      if (lane == 0) note(k, score, done, m, s);
    }
  }
  __syncthreads();
  auto entry = [&](int l, int r, const RowKey& c) {  // the r-th candidate of list l, which is c
    const int k = l / a.pieces;
    const float score = live[k];
    if (score != score) return TotalKey{0ull, 0u};
    if (!over[k]) return total_key(a, k, false, score, rows[k], c);
    return r == 0 && l == k * a.pieces ? total_key(a, k, true, score, rows[k], RowKey{0u, 0u}) : TotalKey{0ull, 0u};
  };
  // As in a piece: of 64 maxima (lists 64 apart, so that every beam has a part in many) the width-th bounds the width-th head
  // from below, and the few heads that reach it are sorted by one wavefront (the join of 4 x 32 x 65536: 11.0 us, with lists of
  // 64 sorted and joined across the block 14.7).  Where they are more than 64, that is done still.
  TotalKey heads = {0ull, 0u};
  if (first < lists_here) heads = entry(first, 0, head_of(q));
  const TotalKey mine = heads;
  auto head = [&](int l) { return l >= lists_here ? TotalKey{0ull, 0u} : l == first ? mine : entry(l, 0, head_of(sums[l])); };
  for (int l = first; l < lists_here; l += waves * 64) atomicMax(&tops[lane], (uint32_t)(head(l).hi >> 32));
  __syncthreads();
  uint32_t least = tops[lane];
  sort64_values(least, lane);
  least = max(1u, (uint32_t)__shfl((int)least, a.width - 1, 64));
  for (int l = first; l - lane < lists_here; l += waves * 64) {
    const TotalKey t = head(l);
    gather(t, (uint32_t)(t.hi >> 32) >= least, lane, few, &found[0]);
  }
  __syncthreads();
  if (found[0] <= 64) {
    if (wave == 0) {
      heads = lane < found[0] ? few[lane] : TotalKey{0ull, 0u};
      sort64(heads, lane);
    }
  } else {
    sort64(heads, lane);
    for (int l = first + waves * 64; l - lane < lists_here; l += waves * 64) {
      TotalKey t = head(l);
      if (__any(t.hi != 0)) {
        sort64(t, lane);
        join<64>(heads, lane_xor<63>(t), lane);
      }
    }
    join_block<64>(heads, tree, wave, waves, lane);
  }
  if (wave == 0 && lane < a.width) best[lane] = heads;
  __syncthreads();

  TotalKey acc = {0ull, 0u};
  constexpr int G = 64 / P;
  const int i = lane & (P - 1), r = P - 1 - i;
  auto kept = [&](int l0) {  // of the lists with the best heads, the l0-th and on, P entries each and the last first
    const int w = l0 + lane / P;
    if (w >= a.width || !best[w].hi) return TotalKey{0ull, 0u};
    const uint32_t flat = ~best[w].lo, k = flat / (uint32_t)a.V;
    const int l = (int)k * a.pieces + (over[k] ? 0 : (int)(flat - k * (uint32_t)a.V) / kPiece);
    return entry(l, r, over[k] ? RowKey{0u, 0u} : lists[(long long)l * P + r]);
  };
  // the last of these heads bounds the result, too
  least = max(1u, (uint32_t)(best[a.width - 1].hi >> 32));
  for (int l0 = wave * G; l0 < a.width; l0 += waves * G) {
    const TotalKey t = kept(l0);
    gather(t, (uint32_t)(t.hi >> 32) >= least, lane, few, &found[1]);
  }
  __syncthreads();
  if (found[1] <= 64) {
    if (wave > 0) return;
    if (lane < found[1]) acc = few[lane];
    sort64(acc, lane);
    write_out(a, b, lane, acc);
    return;
  }
  for (int l0 = wave * G; l0 < a.width; l0 += waves * G) join<P>(acc, kept(l0), lane);
  join_block<P>(acc, tree, wave, waves, lane);
  if (wave == 0) write_out(a, b, lane, acc);
}

int list_lanes(int width) { return width <= 8 ? 8 : width <= 16 ? 16 : width <= 32 ? 32 : 64; }
int pieces_of(int V) { return V <= kPiece ? 0 : (V + kPiece - 1) / kPiece; }
int pow2_up(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

template <class T, int P>
int launch_select(const BeamArgs& a, void* workspace, hipStream_t st) {
  if (a.pieces == 0) {
    const int most = a.V <= 512 ? 16 : 8, waves = a.K >= most ? most : pow2_up(a.K);
    if (a.V <= 512) k_beam_rows<T, 8, P><<<a.B, waves * 64, 0, st>>>(a);
    else if (a.V <= 1024) k_beam_rows<T, 16, P><<<a.B, waves * 64, 0, st>>>(a);
    else k_beam_rows<T, 32, P><<<a.B, waves * 64, 0, st>>>(a);
  } else {
    const long long n = (long long)a.B * a.K * a.pieces;
    PieceSum* sums = static_cast<PieceSum*>(workspace);
    RowKey* lists = reinterpret_cast<RowKey*>(sums + n);
    k_beam_pieces<T, P><<<(unsigned)((n + 3) / 4), 256, 0, st>>>(a, sums, lists);
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
    const int waves = min(16, max(pow2_up((a.K * a.pieces + 63) / 64), pow2_up((a.width * P + 63) / 64)));
    k_beam_join<P><<<a.B, waves * 64, 0, st>>>(a, sums, lists);
  }
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
}
template <class T>
int launch_select_width(const BeamArgs& a, void* workspace, hipStream_t st) {
  switch (list_lanes(a.width)) {
    case 8: return launch_select<T, 8>(a, workspace, st);
    case 16: return launch_select<T, 16>(a, workspace, st);
    case 32: return launch_select<T, 32>(a, workspace, st);
  }
  return launch_select<T, 64>(a, workspace, st);
}

int check_select(int B, int K, int V, int width) {
  if (B < 1 || K < 1 || V < 1 || width < 1) return RNNT_MI355X_INVALID_VALUE;
  // a piece's last symbols are counted past V in an int; a launch has fewer than 2^32 threads
  if (K > kMaxBeams || width > kMaxWidth || (long long)K * V > 0x7fff0000ll || B >= 1 << 22 || (long long)B * K * pieces_of(V) >= 1 << 26)
    return RNNT_MI355X_UNSUPPORTED_SIZE;
  return RNNT_MI355X_OK;
}

// ---- states in their new order ------------------------------------------------------------------------------------------
struct ReorderTensor {
  const char* src;
  char* dst;
  long long outer_bytes, batch_bytes, beam_bytes;  // strides of src; dst is dense [outer, B, width, row]
  long long row_bytes;
  unsigned first, pieces;  // first work item of this tensor, work items a row
};
struct ReorderArgs {
  ReorderTensor t[RNNT_MI355X_REORDER_MAX];
  const int32_t* parent;
  int n, B, K, width;
};
constexpr long long kLaunchItems = 1 << 25;
constexpr int kRowPiece = 4096;  // bytes of a row that one wavefront copies: four 16-byte loads a lane

// A wavefront per piece of a row: bound by memory, or by the launch for the states of a single utterance (4 us); all tensors of
// a step go in one launch.
__global__ __launch_bounds__(256) void k_beam_reorder(ReorderArgs a, unsigned first, unsigned items) {
  const unsigned id = first + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (id >= items) return;
  int n = 0;
#pragma unroll
  for (int i = 1; i < RNNT_MI355X_REORDER_MAX; ++i)
    if (i < a.n && id >= a.t[i].first) n = i;
  const ReorderTensor t = a.t[n];
  const unsigned local = id - t.first, row = local / t.pieces, piece = local - row * t.pieces;
  const unsigned bw = row % (unsigned)(a.B * a.width), outer = row / (unsigned)(a.B * a.width), b = bw / (unsigned)a.width;
  const int parent = a.parent[bw];
  const long long at = (long long)piece * kRowPiece;
  const int n_bytes = (int)min((long long)kRowPiece, t.row_bytes - at);
  char* d = t.dst + (long long)row * t.row_bytes + at;
  const bool there = parent >= 0 && parent < a.K;
  const char* s = t.src + outer * t.outer_bytes + b * t.batch_bytes + (there ? parent : 0) * t.beam_bytes + at;
  u4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int o = (j * 64 + lane) * 16;
    v[j] = u4{0u, 0u, 0u, 0u};
    if (there && o + 16 <= n_bytes) v[j] = *reinterpret_cast<const u4_any*>(s + o);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int o = (j * 64 + lane) * 16;
    if (o + 16 <= n_bytes) *reinterpret_cast<u4_any*>(d + o) = v[j];
  }
  const int tail = n_bytes & ~15;  // the last bytes of a row, one a lane
  if (tail + lane < n_bytes) d[tail + lane] = there ? s[tail + lane] : 0;
}

}  // namespace

extern "C" int rnnt_mi355x_beam_select_workspace_bytes(int B, int K, int V, int width, size_t* out_bytes) {
  if (!out_bytes) return RNNT_MI355X_INVALID_VALUE;
  const int rc = check_select(B, K, V, width);
  if (rc != RNNT_MI355X_OK) return rc;
  *out_bytes = (size_t)B * K * pieces_of(V) * (sizeof(PieceSum) + sizeof(RowKey) * list_lanes(width));
  return RNNT_MI355X_OK;
}

extern "C" int rnnt_mi355x_beam_select(const void* logits, long long logits_batch_stride, long long logits_beam_stride, int dtype,
                                       const void* enc, long long enc_batch_stride, const float* scores, const uint8_t* allowed,
                                       long long allowed_batch_stride, const uint8_t* finished, int end, int B, int K, int V,
                                       int width, float* out_scores, int32_t* out_parent, int32_t* out_token, void* workspace,
                                       void* hip_stream) {
  const int rc = check_select(B, K, V, width);
  if (rc != RNNT_MI355X_OK) return rc;
  if (!logits || !scores || !out_scores || !out_parent || !out_token || logits_batch_stride < 0 || logits_beam_stride < 0 ||
      enc_batch_stride < 0 || allowed_batch_stride < 0 || (finished && (end < 0 || end >= V)) || (pieces_of(V) && !workspace))
    return RNNT_MI355X_INVALID_VALUE;
  BeamArgs a;
  a.logits = logits;
  a.enc = enc;
  a.scores = scores;
  a.allowed = allowed;
  a.finished = finished;
  a.logits_b = logits_batch_stride;
  a.logits_k = logits_beam_stride;
  a.enc_b = enc_batch_stride;
  a.allowed_b = allowed_batch_stride;
  a.B = B;
  a.K = K;
  a.V = V;
  a.width = width;
  a.end = end;
  a.pieces = pieces_of(V);
  a.out_scores = out_scores;
  a.out_parent = out_parent;
  a.out_token = out_token;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (dtype) {
    case RNNT_MI355X_FP32: return launch_select_width<Fp32>(a, workspace, st);
    case RNNT_MI355X_BF16: return launch_select_width<Bf16>(a, workspace, st);
    case RNNT_MI355X_FP16: return launch_select_width<Fp16>(a, workspace, st);
  }
  return RNNT_MI355X_INVALID_VALUE;
}

extern "C" int rnnt_mi355x_beam_reorder(const rnnt_mi355x_reorder_tensor* tensors, int n_tensors, const int32_t* parent, int B, int K,
                                        int width, void* hip_stream) {
  if (!tensors || !parent || n_tensors < 1 || B < 1 || K < 1 || width < 1) return RNNT_MI355X_INVALID_VALUE;
  if (n_tensors > RNNT_MI355X_REORDER_MAX || (long long)B * width > 0x7fffffffll) return RNNT_MI355X_UNSUPPORTED_SIZE;
  ReorderArgs a;
  a.parent = parent;
  a.n = n_tensors;
  a.B = B;
  a.K = K;
  a.width = width;
  long long items = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const rnnt_mi355x_reorder_tensor& t = tensors[i];
    if (!t.src || !t.dst || t.outer < 1 || t.row_bytes < 1 || t.outer_stride < 0 || t.batch_stride < 0 || t.beam_stride < 0)
      return RNNT_MI355X_INVALID_VALUE;
    const long long pieces = (t.row_bytes + kRowPiece - 1) / kRowPiece, rows = t.outer * B * width;
    if (t.outer > 0x7fffffffll || rows > 0x7fffffffll || pieces > 0x7fffffffll || rows * pieces > 0x7fffffffll)
      return RNNT_MI355X_UNSUPPORTED_SIZE;
    a.t[i] = ReorderTensor{static_cast<const char*>(t.src), static_cast<char*>(t.dst), t.outer_stride, t.batch_stride, t.beam_stride,
                           t.row_bytes, (unsigned)items, (unsigned)pieces};
    items += rows * pieces;
    if (items > 0x7fffffffll) return RNNT_MI355X_UNSUPPORTED_SIZE;
  }
  // a launch has fewer than 2^32 threads
  for (long long first = 0; first < items; first += kLaunchItems) {
    const long long n = items - first < kLaunchItems ? items - first : kLaunchItems;
    k_beam_reorder<<<(unsigned)((n + 3) / 4), 256, 0, static_cast<hipStream_t>(hip_stream)>>>(a, (unsigned)first, (unsigned)(first + n));
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
  }
  return RNNT_MI355X_OK;
}
