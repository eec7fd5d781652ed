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

// Bound by memory: dy and the saved tensor read once, dz written once.
template <class T>
__global__ __launch_bounds__(kDzGroups * kDzLanes) void k_layer_dz(DzArgs a) {
  __shared__ float sums[kDzLanes][kDzGroups * 8 + 4];
  load_offset(a.drop);
  const int gx = threadIdx.x % kDzGroups, ty = threadIdx.x / kDzGroups;
  const int n0 = (blockIdx.x * kDzGroups + gx) * 8, left = a.N - n0;
  const int m0 = blockIdx.y * a.rows, m1 = min(a.M, m0 + a.rows);
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
        if (left >= 8) store8<T>(q, v);
        else store_some<T>(q, left, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += v[i];
    }
  }
  if (!a.partial) return;  // uniform
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[ty][gx * 8 + i] = sum[i];
  __syncthreads();
  const int n = blockIdx.x * kDzGroups * 8 + threadIdx.x;
  if (n < a.N) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kDzLanes; ++i) s += sums[i][threadIdx.x];
    a.partial[(long long)blockIdx.y * a.N + n] = s;
  }
}

// db: the row blocks' sums, 64 columns and 16 blocks at a time; the order is fixed.
template <class T>
__global__ __launch_bounds__(1024) void k_layer_db(const float* partial, int blocks, int N, typename T::elem* db) {
  __shared__ float sums[16][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6, n = blockIdx.x * 64 + c;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int i = r; i < blocks; i += 16) s += partial[(long long)i * N + n];
  }
  sums[r][c] = s;
  __syncthreads();
  if (r == 0 && n < N) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += sums[i][c];
    db[n] = from_float<T>(s);
  }
}

// ---- joining the splits of a product -------------------------------------------------------------------------------------
// A block takes 32 groups of eight columns of one tile's rows; 8 lanes share a group's splits.  The order is fixed.
template <class T>
__global__ __launch_bounds__(256) void k_layer_join(GemmArgs g, int bm, int bn) {
  __shared__ float sums[8][32][9];
  const int c = threadIdx.x & 31, s0 = threadIdx.x >> 5, groups = bn / 8, per_tile = bm * groups / 32;
  const int tile = blockIdx.x / per_tile, group = (blockIdx.x - tile * per_tile) * 32 + c;
  int tm, tn;
  place_of(g, g.whole + tile, tm, tn);
  const long long m = (long long)tm * bm + group / groups;
  const int n = tn * bn + 8 * (group % groups), left = g.N - n;
  const bool in = m < g.M && left > 0;
  float v[1][8] = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
  if (in) {
    const float* p = g.partial + (long long)tile * g.splits * bm * bn + 8 * group;
#pragma unroll 4
    for (int s = s0; s < g.splits; s += 8) {
      float w[8];
      unpack8<Fp32>(load8_raw<Fp32>(p + (long long)s * bm * bn), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[0][i] += w[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[s0][c][i] = v[0][i];
  __syncthreads();
  if (s0 != 0 || !in) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int s = 1; s < 8; ++s) v[0][i] += sums[s][c][i];
  DropArgs drop = g.e.drop;
  if (drop.drop) load_offset(drop);
  finish<T, 1>(g.e, drop, {m}, g.M, n, left, v);
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
  // Rounds of one tile a CU are done whole.  The rest would leave CUs idle for a round: it is cut along k until there are
  // two pieces for every CU (one of the largest block), each of four steps of 32 k at least.
  const int want = p.block == kBlock256x256 ? kCUs : 2 * kCUs;
  const int others = (int)(tiles % kCUs);
  p.splits = others == 0 ? 1 : want / others;
  if (p.splits > steps / 4) p.splits = steps / 4;
  if (tiles > 16 * kCUs || p.splits < 2) p.splits = 1;
  p.k_each = ceil_div(ceil_div(K, p.splits), 64) * 64;
  p.splits = ceil_div(K, p.k_each);
  p.whole = (int)(p.splits == 1 ? tiles : tiles - others);
  p.partial_bytes = (size_t)(tiles - p.whole) * p.splits * p.bm * p.bn * sizeof(float);
  return p;
}

// 16-byte pieces that begin on 16-byte boundaries, in a tile whose byte offsets fit 31 bits.
bool can_go_direct(const void* p, long long ld, int inner, int dtype) {
  return dtype != RNNT_MI355X_FP32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && inner % 8 == 0 && ld < (1 << 21);
}

size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

template <class T>
int gemm_of(int product, int block, bool direct, const GemmArgs& g, hipStream_t st) {
  if constexpr (T::code == RNNT_MI355X_FP32) return layer_gemm_fp32(product, block, direct, &g, st);
  else if constexpr (T::code == RNNT_MI355X_BF16) return layer_gemm_bf16(product, block, direct, &g, st);
  else return layer_gemm_fp16(product, block, direct, &g, st);
}

template <class T>
int run_product(int product, const Plan& p, const void* a, long long a_ld, const void* b, long long b_ld, int M, int N, int K,
                const Epilogue& e, float* partial, hipStream_t st) {
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
  g.partial = partial;
  g.e = e;
  const int rc = gemm_of<T>(product, p.block, p.direct, g, st);
  const int others = p.tiles_m * p.tiles_n - p.whole;
  if (rc != RNNT_MI355X_OK || others == 0) return rc;
  k_layer_join<T><<<(unsigned)others * (p.bm * p.bn / 256), 256, 0, st>>>(g, p.bm, p.bn);
  return hipGetLastError() == hipSuccess ? RNNT_MI355X_OK : RNNT_MI355X_LAUNCH_FAILURE;
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
  // 32-bit indexes inside an operand's rows and of its tiles
  if (l->rows > 0x7fff0000ll || l->in > (1 << 24) || l->out > (1 << 24) || ((l->rows + 63) / 64) * ((l->in + 63) / 64) > 0x7fffffffll ||
      ((l->rows + 63) / 64) * ((l->out + 63) / 64) > 0x7fffffffll)
    return RNNT_MI355X_UNSUPPORTED_SIZE;
  return RNNT_MI355X_OK;
}

int saved_by(const rnnt_mi355x_layer* l) {
  if (l->act == kLinear) return kNothing;
  if (l->aux) return kPreActivation;
  const bool from_y = !l->residual && (l->act == kRelu || (l->act == kTanh && l->dtype == RNNT_MI355X_FP32));
  return from_y && l->y ? kOutput : -1;
}

// row blocks of the dz pass: at most 1024 partial sums a column
int dz_rows(long long M) { return M <= 65536 ? 64 : (int)((M + 1023) / 1024 + 7) / 8 * 8; }

// dz's rows in the workspace.  Rows a multiple of 4 KiB apart put the same piece of all rows of a tile into the same few
// memory channels: 32768 x 4096 x 1024 in bfloat16 ran 300 us with such rows and 257 us with rows 128 bytes longer.
long long dz_stride(int out, int dtype) {
  const long long e = dtype == RNNT_MI355X_FP32 ? 4 : 2;
  return out * e % 4096 == 0 ? out + 128 / e : out;
}

struct BackwardPlan {
  bool need_dz;  // else dz is dy
  size_t dz_at, sums_at, partial_at, bytes;
  Plan dx, dk;
};
BackwardPlan plan_backward(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride) {
  BackwardPlan b;
  const int M = (int)l->rows;
  const size_t e = l->dtype == RNNT_MI355X_FP32 ? 4 : 2;
  b.need_dz = l->act != kLinear || l->drop16 != 0;
  b.dz_at = 0;
  b.sums_at = align_up(b.need_dz ? (size_t)M * dz_stride(l->out, l->dtype) * e : 0);
  b.partial_at = b.sums_at + align_up((size_t)ceil_div(M, dz_rows(M)) * l->out * sizeof(float));
  // dz lies in the workspace, on a 256-byte boundary
  const bool dz_direct = b.need_dz ? l->dtype != RNNT_MI355X_FP32 && l->out % 8 == 0 && l->out < (1 << 21) : can_go_direct(dy, dy_stride, l->out, l->dtype);
  b.dx = plan_product(kInputGrad, l->dtype, M, l->in, l->out, dz_direct && can_go_direct(l->kernel, l->kernel_stride, l->out, l->dtype));
  b.dk = plan_product(kKernelGrad, l->dtype, l->in, l->out, M, dz_direct && can_go_direct(l->x, l->x_stride, l->in, l->dtype));
  b.bytes = b.partial_at + (b.dx.partial_bytes > b.dk.partial_bytes ? b.dx.partial_bytes : b.dk.partial_bytes);
  return b;
}
Plan plan_forward(const rnnt_mi355x_layer* l) {
  return plan_product(kForward, l->dtype, (int)l->rows, l->out, l->in,
                      can_go_direct(l->x, l->x_stride, l->in, l->dtype) && can_go_direct(l->kernel, l->kernel_stride, l->out, l->dtype));
}

template <class T>
int forward(const rnnt_mi355x_layer* l, void* workspace, hipStream_t st) {
  Epilogue e = plain_output(l->y, l->out);
  e.bias = l->bias;
  e.residual = l->residual;
  e.residual_ld = l->residual_stride;
  e.aux = l->act == kLinear ? nullptr : l->aux;
  e.act = l->act;
  e.drop = drop_args(l->drop16, l->seed, l->offset, l->offset_dev);
  return run_product<T>(kForward, plan_forward(l), l->x, l->x_stride, l->kernel, l->kernel_stride, (int)l->rows, l->out, l->in, e,
                        static_cast<float*>(workspace), st);
}

template <class T>
int backward(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride, void* dx, void* dkernel, void* dbias, void* workspace, int from,
             hipStream_t st) {
  const BackwardPlan b = plan_backward(l, dy, dy_stride);
  const int M = (int)l->rows;
  char* ws = static_cast<char*>(workspace);
  const void* dz = b.need_dz ? ws + b.dz_at : dy;
  const long long dz_ld = b.need_dz ? dz_stride(l->out, l->dtype) : dy_stride;
  float *sums = reinterpret_cast<float*>(ws + b.sums_at), *partial = reinterpret_cast<float*>(ws + b.partial_at);
  const int blocks = ceil_div(M, dz_rows(M));
  if (b.need_dz || dbias) {
    DzArgs a;
    a.dy = dy;
    a.saved = from == kPreActivation ? l->aux : l->y;
    a.dz = b.need_dz ? ws + b.dz_at : nullptr;
    a.partial = dbias ? sums : nullptr;
    a.dy_ld = dy_stride;
    a.dz_ld = dz_ld;
    a.M = M;
    a.N = l->out;
    a.rows = dz_rows(M);
    a.act = l->act;
    a.from = from;
    a.drop = drop_args(l->drop16, l->seed, l->offset, l->offset_dev);
    k_layer_dz<T><<<dim3((unsigned)ceil_div(l->out, kDzGroups * 8), (unsigned)blocks), kDzGroups * kDzLanes, 0, st>>>(a);
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
  }
  if (dbias) {
    k_layer_db<T><<<(unsigned)ceil_div(l->out, 64), 1024, 0, st>>>(sums, blocks, l->out, static_cast<typename T::elem*>(dbias));
    if (hipGetLastError() != hipSuccess) return RNNT_MI355X_LAUNCH_FAILURE;
  }
  int rc = RNNT_MI355X_OK;
  if (dx) rc = run_product<T>(kInputGrad, b.dx, dz, dz_ld, l->kernel, l->kernel_stride, M, l->in, l->out, plain_output(dx, l->in), partial, st);
  if (rc == RNNT_MI355X_OK && dkernel)
    rc = run_product<T>(kKernelGrad, b.dk, l->x, l->x_stride, dz, dz_ld, l->in, l->out, M, plain_output(dkernel, l->out), partial, st);
  return rc;
}

}  // namespace

extern "C" int rnnt_mi355x_layer_workspace_bytes(const rnnt_mi355x_layer* l, const void* dy, long long dy_stride, size_t* forward_bytes,
                                                 size_t* backward_bytes) {
  const int rc = check_layer(l);
  if (rc != RNNT_MI355X_OK) return rc;
  if (backward_bytes && dy_stride < l->out) return RNNT_MI355X_INVALID_VALUE;
  if (forward_bytes) *forward_bytes = plan_forward(l).partial_bytes;
  if (backward_bytes) *backward_bytes = plan_backward(l, dy, dy_stride).bytes;
  return RNNT_MI355X_OK;
}

extern "C" int rnnt_mi355x_layer_forward(const rnnt_mi355x_layer* l, void* workspace, void* hip_stream) {
  const int rc = check_layer(l);
  if (rc != RNNT_MI355X_OK) return rc;
  if (!l->x || !l->kernel || !l->y || (l->residual && l->residual_stride < l->out)) return RNNT_MI355X_INVALID_VALUE;
  if (!workspace && plan_forward(l).partial_bytes) return RNNT_MI355X_INVALID_VALUE;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  switch (l->dtype) {
    case RNNT_MI355X_FP32: return forward<Fp32>(l, workspace, st);
    case RNNT_MI355X_BF16: return forward<Bf16>(l, workspace, st);
  }
  return forward<Fp16>(l, workspace, st);
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
