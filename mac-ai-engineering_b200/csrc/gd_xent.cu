// Softmax cross entropy of a vocabulary projection that never keeps the logits:
//   l = x W^T,   lse_i = log sum_v exp(l_iv),   loss_i = lse_i - l_i,label(i)
//   D_iv = (exp(l_iv - lse_i) - [v = label(i)]) g_i,   dx = D W,   dW = D^T x
// Forward: one product whose epilogue keeps a maximum and a sum for each row and 128 columns, then their join. Backward: the
// vocabulary in pieces; a piece's logits are formed again and leave as D in 16 bits (the matrix instruction's operand type), then
// one launch of both gradients' products. dW's rows of a piece are final; dx is summed over the pieces in fp32.
#include <cstdint>

#include "gd_gemm.cuh"

namespace gd {
namespace xent {
namespace {

using gemm::Op;
using gemm::Params;

constexpr int kPart = 128;          // columns of one (maximum, sum)
constexpr int kRows = 32;           // rows of a join CTA
constexpr int kJoinWarps = 16;
constexpr float kLn2 = 0.6931471805599453f;
enum Reduction { kNone, kMean, kSum };

struct Labels {
  const void* at;
  int is64;
  long long ignore;
  int V;
  __device__ __forceinline__ long long of(int row) const {
    return is64 ? __ldg(static_cast<const long long*>(at) + row) : __ldg(static_cast<const int*>(at) + row);
  }
};

// Joins each row's parts: its maximum and the logarithm of its sum, its loss (at least 0: a sure row's sum is 1 and more); for a mean or sum the last CTA adds the CTAs' sums in their order.
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const float2* __restrict__ part, const float* __restrict__ target,
                                                               int parts, int n, Labels lab, int reduction,
                                                               float2* __restrict__ lse, float* __restrict__ loss,
                                                               float2* sums, unsigned int* counter) {
  __shared__ float2 sh[kJoinWarps][kRows];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * kRows + lane;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float2 v) {  // (a NaN sum stays)
    const float next = wattn::max3(m, v.x, v.x), ref = next == -INFINITY ? 0.f : next;
    s = s * wattn::ex2((m - ref) * gemm::kLog2e) + v.y * wattn::ex2((v.x - ref) * gemm::kLog2e);
    m = next;
  };
  if (row < n) {
    int p = warp;
    for (; p + 3 * kJoinWarps < parts; p += 4 * kJoinWarps) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __ldcs(part + (long long)(p + i * kJoinWarps) * n + row);
#pragma unroll
      for (int i = 0; i < 4; ++i) add(v[i]);
    }
    for (; p < parts; p += kJoinWarps) add(__ldcs(part + (long long)p * n + row));
  }
  sh[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp == 0) {
    m = -INFINITY, s = 0.f;
    for (int w = 0; w < kJoinWarps; ++w) add(sh[w][lane]);
    float x = 0.f, kept = 0.f;
    if (row < n) {
      const long long l = lab.of(row);
      const float rest = log2f(s);
      if (l != lab.ignore) {
        kept = 1.f;
        x = l < 0 || l >= lab.V ? NAN : (m - target[row]) + kLn2 * rest;
      }
      if (lse != nullptr) lse[row] = make_float2(m, rest);
      if (reduction == kNone) loss[row] = x;
    }
    if (reduction != kNone) {
      x = warp_sum(x);
      kept = warp_sum(kept);
      if (lane == 0) {
        sums[blockIdx.x] = make_float2(x, kept);
        __threadfence();
        last = atomicAdd(counter, 1u) + 1u == gridDim.x;
      }
    }
  }
  if (reduction == kNone) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float x = 0.f, kept = 0.f;  // (a thread's CTAs in order, then the threads': the same sum every run)
  for (unsigned int i = threadIdx.x; i < gridDim.x; i += 32 * kJoinWarps) {
    const float2 v = __ldcg(sums + i);
    x += v.x;
    kept += v.y;
  }
  x = warp_sum(x);
  kept = warp_sum(kept);
  if (lane == 0) sh[warp][0] = make_float2(x, kept);
  __syncthreads();
  if (threadIdx.x == 0) {
    x = kept = 0.f;
    for (int w = 0; w < kJoinWarps; ++w) x += sh[w][0].x, kept += sh[w][0].y;
    loss[0] = reduction == kMean ? x / kept : x;  // (no row: NaN)
  }
}

// What each row's softmax - onehot is multiplied by before it is rounded, and what the products are multiplied by: g_i over the
// largest |g| of the call, and that. A row that knows nothing of its label then has -1 exactly where it would have the rounded
// -g_i, an error all rows of a mean share (up to 2^-8 of both gradients). float16 carries 2^15 more, so that D keeps its 11 bits
// over 28 binades below its largest value. One CTA.
__global__ void __launch_bounds__(1024) factors_kernel(const float* __restrict__ g, Labels lab, int n, int reduction, bool half,
                                                       float* __restrict__ row_scale, float* __restrict__ factor) {
  __shared__ float sh[32];
  __shared__ float share;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto all = [&](float v, bool add) {  // the sum or the maximum over the CTA
    v = add ? warp_sum(v) : __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = sh[lane];
      v = add ? warp_sum(v) : __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
      if (lane == 0) share = v;
    }
    __syncthreads();
    return share;
  };
  float one = 0.f, top = 0.f;
  if (reduction != kNone) {
    float c = 0.f;  // (whole numbers up to 2^24: exact)
    for (int i = threadIdx.x; i < n; i += 1024) c += lab.of(i) != lab.ignore ? 1.f : 0.f;
    c = all(c, true);
    one = reduction == kMean ? g[0] / c : g[0];
    top = c > 0.f ? fabsf(one) : 0.f;
  } else {
    for (int i = threadIdx.x; i < n; i += 1024)
      if (lab.of(i) != lab.ignore) top = wattn::max3(top, fabsf(g[i]), top);
    top = all(top, false);
  }
  const float lift = half ? 32768.f : 1.f;
  const bool plain = !(top < INFINITY);  // an infinity or NaN goes the way it came
  if (threadIdx.x == 0) *factor = plain ? 1.f : top / lift;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const long long l = lab.of(i);
    const float x = reduction == kNone ? g[i] : one;
    row_scale[i] = l == lab.ignore ? 0.f : l < 0 || l >= lab.V ? NAN : plain ? x : top > 0.f ? x / top * lift : 0.f;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr size_t kHead = 256;  // the error word, the join's counter (at 64), the products' factor (at 128)
size_t up(size_t n) { return (n + 255) / 256 * 256; }

struct FwdPlan {
  int parts, ctas;
  size_t part, target, sums, total;
};
FwdPlan fwd_plan(long long n, int V) {
  FwdPlan f;
  f.parts = gemm::blocks_of(V, kPart);
  f.ctas = gemm::blocks_of(n, kRows);
  f.part = kHead;
  f.target = f.part + up((size_t)f.parts * n * sizeof(float2));
  f.sums = f.target + up((size_t)n * sizeof(float));
  f.total = f.sums + up((size_t)f.ctas * sizeof(float2));
  return f;
}

// The pieces of the vocabulary: D of one piece takes at most kPieceBytes (a multiple of a tile's columns, at least one tile).
constexpr size_t kPieceBytes = (size_t)256 << 20;
struct BwdPlan {
  int pieces, cols;  // cols: of every piece but the last
  long long ldd;
  size_t rows, d, sum, total;
};
BwdPlan bwd_plan(long long n, int D, int V) {
  BwdPlan b;
  long long most = (long long)(kPieceBytes / 2) / n / gemm::kTileN * gemm::kTileN;
  if (most < gemm::kTileN) most = gemm::kTileN;
  b.pieces = gemm::blocks_of(V, (int)(most < V ? most : V));
  b.cols = gemm::blocks_of(gemm::blocks_of(V, b.pieces), gemm::kTileN) * gemm::kTileN;
  b.pieces = gemm::blocks_of(V, b.cols);
  b.ldd = b.pieces > 1 ? b.cols : (V + 63ll) / 64 * 64;
  b.rows = kHead;
  b.d = b.rows + up((size_t)n * sizeof(float));
  b.sum = b.d + up((size_t)n * b.ldd * 2);
  b.total = b.sum + (b.pieces > 1 ? (size_t)gemm::blocks_of(n, gemm::kTileM) * gemm::blocks_of(D, gemm::kTileN) *
                                        (gemm::kTileM * gemm::kTileN * sizeof(float))
                                  : 0);
  return b;
}

struct Problem {
  const void *x, *w;
  long long ldx, ldw;
  int n, D, V;
  Labels lab;
  int reduction;
};

void label_params(Params& p, const Problem& q, ErrorWord* err) {
  p.labels = q.lab.at, p.label64 = q.lab.is64, p.ignore = q.lab.ignore, p.err = err;
}

void shape(Op& op, long long M, long long N) {
  op.M = (int)M, op.N = (int)N;
  op.tiles_m = gemm::blocks_of(M, gemm::kTileM), op.tiles_n = gemm::blocks_of(N, gemm::kTileN);
}

template <typename T>
int forward(const Problem& q, float* loss, float2* lse, char* ws, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const FwdPlan f = fwd_plan(q.n, q.V);
  Params p = {};
  p.ops = 1;
  label_params(p, q, reinterpret_cast<ErrorWord*>(ws));
  p.part = reinterpret_cast<float2*>(ws + f.part);
  p.target = reinterpret_cast<float*>(ws + f.target);
  Op& o = p.op[0];
  shape(o, q.n, q.V);
  o.kb[0] = gemm::blocks_of(q.D, gemm::kBlockK);
  if (!gemm::operand_map(&o.a[0], q.x, dt, q.n, q.D, q.ldx, false) || !gemm::operand_map(&o.b[0], q.w, dt, q.V, q.D, q.ldw, false))
    return GD_ERR_LAUNCH;
  if (const int st = gemm::launch<T, gemm::kLse>(p, stream)) return st;
  join_kernel<<<f.ctas, 32 * kJoinWarps, 0, stream>>>(p.part, p.target, f.parts, q.n, q.lab, q.reduction, lse, loss,
                                                     reinterpret_cast<float2*>(ws + f.sums),
                                                     reinterpret_cast<unsigned int*>(ws + 64));
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T>
int backward(const Problem& q, const float2* lse, const float* dloss, void* dx, void* dw, char* ws, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const BwdPlan b = bwd_plan(q.n, q.D, q.V);
  float* const row_scale = reinterpret_cast<float*>(ws + b.rows);
  float* const factor = reinterpret_cast<float*>(ws + 128);
  factors_kernel<<<1, 1024, 0, stream>>>(dloss, q.lab, q.n, q.reduction, std::is_same<T, __half>::value, row_scale, factor);
  if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  void* const d = ws + b.d;
  const int kd = gemm::blocks_of(q.D, gemm::kBlockK);
  for (int i = 0; i < b.pieces; ++i) {
    const long long v0 = (long long)i * b.cols;
    const int cols = (int)(q.V - v0 < b.cols ? q.V - v0 : b.cols);
    const char* w = static_cast<const char*>(q.w) + v0 * q.ldw * 2;
    Params p = {};
    p.ops = 1;
    label_params(p, q, reinterpret_cast<ErrorWord*>(ws));
    p.v0 = (int)v0, p.lse = lse, p.row_scale = row_scale;
    Op& o = p.op[0];
    shape(o, q.n, cols);
    o.kb[0] = kd;
    if (!gemm::operand_map(&o.a[0], q.x, dt, q.n, q.D, q.ldx, false) || !gemm::operand_map(&o.b[0], w, dt, cols, q.D, q.ldw, false) ||
        !gemm::slab_map(&o.c, d, dt, q.n, cols, b.ldd))
      return GD_ERR_LAUNCH;
    if (const int st = gemm::launch<T, gemm::kDLogit>(p, stream)) return st;
    Params r = {};
    r.err = p.err;
    bool ok = true;
    if (dx != nullptr) {  // dx += D W
      Op& g = r.op[r.ops++];
      shape(g, q.n, q.D);
      g.kb[0] = gemm::blocks_of(cols, gemm::kBlockK);
      g.b_mn = true;
      g.sum_mode = b.pieces == 1 ? 0 : i == 0 ? 1 : i + 1 < b.pieces ? 2 : 3;
      g.sum = reinterpret_cast<float*>(ws + b.sum);
      g.factor = factor;
      ok = ok && gemm::operand_map(&g.a[0], d, dt, q.n, cols, b.ldd, false) &&
           gemm::operand_map(&g.b[0], w, dt, cols, q.D, q.ldw, true) && gemm::slab_map(&g.c, dx, dt, q.n, q.D, q.D);
    }
    if (dw != nullptr) {  // dW = D^T x
      Op& g = r.op[r.ops++];
      shape(g, cols, q.D);
      g.kb[0] = gemm::blocks_of(q.n, gemm::kBlockK);
      g.a_mn = g.b_mn = true;
      g.factor = factor;
      ok = ok && gemm::operand_map(&g.a[0], d, dt, q.n, cols, b.ldd, true) &&
           gemm::operand_map(&g.b[0], q.x, dt, q.n, q.D, q.ldx, true) &&
           gemm::slab_map(&g.c, static_cast<char*>(dw) + v0 * q.D * 2, dt, cols, q.D, q.D);
    }
    if (!ok) return GD_ERR_LAUNCH;
    if (const int st = gemm::launch<T, gemm::kStore>(r, stream)) return st;
  }
  return GD_OK;
}

int check(int dtype, int reduction, long long rows, int D, int V, long long ldx, long long ldw) {
  if ((dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) || reduction < kNone || reduction > kSum) return GD_ERR_ARG;
  if (rows < 0 || rows > (1ll << 24) || D <= 0 || D % 8 || D > (1 << 24) || V <= 0 || V > (1 << 24) || ldx < D || ldw < D ||
      ldx >= (1ll << 38) || ldw >= (1ll << 38))
    return GD_ERR_SHAPE;
  return ldx % 8 || ldw % 8 ? GD_ERR_ALIGN : GD_OK;
}

bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

}  // namespace
}  // namespace xent
}  // namespace gd

extern "C" size_t gd_xent_workspace_bytes(long long rows, int D, int V, int for_backward) {
  using namespace gd::xent;
  if (check(GD_BFLOAT16, kNone, rows, D, V, D, D) != GD_OK || rows == 0) return 0;
  return for_backward ? bwd_plan(rows, D, V).total : fwd_plan(rows, V).total;
}

extern "C" int gd_xent_fwd(const void* x, const void* w, const void* labels, int label64, float* loss, float* lse,
                           int reduction, long long ignore, int dtype, long long rows, int D, int V, long long ldx,
                           long long ldw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gd::xent;
  if (const int st = check(dtype, reduction, rows, D, V, ldx, ldw)) return st;
  if (rows == 0) return GD_OK;
  if (x == nullptr || w == nullptr || labels == nullptr || loss == nullptr) return GD_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(lse) || !aligned16(workspace)) return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_xent_workspace_bytes(rows, D, V, 0)) return GD_ERR_WORKSPACE;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(workspace, 0, kHead, cs) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const Problem q = {x, w, ldx, ldw, (int)rows, D, V, {labels, label64, ignore, V}, reduction};
  char* ws = static_cast<char*>(workspace);
  float2* const kept = reinterpret_cast<float2*>(lse);
  return dtype == GD_FLOAT16 ? forward<__half>(q, loss, kept, ws, cs) : forward<__nv_bfloat16>(q, loss, kept, ws, cs);
}

extern "C" int gd_xent_bwd(const void* x, const void* w, const void* labels, int label64, const float* lse, const float* dloss,
                           void* dx, void* dw, int reduction, long long ignore, int dtype, long long rows, int D, int V,
                           long long ldx, long long ldw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gd::xent;
  if (const int st = check(dtype, reduction, rows, D, V, ldx, ldw)) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return dw == nullptr || cudaMemsetAsync(dw, 0, (size_t)V * D * 2, cs) == cudaSuccess ? GD_OK
                                                                                         : (cudaGetLastError(), GD_ERR_LAUNCH);
  if (x == nullptr || w == nullptr || labels == nullptr || lse == nullptr || dloss == nullptr) return GD_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(dx) || !aligned16(dw) || !aligned16(lse) || !aligned16(workspace))
    return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_xent_workspace_bytes(rows, D, V, 1)) return GD_ERR_WORKSPACE;
  if (dx == nullptr && dw == nullptr) return GD_OK;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  if (cudaMemsetAsync(workspace, 0, kHead, cs) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const Problem q = {x, w, ldx, ldw, (int)rows, D, V, {labels, label64, ignore, V}, reduction};
  char* ws = static_cast<char*>(workspace);
  const float2* const kept = reinterpret_cast<const float2*>(lse);
  return dtype == GD_FLOAT16 ? backward<__half>(q, kept, dloss, dx, dw, ws, cs)
                             : backward<__nv_bfloat16>(q, kept, dloss, dx, dw, ws, cs);
}
