// Softmax cross entropy of a vocabulary projection that never keeps the logits:
//   l = x W^T,   lse_i = log sum_v exp(l_iv),   loss_i = lse_i - l_i,label(i)
//   D_iv = (exp(l_iv - lse_i) - [v = label(i)]) g_i,   dx = D W,   dW = D^T x
// Rows whose label is ignored take no part: the others' x is gathered first (packed rows of x, `live` of them, a number that only
// the device knows; the products' tiles are counted there). Forward: one product whose epilogue keeps a maximum and a sum for each
// row and 128 columns, then their join. Backward: the vocabulary in pieces; a piece's logits are formed again and leave as D in 16
// bits (the matrix instruction's operand type), then one launch of both gradients' products. dW's rows of a piece are final; dx is
// summed over the pieces in fp32, and spread over its rows at the end.
#include <cstdint>

#include "gd_gemm.cuh"

namespace gd {
namespace xent {
namespace {

using gemm::Op;
using gemm::Params;

constexpr int kPart = 128;          // columns of one (maximum, sum)
constexpr int kRows = 8;            // rows of a join CTA
constexpr int kJoinThreads = 256, kJoinGroups = kJoinThreads / kRows;
constexpr float kLn2 = 0.6931471805599453f;
enum Reduction { kNone, kMean, kSum };

struct Labels {
  const void* at;
  int is64;
  long long ignore;
  int V;
  __device__ __forceinline__ long long of(long long row) const {
    return is64 ? __ldg(static_cast<const long long*>(at) + row) : __ldg(static_cast<const int*>(at) + row);
  }
};

// What the forward finds out about the labels and the backward needs again, int32: the number of live rows, (three unused,)
// each row's place among them (-1: ignored) [n], each live row's label (-1: not in the vocabulary) [n].
struct Plan {
  int *live, *place, *label;
  __host__ __device__ static Plan of(int* at, int n) { return {at, at + 4, at + 4 + n}; }
};
constexpr int kPlanInts(int n) { return 4 + 2 * n; }

// The sum over the CTA's threads (every thread gets it).
template <int WARPS>
__device__ __forceinline__ int cta_sum(int v, int* sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) s += sh[w];
  return s;
}

__device__ __forceinline__ void copy_row(const uint16_t* from, uint16_t* to, int D, int lane) {
  int c = lane * 8;
  for (; c + 768 < D; c += 1024) {  // (four loads on their way)
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldg(reinterpret_cast<const uint4*>(from + c + 256 * i));
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(to + c + 256 * i) = v[i];
  }
  for (; c < D; c += 256) *reinterpret_cast<uint4*>(to + c) = __ldg(reinterpret_cast<const uint4*>(from + c));
}
// Rows of the packed x: at least a stage's, so that the loads of few rows find memory (zeros) where they would be filled. (4 rows,
// 2,048 wide, 128,000 words: the loss takes 105 us, with a matrix of 4 rows 150; from 32 rows on there is no difference.)
__host__ __device__ constexpr int packed_rows(int n) { return n < 64 ? 64 : n; }
// zeros in what is left of the live rows' last tile of the contraction (dW sums over the rows of whole stages)
__device__ __forceinline__ void clear_rows(uint16_t* out, long long ld, int live, int n, int D, int w0, int warps, int lane) {
  const int end = min(packed_rows(n), (live + gemm::kBlockK - 1) / gemm::kBlockK * gemm::kBlockK);
  for (int r = live + w0; r < end; r += warps)
    for (int c = lane * 8; c < D; c += 256) *reinterpret_cast<uint4*>(out + r * ld + c) = make_uint4(0, 0, 0, 0);
}

// The plan of the rows [r0, r1) of each CTA, and their x, the live ones packed, `ld` elements from row to row. A CTA counts the live
// rows before its own by itself (reading up to 8 n bytes of labels, 592 CTAs at most), so that one launch numbers and moves them all.
// The first CTA clears the workspace's head, the last writes the total.
constexpr int kPlanThreads = 256;
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(Labels lab, const uint16_t* __restrict__ x, long long ldx, int n, int D,
                                                            int step, Plan plan, uint16_t* __restrict__ out, long long ld, int* head) {
  constexpr int kWarps = kPlanThreads / 32;
  __shared__ int sh[kWarps], before[kWarps];
  const int r0 = (int)min((long long)blockIdx.x * step, (long long)n), r1 = (int)min((long long)r0 + step, (long long)n);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x < 64) head[threadIdx.x] = 0;
  int c = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < r0; i += kPlanThreads) c += lab.of(i) != lab.ignore;
  int base = cta_sum<kWarps>(c, sh);
  for (int r = r0; r < r1; r += kPlanThreads) {
    const int i = r + threadIdx.x;
    const long long l = i < r1 ? lab.of(i) : lab.ignore;
    const bool keep = l != lab.ignore;
    const unsigned mask = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) before[warp] = __popc(mask);
    __syncthreads();
    int at = base, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) at += before[w];
      all += before[w];
    }
    at += __popc(mask & ((1u << lane) - 1u));
    if (i < r1) plan.place[i] = keep ? at : -1;
    if (keep) plan.label[at] = l < 0 || l >= lab.V ? -1 : (int)l;
    base += all;
  }
  __syncthreads();  // the CTA's places
  for (int i = r0 + warp; i < r1; i += kWarps) {
    const int r = plan.place[i];
    if (r >= 0) copy_row(x + i * ldx, out + r * ld, D, lane);
  }
  if (r1 == n) {  // (the last CTA)
    if (threadIdx.x == 0) *plan.live = base;
    clear_rows(out, ld, base, n, D, warp, kWarps, lane);
  }
}

// The same rows again, for the backward; also clears its workspace's head. A warp a row.
__global__ void __launch_bounds__(256) gather_kernel(const uint16_t* __restrict__ x, long long ldx, int n, int D, Plan plan,
                                                     uint16_t* __restrict__ out, long long ld, int* head) {
  const int warps = gridDim.x * 8, w0 = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x < 64) head[threadIdx.x] = 0;
  for (int i = w0; i < n; i += warps) {
    const int r = __ldg(plan.place + i);
    if (r >= 0) copy_row(x + i * ldx, out + r * ld, D, lane);
  }
  clear_rows(out, ld, __ldg(plan.live), n, D, w0, warps, lane);
}

// Every row of dx: its live row's, or zeros. A warp a row.
__global__ void __launch_bounds__(256) spread_kernel(const uint16_t* __restrict__ in, long long ld, int n, int D,
                                                     const int* __restrict__ place, uint16_t* __restrict__ dx) {
  const int warps = gridDim.x * 8, lane = threadIdx.x & 31;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += warps) {
    const int r = __ldg(place + i);
    for (int c = lane * 8; c < D; c += 256)
      *reinterpret_cast<uint4*>(dx + (long long)i * D + c) =
          r < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(in + r * ld + c);
  }
}
// Joins each row's parts: its maximum and the logarithm of its sum, its loss (at least 0: a sure row's sum is 1 and more); for a
// mean or sum the last CTA adds the CTAs' sums in their order. Parts and targets lie by live rows, losses by rows. A thread takes
// every 32nd part of a row. (777 rows of 393 parts: 6 us, with 32 rows a CTA 8 us; 7,370 of 1,000: 20 us, 26 us)
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const float2* __restrict__ part, const float* __restrict__ target,
                                                            int parts, int n, Plan plan, int reduction,
                                                            float2* __restrict__ lse, float* __restrict__ loss, float* sums,
                                                            unsigned int* counter) {
  __shared__ float2 sh[kJoinGroups][kRows];
  __shared__ float warps[kJoinThreads / 32];
  __shared__ bool last;
  const int group = threadIdx.x / kRows, at = threadIdx.x % kRows, i = blockIdx.x * kRows + at;
  const int row = i < n ? __ldg(plan.place + i) : -1;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float2 v) {  // (a NaN sum stays)
    const float next = wattn::max3(m, v.x, v.x), ref = next == -INFINITY ? 0.f : next;
    s = s * wattn::ex2((m - ref) * gemm::kLog2e) + v.y * wattn::ex2((v.x - ref) * gemm::kLog2e);
    m = next;
  };
  if (row >= 0) {
    int p = group;
    for (; p + 3 * kJoinGroups < parts; p += 4 * kJoinGroups) {
      float2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __ldcs(part + (long long)(p + j * kJoinGroups) * n + row);
#pragma unroll
      for (int j = 0; j < 4; ++j) add(v[j]);
    }
    for (; p < parts; p += kJoinGroups) add(__ldcs(part + (long long)p * n + row));
  }
  sh[group][at] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < 32) {
    float x = 0.f;
    if (threadIdx.x < kRows) {
      m = -INFINITY, s = 0.f;
      for (int g = 0; g < kJoinGroups; ++g) add(sh[g][at]);
      if (row >= 0) {
        const float rest = log2f(s);
        x = __ldg(plan.label + row) < 0 ? NAN : fmaf(kLn2, rest, m - target[row]);
        if (lse != nullptr) lse[row] = make_float2(m, rest);
      }
      if (reduction == kNone && i < n) loss[i] = x;
    }
    if (reduction != kNone) {
      x = warp_sum(x);
      if (threadIdx.x == 0) {
        sums[blockIdx.x] = x;
        __threadfence();
        last = atomicAdd(counter, 1u) + 1u == gridDim.x;
      }
    }
  }
  if (reduction == kNone) return;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float x = 0.f;  // (a thread's CTAs in order, then the threads': the same sum every run)
  for (unsigned int j = threadIdx.x; j < gridDim.x; j += kJoinThreads) x += __ldcg(sums + j);
  x = warp_sum(x);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    x = 0.f;
    for (int w = 0; w < kJoinThreads / 32; ++w) x += warps[w];
    loss[0] = reduction == kMean ? x / (float)*plan.live : x;  // (no row: NaN)
  }
}

// What each live row's softmax - onehot is multiplied by before it is rounded, and what the products are multiplied by: g_i over
// the largest |g| of the call, and that. A row that knows nothing of its label then has -1 exactly where it would have the rounded
// -g_i, an error all rows of a mean share (up to 2^-8 of both gradients). float16 carries 2^15 more, so that D keeps its 11 bits
// over 28 binades below its largest value. One CTA.
__global__ void __launch_bounds__(1024) factors_kernel(const float* __restrict__ g, Plan plan, int n, int reduction, bool half,
                                                       float* __restrict__ row_scale, float* __restrict__ factor) {
  __shared__ float sh[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, live = *plan.live;
  float one = 0.f, top = 0.f;
  if (reduction != kNone) {
    one = reduction == kMean ? g[0] / (float)live : g[0];
    top = live > 0 ? fabsf(one) : 0.f;
  } else {
    for (int i = threadIdx.x; i < n; i += 1024)
      if (__ldg(plan.place + i) >= 0) top = wattn::max3(top, fabsf(g[i]), top);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if (lane == 0) sh[warp] = top;
    __syncthreads();
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(sh[lane])));
  }
  const float lift = half ? 32768.f : 1.f;
  const bool plain = !(top < INFINITY);  // an infinity or NaN goes the way it came
  if (threadIdx.x == 0) *factor = plain ? 1.f : top / lift;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const int r = __ldg(plan.place + i);
    if (r < 0) continue;
    const float x = reduction == kNone ? g[i] : one;
    row_scale[r] = __ldg(plan.label + r) < 0 ? NAN : plain ? x : top > 0.f ? x / top * lift : 0.f;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr size_t kHead = 256;  // the error word, the join's counter (at 64), the products' factor (at 128)
size_t up(size_t n) { return (n + 255) / 256 * 256; }
long long pitch(int D) { return (D + 63) / 64 * 64; }  // of the packed rows: whole 128-byte lines
int grid_of(long long rows) { return (int)(rows < 8 * 592 ? (rows + 7) / 8 : 592); }

struct FwdPlan {
  int parts, ctas;
  size_t plan, rows, part, target, sums, total;
};
FwdPlan fwd_plan(long long n, int D, int V) {
  FwdPlan f;
  f.parts = gemm::blocks_of(V, kPart);
  f.ctas = gemm::blocks_of(n, kRows);
  f.plan = kHead;
  f.rows = f.plan + up((size_t)kPlanInts((int)n) * 4);
  f.part = f.rows + up((size_t)packed_rows((int)n) * pitch(D) * 2);
  f.target = f.part + up((size_t)f.parts * n * sizeof(float2));
  f.sums = f.target + up((size_t)n * sizeof(float));
  f.total = f.sums + up((size_t)f.ctas * sizeof(float));
  return f;
}

// The pieces of the vocabulary: D of one piece takes at most kPieceBytes (a multiple of a tile's columns, at least one tile).
// One piece and few tiles of dx: its contraction over the vocabulary, far longer than a tile of dW's over the rows, is cut into
// slices with fp32 sums of their own. At 1,500 rows (half of them live), 768 wide, a
// vocabulary of 32,003, both gradients' products take 54 us; uncut, the longest tile alone takes 250 us.
constexpr size_t kPieceBytes = (size_t)256 << 20;
struct BwdPlan {
  int pieces, cols;  // cols: of every piece but the last
  gemm::Cut cut;     // of dx's contraction
  long long ldd;
  size_t scale, rows, dx, d, sum, total;
};
BwdPlan bwd_plan(long long n, int D, int V) {
  BwdPlan b;
  long long most = (long long)(kPieceBytes / 2) / n / gemm::kTileN * gemm::kTileN;
  if (most < gemm::kTileN) most = gemm::kTileN;
  b.pieces = gemm::blocks_of(V, (int)(most < V ? most : V));
  b.cols = gemm::blocks_of(gemm::blocks_of(V, b.pieces), gemm::kTileN) * gemm::kTileN;
  b.pieces = gemm::blocks_of(V, b.cols);
  b.ldd = b.pieces > 1 ? b.cols : (V + 63ll) / 64 * 64;
  const long long tiles_m = gemm::blocks_of(n, gemm::kTileM), tiles_n = gemm::blocks_of(D, gemm::kTileN);
  const long long kn = gemm::blocks_of(n, gemm::kBlockK);
  b.cut = {1, 0};
  if (b.pieces == 1)
    b.cut = gemm::cut_of(tiles_m * tiles_n, gemm::blocks_of(V, gemm::kBlockK),
                         gemm::blocks_of(V, gemm::kTileM) * tiles_n * gemm::length_of(kn), D);
  b.scale = kHead;
  b.rows = b.scale + up((size_t)n * sizeof(float));
  b.dx = b.rows + up((size_t)packed_rows((int)n) * pitch(D) * 2);
  b.d = b.dx + up((size_t)n * pitch(D) * 2);
  b.sum = b.d + up((size_t)n * b.ldd * 2);
  b.total = b.sum + (b.pieces > 1 ? (size_t)tiles_m * tiles_n * gemm::kTileM * gemm::kTileN * 4
                                  : gemm::cut_bytes(b.cut, tiles_m * tiles_n));
  return b;
}

struct Problem {
  const void *x, *w;
  long long ldx, ldw;
  int n, D, V;
  Plan plan;
  int reduction;
};

void shape(Op& op, long long M, long long N) {
  op.M = (int)M, op.N = (int)N;
  op.tiles_m = gemm::blocks_of(M, gemm::kTileM), op.tiles_n = gemm::blocks_of(N, gemm::kTileN);
}

template <typename T>
int forward(const Problem& q, const Labels& lab, float* loss, float2* lse, char* ws, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const FwdPlan f = fwd_plan(q.n, q.D, q.V);
  const int step = gemm::blocks_of(q.n, 592) < 8 ? 8 : gemm::blocks_of(q.n, 592);  // (a row a warp)
  plan_kernel<<<gemm::blocks_of(q.n, step), kPlanThreads, 0, stream>>>(lab, static_cast<const uint16_t*>(q.x), q.ldx, q.n, q.D, step,
                                                                      q.plan, reinterpret_cast<uint16_t*>(ws + f.rows), pitch(q.D),
                                                                      reinterpret_cast<int*>(ws));
  if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  Params p = {};
  p.ops = 1, p.err = reinterpret_cast<ErrorWord*>(ws), p.live = q.plan.live, p.labels = q.plan.label;
  p.part = reinterpret_cast<float2*>(ws + f.part);
  p.target = reinterpret_cast<float*>(ws + f.target);
  Op& o = p.op[0];
  shape(o, q.n, q.V);
  o.m_live = true;
  o.kb[0] = gemm::blocks_of(q.D, gemm::kBlockK);
  if (!gemm::operand_map(&o.a[0], ws + f.rows, dt, packed_rows(q.n), q.D, pitch(q.D), false) ||
      !gemm::operand_map(&o.b[0], q.w, dt, q.V, q.D, q.ldw, false))
    return GD_ERR_LAUNCH;
  if (const int st = gemm::launch<T, gemm::kLse>(p, stream)) return st;
  join_kernel<<<f.ctas, kJoinThreads, 0, stream>>>(p.part, p.target, f.parts, q.n, q.plan, q.reduction, lse, loss,
                                                     reinterpret_cast<float*>(ws + f.sums),
                                                     reinterpret_cast<unsigned int*>(ws + 64));
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T>
int backward(const Problem& q, const float2* lse, const float* dloss, void* dx, void* dw, char* ws, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const BwdPlan b = bwd_plan(q.n, q.D, q.V);
  const long long ld = pitch(q.D);
  void *const rows = ws + b.rows, *const dxc = ws + b.dx, *const d = ws + b.d;
  float* const row_scale = reinterpret_cast<float*>(ws + b.scale);
  float* const factor = reinterpret_cast<float*>(ws + 128);
  gather_kernel<<<grid_of(q.n), 256, 0, stream>>>(static_cast<const uint16_t*>(q.x), q.ldx, q.n, q.D, q.plan,
                                                  static_cast<uint16_t*>(rows), ld, reinterpret_cast<int*>(ws));
  if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  factors_kernel<<<1, 1024, 0, stream>>>(dloss, q.plan, q.n, q.reduction, std::is_same<T, __half>::value, row_scale, factor);
  if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const int kd = gemm::blocks_of(q.D, gemm::kBlockK);
  for (int i = 0; i < b.pieces; ++i) {
    const long long v0 = (long long)i * b.cols;
    const int cols = (int)(q.V - v0 < b.cols ? q.V - v0 : b.cols);
    const char* w = static_cast<const char*>(q.w) + v0 * q.ldw * 2;
    Params p = {};
    p.ops = 1, p.err = reinterpret_cast<ErrorWord*>(ws), p.live = q.plan.live, p.labels = q.plan.label;
    p.v0 = (int)v0, p.lse = lse, p.row_scale = row_scale;
    Op& o = p.op[0];
    shape(o, q.n, cols);
    o.m_live = true;
    o.kb[0] = kd;
    if (!gemm::operand_map(&o.a[0], rows, dt, packed_rows(q.n), q.D, ld, false) || !gemm::operand_map(&o.b[0], w, dt, cols, q.D, q.ldw, false) ||
        !gemm::slab_map(&o.c, d, dt, q.n, cols, b.ldd))
      return GD_ERR_LAUNCH;
    if (const int st = gemm::launch<T, gemm::kDLogit>(p, stream)) return st;
    Params r = {};
    r.err = p.err, r.live = q.plan.live;
    bool ok = true;
    if (dx != nullptr) {  // dx += D W
      Op& g = r.op[r.ops++];
      shape(g, q.n, q.D);
      g.m_live = true;
      g.kb[0] = gemm::blocks_of(cols, gemm::kBlockK);
      g.b_mn = true;
      g.slices = b.cut.slices, g.per = b.cut.per;
      g.sum_mode = b.cut.slices > 1 ? 1 : b.pieces == 1 ? 0 : i == 0 ? 1 : i + 1 < b.pieces ? 2 : 3;
      g.sum = reinterpret_cast<float*>(ws + b.sum);
      g.factor = factor;
      ok = ok && gemm::operand_map(&g.a[0], d, dt, q.n, cols, b.ldd, false) &&
           gemm::operand_map(&g.b[0], w, dt, cols, q.D, q.ldw, true) && gemm::slab_map(&g.c, dxc, dt, q.n, q.D, ld);
    }
    if (dw != nullptr) {  // dW = D^T x
      Op& g = r.op[r.ops++];
      shape(g, cols, q.D);
      g.k_live = true;
      g.kb[0] = gemm::blocks_of(q.n, gemm::kBlockK);
      g.a_mn = g.b_mn = true;
      g.factor = factor;
      ok = ok && gemm::operand_map(&g.a[0], d, dt, q.n, cols, b.ldd, true) &&
           gemm::operand_map(&g.b[0], rows, dt, packed_rows(q.n), q.D, ld, true) &&
           gemm::slab_map(&g.c, static_cast<char*>(dw) + v0 * q.D * 2, dt, cols, q.D, q.D);
    }
    if (!ok) return GD_ERR_LAUNCH;
    if (const int st = gemm::launch<T, gemm::kStore>(r, stream)) return st;
  }
  if (dx != nullptr) {
    if (b.cut.slices > 1) {
      Op g = {};
      shape(g, q.n, q.D);
      g.slices = b.cut.slices, g.factor = factor;
      if (const int st = gemm::sum_slices<T>(reinterpret_cast<const float*>(ws + b.sum), g, q.n, q.D, q.plan.live,
                                             q.plan.place, nullptr, nullptr, dx, stream))
        return st;
    } else {
      spread_kernel<<<grid_of(q.n), 256, 0, stream>>>(static_cast<const uint16_t*>(dxc), ld, q.n, q.D, q.plan.place,
                                                      static_cast<uint16_t*>(dx));
      if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
    }
  }
  return GD_OK;
}

int check(int dtype, int reduction, long long rows, int D, int V, long long ldx, long long ldw) {
  if ((dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) || reduction < kNone || reduction > kSum) return GD_ERR_ARG;
  if (rows < 0 || rows > (1ll << 24) || D <= 0 || D % 8 || D > (1 << 24) || V <= 0 || V > (1 << 24) || ldx < D || ldw < D ||
      ldx >= (1ll << 38) || ldw >= (1ll << 38) || !gemm::countable(rows, V) || !gemm::countable(rows, D) || !gemm::countable(V, D))
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
  return for_backward ? bwd_plan(rows, D, V).total : fwd_plan(rows, D, V).total;
}

extern "C" int gd_xent_fwd(const void* x, const void* w, const void* labels, int label64, float* loss, float* lse,
                           int* plan, int reduction, long long ignore, int dtype, long long rows, int D, int V, long long ldx,
                           long long ldw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gd::xent;
  if (const int st = check(dtype, reduction, rows, D, V, ldx, ldw)) return st;
  if (rows == 0) return GD_OK;
  if (x == nullptr || w == nullptr || labels == nullptr || loss == nullptr) return GD_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(lse) || !aligned16(workspace)) return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_xent_workspace_bytes(rows, D, V, 0)) return GD_ERR_WORKSPACE;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  int* const at = plan != nullptr ? plan : reinterpret_cast<int*>(ws + fwd_plan(rows, D, V).plan);
  const Problem q = {x, w, ldx, ldw, (int)rows, D, V, Plan::of(at, (int)rows), reduction};
  const Labels lab = {labels, label64, ignore, V};
  float2* const kept = reinterpret_cast<float2*>(lse);
  return dtype == GD_FLOAT16 ? forward<__half>(q, lab, loss, kept, ws, cs) : forward<__nv_bfloat16>(q, lab, loss, kept, ws, cs);
}

extern "C" int gd_xent_bwd(const void* x, const void* w, const float* lse, const int* plan, const float* dloss, void* dx, void* dw,
                           int reduction, int dtype, long long rows, int D, int V, long long ldx, long long ldw, void* workspace,
                           size_t workspace_bytes, void* stream) {
  using namespace gd::xent;
  if (const int st = check(dtype, reduction, rows, D, V, ldx, ldw)) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return dw == nullptr || cudaMemsetAsync(dw, 0, (size_t)V * D * 2, cs) == cudaSuccess ? GD_OK
                                                                                         : (cudaGetLastError(), GD_ERR_LAUNCH);
  if (x == nullptr || w == nullptr || lse == nullptr || plan == nullptr || dloss == nullptr) return GD_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(dx) || !aligned16(dw) || !aligned16(lse) || !aligned16(workspace))
    return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_xent_workspace_bytes(rows, D, V, 1)) return GD_ERR_WORKSPACE;
  if (dx == nullptr && dw == nullptr) return GD_OK;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const Problem q = {x, w, ldx, ldw, (int)rows, D, V, Plan::of(const_cast<int*>(plan), (int)rows), reduction};
  char* ws = static_cast<char*>(workspace);
  const float2* const kept = reinterpret_cast<const float2*>(lse);
  return dtype == GD_FLOAT16 ? backward<__half>(q, kept, dloss, dx, dw, ws, cs)
                             : backward<__nv_bfloat16>(q, kept, dloss, dx, dw, ws, cs);
}
