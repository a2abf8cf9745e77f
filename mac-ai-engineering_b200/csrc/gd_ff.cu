// The gated feed-forward block:  h = silu(x Wg^T) * (x Wu^T),  y = h Wd^T,  and its gradients.
#include <cstdint>

#include "gd_ff.cuh"
#include "gd_gemm.cuh"

namespace gd {
namespace ff {
namespace {

using gemm::Op;
using gemm::Params;

// max over dy's rows of the sum of absolute values, max |w_down|, as float bits (float16 only; both 8 columns at a time)
__global__ void __launch_bounds__(256) bounds_kernel(const __half* __restrict__ dy, long long ldy, int rows, int O,
                                                     const __half* __restrict__ wd, long long ldd, int F, uint32_t* bounds) {
  const int warps = gridDim.x * 8, w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  float top_sum = 0.f, top = 0.f;
  for (int r = w; r < rows + O; r += warps) {
    const bool is_dy = r < rows;
    const __half* p = is_dy ? dy + r * ldy : wd + (r - rows) * ldd;
    const int n = is_dy ? O : F;
    float sum = 0.f, m = 0.f;
#pragma unroll 4
    for (int c = lane * 8; c < n; c += 256) {
      float v[8];
      load8<__half>(p + c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum += fabsf(v[i]);
        m = wattn::max3(m, fabsf(v[i]), m);
      }
    }
    if (is_dy) top_sum = wattn::max3(top_sum, warp_sum(sum), top_sum);
    else top = wattn::max3(top, m, top);
  }
  __shared__ uint32_t sh[2][8];
  const uint32_t high = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (lane == 0) sh[0][threadIdx.x >> 5] = __float_as_uint(top_sum), sh[1][threadIdx.x >> 5] = high;
  __syncthreads();
  if (threadIdx.x < 2) {  // (one atomic a CTA and maximum)
    uint32_t m = 0;
    for (int i = 0; i < 8; ++i) m = max(m, sh[threadIdx.x][i]);
    atomicMax(bounds + threadIdx.x, m);
  }
}

void shape(Op& op, long long M, long long N, int tile_n = gemm::kTileN) {
  op.M = (int)M, op.N = (int)N;
  op.tiles_m = gemm::blocks_of(M, gemm::kTileM), op.tiles_n = gemm::blocks_of(N, tile_n);
  op.kb[1] = 0;
}

// Few tiles of y, or of dx beside the weights' gradients, have their contraction cut (gemm::cut_of; as if all gradients were asked
// for, so that each has the same bits whichever are). 129 rows, 4,096 x 12,288: a call takes 88 us, uncut 116.
gemm::Cut cut_y(long long n, int F, int O) {
  const long long tiles = (long long)gemm::blocks_of(n, gemm::kTileM) * gemm::blocks_of(O, gemm::kTileN);
  return gemm::cut_of(tiles, gemm::blocks_of(F, gemm::kBlockK), 0, O);
}
gemm::Cut cut_dx(long long n, int D, int F, int O) {
  auto tiles = [](long long M, long long N) {
    return (long long)gemm::blocks_of(M, gemm::kTileM) * gemm::blocks_of(N, gemm::kTileN);
  };
  return gemm::cut_of(tiles(n, D), 2ll * gemm::blocks_of(F, gemm::kBlockK),
                      (2 * tiles(F, D) + tiles(O, F)) * gemm::length_of(gemm::blocks_of(n, gemm::kBlockK)), D);
}
size_t sum_bytes(const gemm::Cut& c, long long n, int D) {
  return gemm::cut_bytes(c, (long long)gemm::blocks_of(n, gemm::kTileM) * gemm::blocks_of(D, gemm::kTileN));
}

template <typename T>
int forward(const Problem& q, void* const* kept, void* h, float* sum, void* y, uint32_t* bounds, ErrorWord* err, bool expire,
            cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const long long n = q.rows;
  Params p = {};
  p.ops = 1, p.err = err, p.keep = kept[0] != nullptr, p.bounds = bounds, p.expire = expire ? 85 : 0;
  Op& o = p.op[0];
  shape(o, n, q.F, gemm::kHalf);
  o.kb[0] = gemm::blocks_of(q.D, gemm::kBlockK);
  bool ok = gemm::operand_map(&o.a[0], q.x, dt, n, q.D, q.ldx, false) &&
            gemm::operand_map(&o.b[0], q.wg, dt, q.F, q.D, q.ldg, false) &&
            gemm::operand_map(&o.b[1], q.wu, dt, q.F, q.D, q.ldu, false) && gemm::strip_map(&o.c, h, dt, n, q.F, pitch(q.F));
  for (int i = 0; p.keep && i < 3; ++i) ok = ok && gemm::strip_map(&p.x[i], kept[i], dt, n, q.F, pitch(q.F));
  if (!ok) return GD_ERR_LAUNCH;
  if (const int st = gemm::launch<T, gemm::kSwiglu>(p, stream)) return st;
  Params r = {};
  r.ops = 1, r.err = err;
  Op& d = r.op[0];
  shape(d, n, q.O);
  d.kb[0] = gemm::blocks_of(q.F, gemm::kBlockK);
  if (!gemm::operand_map(&d.a[0], h, dt, n, q.F, pitch(q.F), false) ||
      !gemm::operand_map(&d.b[0], q.wd, dt, q.O, q.F, q.ldd, false) || !gemm::slab_map(&d.c, y, dt, n, q.O, q.O))
    return GD_ERR_LAUNCH;
  const gemm::Cut c = cut_y(n, q.F, q.O);
  d.slices = c.slices, d.per = c.per, d.sum_mode = c.slices > 1 ? 1 : 0, d.sum = sum;
  if (const int st = gemm::launch<T, gemm::kStore>(r, stream)) return st;
  return c.slices > 1 ? gemm::sum_slices<T>(sum, d, (int)n, q.O, nullptr, nullptr, nullptr, nullptr, y, stream) : GD_OK;
}

struct Grads {
  void *dx, *dwg, *dwu, *dwd;
};

template <typename T>
int backward(const Problem& q, const void* const* kept, const void* dy, long long ldy, const Grads& out, void* dg, void* du,
             void* h, float* sum, const uint32_t* bounds, uint32_t* own, ErrorWord* err, bool expire, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  const long long n = q.rows, lf = pitch(q.F);
  if (bounds != nullptr) {
    const int rows = q.rows + q.O;
    bounds_kernel<<<rows < 8 * 592 ? (rows + 7) / 8 : 592, 256, 0, stream>>>(
        static_cast<const __half*>(dy), ldy, q.rows, q.O, static_cast<const __half*>(q.wd), q.ldd, q.F, own);
    if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  }
  Params p = {};
  p.ops = 1, p.err = err, p.keep = out.dwd != nullptr, p.bounds = const_cast<uint32_t*>(bounds), p.more = own;
  p.expire = expire ? 86 : 0;
  Op& o = p.op[0];
  shape(o, n, q.F);  // dh = dy Wd
  o.kb[0] = gemm::blocks_of(q.O, gemm::kBlockK);
  o.b_mn = true;
  if (!gemm::operand_map(&o.a[0], dy, dt, n, q.O, ldy, false) || !gemm::operand_map(&o.b[0], q.wd, dt, q.O, q.F, q.ldd, true) ||
      !gemm::strip_map(&o.c, dg, dt, n, q.F, lf) || !gemm::strip_map(&p.y[0], du, dt, n, q.F, lf) ||
      (p.keep && !gemm::strip_map(&p.y[1], h, dt, n, q.F, lf)))
    return GD_ERR_LAUNCH;
  for (int i = 0; i < 3; ++i)
    if (!gemm::strip_map(&p.x[i], kept[i], dt, n, q.F, lf)) return GD_ERR_LAUNCH;
  if (const int st = gemm::launch<T, gemm::kDSwiglu>(p, stream)) return st;
  Params r = {};
  r.err = err, r.bounds = const_cast<uint32_t*>(bounds), r.more = own;
  bool ok = true;
  const int kn = gemm::blocks_of(n, gemm::kBlockK);
  auto weight = [&](void* dw, const void* a, long long lda, long long M, const void* b, long long ldb, long long N, bool scaled) {
    if (dw == nullptr) return;  // dW = a^T b, both with rows of tokens
    Op& w = r.op[r.ops++];
    shape(w, M, N);
    w.kb[0] = kn, w.a_mn = w.b_mn = true, w.unscale = scaled;
    ok = ok && gemm::operand_map(&w.a[0], a, dt, n, M, lda, true) && gemm::operand_map(&w.b[0], b, dt, n, N, ldb, true) &&
         gemm::slab_map(&w.c, dw, dt, M, N, N);
  };
  weight(out.dwg, dg, lf, q.F, q.x, q.ldx, q.D, true);
  weight(out.dwu, du, lf, q.F, q.x, q.ldx, q.D, true);
  weight(out.dwd, dy, ldy, q.O, h, lf, q.F, false);
  const gemm::Cut c = cut_dx(n, q.D, q.F, q.O);
  Op dx = {};
  if (out.dx != nullptr) {
    Op& w = r.op[r.ops++];
    shape(w, n, q.D);  // dx = dg Wg + du Wu
    w.kb[0] = w.kb[1] = gemm::blocks_of(q.F, gemm::kBlockK);
    w.b_mn = true, w.unscale = true;
    w.slices = c.slices, w.per = c.per, w.sum_mode = c.slices > 1 ? 1 : 0, w.sum = sum;
    dx = w;
    ok = ok && gemm::operand_map(&w.a[0], dg, dt, n, q.F, lf, false) && gemm::operand_map(&w.a[1], du, dt, n, q.F, lf, false) &&
         gemm::operand_map(&w.b[0], q.wg, dt, q.F, q.D, q.ldg, true) &&
         gemm::operand_map(&w.b[1], q.wu, dt, q.F, q.D, q.ldu, true) && gemm::slab_map(&w.c, out.dx, dt, n, q.D, q.D);
  }
  if (!ok) return GD_ERR_LAUNCH;
  if (const int st = gemm::launch<T, gemm::kStore>(r, stream)) return st;
  if (out.dx == nullptr || c.slices == 1) return GD_OK;
  return gemm::sum_slices<T>(sum, dx, (int)n, q.D, nullptr, nullptr, bounds, own, out.dx, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr size_t kHead = 256;  // the error word
size_t matrix_bytes(long long rows, int F) { return ((size_t)rows * pitch(F) * 2 + 255) / 256 * 256; }

int check(int dtype, long long rows, int D, int F, int O, const long long* ld, int n_ld) {
  if (dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) return GD_ERR_ARG;
  constexpr int kMost = 1 << 24;
  if (rows < 0 || rows > (1ll << 30) || D <= 0 || F <= 0 || O <= 0 || D % 8 || F % 8 || O % 8 || D > kMost || F > kMost ||
      O > kMost || !gemm::countable(rows, F) || !gemm::countable(rows, D) || !gemm::countable(rows, O) || !gemm::countable(F, D) ||
      !gemm::countable(F, O))
    return GD_ERR_SHAPE;
  if (ld == nullptr) return GD_ERR_ARG;
  const long long least[5] = {D, D, D, F, O};
  for (int i = 0; i < n_ld; ++i) {
    if (ld[i] < least[i]) return GD_ERR_SHAPE;
    if (ld[i] % 8) return GD_ERR_ALIGN;
    if (ld[i] >= (1ll << 38)) return GD_ERR_SHAPE;
  }
  return GD_OK;
}

// Tensor maps are encoded by the driver, which wants the device's context bound to the calling thread (autograd's has none
// until the runtime binds it).
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

}  // namespace
}  // namespace ff
}  // namespace gd

extern "C" size_t gd_ff_workspace_bytes(long long rows, int D, int F, int O, int for_backward) {
  const long long ld[5] = {D, D, D, F, O};
  if (gd::ff::check(GD_BFLOAT16, rows, D, F, O, ld, 5) != GD_OK || rows == 0) return 0;
  using namespace gd::ff;
  return kHead + (for_backward ? 3 * matrix_bytes(rows, F) + sum_bytes(cut_dx(rows, D, F, O), rows, D)
                               : matrix_bytes(rows, F) + sum_bytes(cut_y(rows, F, O), rows, O));
}

extern "C" int gd_ff_fwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, void* kept,
                         unsigned int* bounds, void* y, int dtype, long long rows, int D, int F, int O, const long long* ld,
                         void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gd::ff;
  const bool expire = dtype & GD_TEST_WAIT_EXPIRES;
  dtype &= ~GD_TEST_WAIT_EXPIRES;
  if (expire && kept == nullptr) return GD_ERR_ARG;
  if (const int st = check(dtype, rows, D, F, O, ld, 4)) return st;
  if (rows == 0) return GD_OK;
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr || y == nullptr ||
      (dtype == GD_FLOAT16 && (kept == nullptr) != (bounds == nullptr)))
    return GD_ERR_ARG;
  for (const void* t : {x, w_gate, w_up, w_down, (const void*)kept, (const void*)y, (const void*)workspace, (const void*)bounds})
    if (!aligned16(t)) return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_ff_workspace_bytes(rows, D, F, O, 0)) return GD_ERR_WORKSPACE;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  gd::ErrorWord* err = static_cast<gd::ErrorWord*>(workspace);
  const Problem q = {x, w_gate, w_up, w_down, ld[0], ld[1], ld[2], ld[3], (int)rows, D, F, O};
  void* h = static_cast<char*>(workspace) + kHead;
  if (kept == nullptr && rows <= kFew) return forward_few(q, dtype, h, y, cs);
  if (cudaMemsetAsync(err, 0, sizeof(*err), cs) != cudaSuccess ||
      (dtype == GD_FLOAT16 && bounds != nullptr && cudaMemsetAsync(bounds, 0, 16, cs) != cudaSuccess))
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  float* const sum = reinterpret_cast<float*>(static_cast<char*>(h) + matrix_bytes(rows, F));
  void* planes[3];
  for (int i = 0; i < 3; ++i) planes[i] = kept == nullptr ? nullptr : static_cast<char*>(kept) + i * (size_t)rows * pitch(F) * 2;
  return dtype == GD_FLOAT16 ? forward<__half>(q, planes, h, sum, y, bounds, err, expire, cs)
                             : forward<__nv_bfloat16>(q, planes, h, sum, y, nullptr, err, expire, cs);
}

extern "C" int gd_ff_bwd(const void* x, const void* w_gate, const void* w_up, const void* w_down, const void* kept,
                         const unsigned int* bounds, const void* dy, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                         int dtype, long long rows, int D, int F, int O, const long long* ld, void* workspace,
                         size_t workspace_bytes, void* stream) {
  using namespace gd::ff;
  const bool expire = dtype & GD_TEST_WAIT_EXPIRES;
  dtype &= ~GD_TEST_WAIT_EXPIRES;
  if (const int st = check(dtype, rows, D, F, O, ld, 5)) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t wide = (size_t)F * D * 2;
    if ((dw_gate != nullptr && cudaMemsetAsync(dw_gate, 0, wide, cs) != cudaSuccess) ||
        (dw_up != nullptr && cudaMemsetAsync(dw_up, 0, wide, cs) != cudaSuccess) ||
        (dw_down != nullptr && cudaMemsetAsync(dw_down, 0, (size_t)O * F * 2, cs) != cudaSuccess))
      return (cudaGetLastError(), GD_ERR_LAUNCH);
    return GD_OK;
  }
  if (x == nullptr || w_gate == nullptr || w_up == nullptr || w_down == nullptr || kept == nullptr || dy == nullptr ||
      (dtype == GD_FLOAT16 && bounds == nullptr))
    return GD_ERR_ARG;
  for (const void* t : {x, w_gate, w_up, w_down, kept, dy, (const void*)dx, (const void*)dw_gate, (const void*)dw_up,
                        (const void*)dw_down, (const void*)workspace, (const void*)bounds})
    if (!aligned16(t)) return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < gd_ff_workspace_bytes(rows, D, F, O, 1)) return GD_ERR_WORKSPACE;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  gd::ErrorWord* err = static_cast<gd::ErrorWord*>(workspace);
  char* const at = static_cast<char*>(workspace);
  if (cudaMemsetAsync(workspace, 0, kHead, cs) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  uint32_t* const own = reinterpret_cast<uint32_t*>(at + 128);  // float16's two maxima of this call
  const Problem q = {x, w_gate, w_up, w_down, ld[0], ld[1], ld[2], ld[3], (int)rows, D, F, O};
  const Grads out = {dx, dw_gate, dw_up, dw_down};
  const size_t m = matrix_bytes(rows, F);
  void *dg = at + kHead, *du = at + kHead + m, *h = at + kHead + 2 * m;
  float* const sum = reinterpret_cast<float*>(at + kHead + 3 * m);
  const void* planes[3];
  for (int i = 0; i < 3; ++i) planes[i] = static_cast<const char*>(kept) + i * (size_t)rows * pitch(F) * 2;
  return dtype == GD_FLOAT16
             ? backward<__half>(q, planes, dy, ld[4], out, dg, du, h, sum, bounds, own, err, expire, cs)
             : backward<__nv_bfloat16>(q, planes, dy, ld[4], out, dg, du, h, sum, nullptr, nullptr, err, expire, cs);
}
