// The C entry points of the softmax attention (include/gated_delta_b200.h): argument checks, workspaces, launches.
#include <cmath>
#include <cstdint>

#include "gd_wattn.cuh"

namespace {

using gd::ErrorWord;
using gd::wattn::Problem;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// strides: every (batch, token, head) stride a positive multiple of 8 elements (TMA's 16 bytes) where the dimension has one
bool strides_ok(const long long* s, int B, int T, int heads) {
  auto ok = [](long long x, int n) { return n <= 1 || (x > 0 && x % 8 == 0 && x < (1ll << 38)); };
  return ok(s[0], B) && ok(s[1], T) && ok(s[2], heads);
}

// Tensor maps are encoded by the driver, which wants the device's context bound to the calling thread; a thread whose first
// call this is (autograd's) has none until the runtime binds it.
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

int check(const void* q, const void* k, const void* v, const long long* strides, const int* cu, int N, int dtype, int B,
          int Tq, int Tk, int H, int HK, int D, int window, int sinks, float scale) {
  if (dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) return GD_ERR_ARG;
  if (B < 0 || Tq < 0 || Tk < 0 || B > 65535 || Tq > (1 << 29) || Tk > (1 << 29) || H <= 0 || HK <= 0 || H > 65535 ||
      H % HK != 0 || (long long)Tq * H >= (1ll << 31) || D <= 0 || D % 8 != 0 || D > 256 || window < 0 || sinks < 0 ||
      !std::isfinite(scale))
    return GD_ERR_SHAPE;
  if (cu != nullptr && (B != 1 || Tq != Tk || N <= 0 || N > (1 << 24))) return GD_ERR_SHAPE;
  if (B == 0 || Tq == 0) return GD_OK;
  if (strides == nullptr || q == nullptr || (Tk > 0 && (k == nullptr || v == nullptr))) return GD_ERR_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return GD_ERR_ALIGN;
  if (!strides_ok(strides, B, Tq, H) || !strides_ok(strides + 3, B, Tk, HK) || !strides_ok(strides + 6, B, Tk, HK))
    return GD_ERR_ALIGN;
  return GD_OK;
}

Problem problem(const int* cu, int N, int B, int Tq, int Tk, int H, int HK, int D, int window, int sinks, float scale) {
  Problem p;
  p.B = B, p.Tq = Tq, p.Tk = Tk, p.H = H, p.HK = HK, p.D = D;
  p.window = window == 0 || window > gd::wattn::kNoWindow ? gd::wattn::kNoWindow : window;
  p.sinks = sinks < Tk ? sinks : Tk;
  p.scale = scale;
  p.scale_log2 = scale * gd::wattn::kLog2e;
  p.negate = false;
  p.cu = cu;
  p.N = N;
  return p;
}

// The backward's workspace: the error word, delta [B, H, Tq], the partial tiles of the key tiles that are cut.
size_t delta_at() { return 256; }
size_t delta_bytes(int B, int Tq, int H) { return ((size_t)B * H * Tq * sizeof(float) + 255) / 256 * 256; }

// Key tiles that more queries see than a fair share of the GPU's work (all of the later queries: the first tokens that
// stay visible, or a row without a window) are cut: the first `heavy` tiles into `parts` CTAs each, so that no CTA has
// much more than the average of an SM. Work is counted in (query tile, head) steps. At 1 x 8192 x 16 (4 key heads), D 128,
// window 2048, 16 first tokens, the first key tile alone would be 256 steps where the others are 68 and an SM's share is 108:
// it is cut in three, and the kernel takes 297 us with 3 us for the sum.
struct Cut {
  int heavy, parts;
};
Cut cut_of(int B, int Tq, int Tk, int H, int HK, int D, int window, int sinks) {
  using gd::wattn::kTile;
  const long long off = (long long)Tk - Tq, G = H / HK, tiles = (Tk + kTile - 1) / kTile;
  const long long lanes = (long long)B * HK * (D > 128 ? 2 : 1);
  auto steps = [&](long long t) {  // of key tile t
    const long long c0 = t * kTile, from = c0 - off > 0 ? c0 - off : 0;
    long long last = Tq - 1;
    if (c0 >= sinks && c0 + kTile - 1 + window - 1 - off < last) last = c0 + kTile - 1 + window - 1 - off;
    return last >= from ? G * (last / kTile - from / kTile + 1) : 0;
  };
  long long total = 0, top = 0;
  for (long long t = 0; t < tiles; ++t) {
    const long long s = steps(t);
    total += s;
    if (s > top) top = s;
  }
  const long long fair = (total * lanes + 147) / 148;
  if (tiles == 0 || top <= fair + fair / 4 || top < 8) return {0, 1};
  long long heavy = 0;
  while (heavy < tiles && steps(heavy) > fair) ++heavy;
  long long parts = (steps(0) + fair - 1) / (fair > 0 ? fair : 1);
  if (parts > 16) parts = 16;
  if (heavy == 0 || parts < 2) return {0, 1};
  return {(int)heavy, (int)parts};
}
size_t part_bytes(const Cut& c, int B, int HK, int D) {
  return c.parts > 1 ? (size_t)B * HK * c.heavy * c.parts * 2 * gd::wattn::kTile * D * sizeof(float) : 0;
}

}  // namespace

extern "C" size_t gd_wattn_workspace_bytes(int B, int Tq, int Tk, int H, int HK, int D, int window, int sinks, int packed,
                                           int for_backward) {
  if (B < 0 || Tq < 0 || Tk < 0 || H <= 0 || HK <= 0 || H % HK != 0 || D <= 0 || D > 256 || window < 0 || sinks < 0)
    return 0;
  if (!for_backward) return sizeof(ErrorWord);
  const Problem p = problem(nullptr, 0, B, Tq, Tk, H, HK, D, window, sinks, 1.f);
  const Cut c = packed ? Cut{0, 1} : cut_of(B, Tq, Tk, H, HK, D, p.window, p.sinks);
  return delta_at() + delta_bytes(B, Tq, H) + part_bytes(c, B, HK, D);
}

extern "C" int gd_wattn_fwd(const void* q, const void* k, const void* v, void* o, void* o_low, float* lse,
                            const int* cu_seqlens, int N, int dtype, int B, int Tq, int Tk, int H, int HK, int D,
                            const long long* strides, int window, int sinks, float scale, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int st = check(q, k, v, strides, cu_seqlens, N, dtype, B, Tq, Tk, H, HK, D, window, sinks, scale)) return st;
  if (B == 0 || Tq == 0) return GD_OK;
  if (o == nullptr || (lse == nullptr && o_low != nullptr)) return GD_ERR_ARG;
  if (!aligned16(o) || !aligned16(o_low) || !aligned16(workspace)) return GD_ERR_ALIGN;
  if (workspace != nullptr && workspace_bytes < sizeof(ErrorWord)) return GD_ERR_WORKSPACE;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  if (workspace != nullptr && cudaMemsetAsync(workspace, 0, sizeof(ErrorWord), cs) != cudaSuccess)
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  Problem p = problem(cu_seqlens, N, B, Tq, Tk, H, HK, D, window, sinks, scale);
  // a scale of 0 as a tiny one: finite scores vanish beside 1, and a masked one stays -inf
  p.scale_log2 = scale == 0.f ? 1e-30f : std::fabs(p.scale_log2);
  p.negate = scale < 0.f;
  if (Tk == 0) {  // no keys at all: zeros
    const size_t n = (size_t)B * Tq * H * D * 2;
    if (cudaMemsetAsync(o, 0, n, cs) != cudaSuccess ||
        (o_low != nullptr && cudaMemsetAsync(o_low, 0, n, cs) != cudaSuccess) ||
        // 3.4e38: as good as +inf
        (lse != nullptr && cudaMemsetAsync(lse, 0x7f, (size_t)B * H * Tq * sizeof(float), cs) != cudaSuccess))
      return (cudaGetLastError(), GD_ERR_LAUNCH);
    return GD_OK;
  }
  return gd::wattn::forward(q, k, v, strides, p, dtype, o, o_low, lse, static_cast<ErrorWord*>(workspace), cs);
}

extern "C" int gd_wattn_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_low,
                            const float* lse, const void* d_o, void* dq, void* dk, void* dv, const int* cu_seqlens,
                            int N, int dtype, int B, int Tq, int Tk, int H, int HK, int D, const long long* strides,
                            int window, int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int st = check(q, k, v, strides, cu_seqlens, N, dtype, B, Tq, Tk, H, HK, D, window, sinks, scale)) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (B == 0 || Tq == 0 || Tk == 0) {  // no pair: zero gradients
    const size_t nq = (size_t)B * Tq * H * D * 2, nk = (size_t)B * Tk * HK * D * 2;
    if ((nq > 0 && dq == nullptr) || (nk > 0 && (dk == nullptr || dv == nullptr))) return GD_ERR_ARG;
    if ((nq > 0 && cudaMemsetAsync(dq, 0, nq, cs) != cudaSuccess) ||
        (nk > 0 && cudaMemsetAsync(dk, 0, nk, cs) != cudaSuccess) ||
        (nk > 0 && cudaMemsetAsync(dv, 0, nk, cs) != cudaSuccess))
      return (cudaGetLastError(), GD_ERR_LAUNCH);
    return GD_OK;
  }
  if (o == nullptr || o_low == nullptr || lse == nullptr || d_o == nullptr || dq == nullptr || dk == nullptr ||
      dv == nullptr)
    return GD_ERR_ARG;
  if (!aligned16(o) || !aligned16(o_low) || !aligned16(d_o) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      !aligned16(workspace))
    return GD_ERR_ALIGN;
  if (!strides_ok(strides + 9, B, Tq, H)) return GD_ERR_ALIGN;
  if (workspace == nullptr ||
      workspace_bytes < gd_wattn_workspace_bytes(B, Tq, Tk, H, HK, D, window, sinks, cu_seqlens != nullptr, 1))
    return GD_ERR_WORKSPACE;
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  // the error word, with float16's largest norms in it; bfloat16's first kernel clears it
  if (dtype == GD_FLOAT16 && cudaMemsetAsync(workspace, 0, sizeof(ErrorWord), cs) != cudaSuccess)
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  const Problem p = problem(cu_seqlens, N, B, Tq, Tk, H, HK, D, window, sinks, scale);
  // packed rows are not cut: where their sequences end, and so which tiles are heavy, is known on the device only
  const Cut c = cu_seqlens != nullptr ? Cut{0, 1} : cut_of(B, Tq, Tk, H, HK, D, p.window, p.sinks);
  char* ws = static_cast<char*>(workspace);
  return gd::wattn::backward(q, k, v, o, o_low, d_o, strides, p, dtype, lse, reinterpret_cast<float*>(ws + delta_at()),
                             dq, dk, dv, c.heavy, c.parts,
                             reinterpret_cast<float*>(ws + delta_at() + delta_bytes(B, Tq, H)),
                             static_cast<ErrorWord*>(workspace), cs);
}
