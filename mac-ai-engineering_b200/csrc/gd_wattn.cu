// The C entry points of the softmax attention (include/gated_delta_b200.h): argument checks, workspaces, launches.
#include <cmath>
#include <cstdint>

#include "gd_wattn.cuh"

namespace {

using gd::ErrorWord;
using gd::wattn::Problem;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// strides: every (batch, token, head) stride a multiple of 8 elements (TMA's 16 bytes) where the dimension has one
bool strides_ok(const long long* s, int B, int T, int heads) {
  auto ok = [](long long x, int n) { return n <= 1 || (x >= 0 && x % 8 == 0 && x < (1ll << 38)); };
  return ok(s[0], B) && ok(s[1], T) && ok(s[2], heads);
}

int check(const void* q, const void* k, const void* v, const long long* strides, const int* cu, int N, int dtype, int B,
          int Tq, int Tk, int H, int HK, int D, int window, int sinks, float scale) {
  if (dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) return GD_ERR_ARG;
  if (B < 0 || Tq < 0 || Tk < 0 || B > 65535 || Tq > (1 << 29) || Tk > (1 << 29) || H <= 0 || HK <= 0 || H > 65535 ||
      H % HK != 0 || D <= 0 || D % 8 != 0 || D > 256 || window < 0 || sinks < 0 || !std::isfinite(scale))
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
  p.cu = cu;
  p.N = N;
  return p;
}

}  // namespace

extern "C" size_t gd_wattn_workspace_bytes(int B, int Tq, int Tk, int H, int HK, int D, int for_backward) {
  if (B < 0 || Tq < 0 || Tk < 0 || H <= 0 || HK <= 0 || D <= 0 || D > 256) return 0;
  return sizeof(ErrorWord);
}

extern "C" int gd_wattn_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* cu_seqlens,
                            int N, int dtype, int B, int Tq, int Tk, int H, int HK, int D, const long long* strides,
                            int window, int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int st = check(q, k, v, strides, cu_seqlens, N, dtype, B, Tq, Tk, H, HK, D, window, sinks, scale)) return st;
  if (B == 0 || Tq == 0) return GD_OK;
  if (o == nullptr || lse == nullptr) return GD_ERR_ARG;
  if (!aligned16(o) || !aligned16(workspace)) return GD_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < sizeof(ErrorWord)) return GD_ERR_WORKSPACE;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (cudaMemsetAsync(workspace, 0, sizeof(ErrorWord), cs) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const Problem p = problem(cu_seqlens, N, B, Tq, Tk, H, HK, D, window, sinks, scale);
  if (Tk == 0) {  // no keys at all: zeros
    if (cudaMemsetAsync(o, 0, (size_t)B * Tq * H * D * 2, cs) != cudaSuccess ||
        cudaMemsetAsync(lse, 0x7f, (size_t)B * H * Tq * sizeof(float), cs) != cudaSuccess)  // 3.4e38: as good as +inf
      return (cudaGetLastError(), GD_ERR_LAUNCH);
    return GD_OK;
  }
  return gd::wattn::forward(q, k, v, strides, p, dtype, o, lse, static_cast<ErrorWord*>(workspace), cs);
}
