// Rotary positions of the queries and keys of a softmax-attention layer, both in one pass. The first R channels of a
// head are pairs turned by the token's angles, the others pass through:
//   a' = a cos - b sin,  b' = b cos + a sin       (fp32, one rounding)
// with pairs (i, i + R/2) (half layout) or (2 i, 2 i + 1) (interleaved), cos and sin from a table [P, R/2, 2] in fp32
// indexed by the token's position. The backward is the turn by the opposite angle (sign = -1).
//
// Bound by HBM: every channel of q and k is read and written once; a token's R/2 angles serve all its heads (they come
// from L1 and L2 after the first). q and k may be views of a fused projection (any batch, token and head stride);
// outputs are contiguous. A unit of work is V channels of a head that pass through or are turned among themselves
// (interleaved), or the two V-channel halves of V pairs; V is the widest that divides widths, strides and addresses.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gated_delta_b200.h"

namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;  // units a thread has in flight

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

struct Rows {  // element strides of one input [B, T, heads, D]
  long long b, t, h;
};
struct Args {
  Rows q, k;
  const float2* table;
  const void* positions;  // NULL: the token's index
  long long pos_b;        // positions' batch stride (0: one list for all rows)
  int pos64;
  long long P;
  int B, T, H, HK, D, R;
  float sign;
};

template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                          T* __restrict__ oq, T* __restrict__ ok, const Args a,
                                                          const int turn_units, const int units, long long items) {
  constexpr int N = IL && V == 1 ? 2 : V;  // channels of a unit (of each half of its pairs in the half layout)
  using Pk = Pack<T, V>;
  const long long first = (long long)blockIdx.x * (kThreads * kItems) + threadIdx.x;
  const int heads = a.H + a.HK;
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    const long long item = first + it * kThreads;
    if (item >= items) return;
    // item -> (token, head, unit); 32-bit divisions inside the token
    const int per_token = heads * units;
    const long long token = item < 0x7fffffff ? (long long)((unsigned)item / (unsigned)per_token) : item / per_token;
    const unsigned rest = (unsigned)(item - token * per_token);
    const int hh = rest / units, u = rest - hh * units;
    const int b = token < 0x7fffffff ? (int)((unsigned)token / (unsigned)a.T) : (int)(token / a.T);
    const int t = (int)(token - (long long)b * a.T);
    const bool is_q = hh < a.H;
    const int h = is_q ? hh : hh - a.H;
    const T* src = is_q ? q + b * a.q.b + t * a.q.t + h * a.q.h : k + b * a.k.b + t * a.k.t + h * a.k.h;
    T* dst = is_q ? oq + (token * a.H + h) * a.D : ok + (token * a.HK + h) * a.D;
    if (u >= turn_units) {  // channels past R
      const int c = a.R + (u - turn_units) * V;
      *reinterpret_cast<Pk*>(dst + c) = *reinterpret_cast<const Pk*>(src + c);
      continue;
    }
    long long p = t;
    if (a.positions != nullptr) {
      const long long at = b * a.pos_b + t;
      p = a.pos64 ? __ldg(static_cast<const long long*>(a.positions) + at)
                  : (long long)__ldg(static_cast<const int*>(a.positions) + at);
    }
    p = p < 0 ? 0 : p >= a.P ? a.P - 1 : p;  // never outside the table
    const float2* tab = a.table + p * (a.R / 2);
    if constexpr (IL) {
      const int c = u * N;
      T x[N];
#pragma unroll
      for (int i = 0; i < N / V; ++i) {
        const Pk pk = *reinterpret_cast<const Pk*>(src + c + i * V);
#pragma unroll
        for (int e = 0; e < V; ++e) x[i * V + e] = pk.v[e];
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 cs = __ldg(tab + c / 2 + i);
        const float sn = cs.y * a.sign, f = to_f<T>(x[2 * i]), g = to_f<T>(x[2 * i + 1]);
        x[2 * i] = from_f<T>(f * cs.x - g * sn);
        x[2 * i + 1] = from_f<T>(g * cs.x + f * sn);
      }
#pragma unroll
      for (int i = 0; i < N / V; ++i) {
        Pk pk;
#pragma unroll
        for (int e = 0; e < V; ++e) pk.v[e] = x[i * V + e];
        *reinterpret_cast<Pk*>(dst + c + i * V) = pk;
      }
    } else {
      const int c = u * V;
      Pk x = *reinterpret_cast<const Pk*>(src + c), y = *reinterpret_cast<const Pk*>(src + c + a.R / 2);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = __ldg(tab + c + e);
        const float sn = cs.y * a.sign, f = to_f<T>(x.v[e]), g = to_f<T>(y.v[e]);
        x.v[e] = from_f<T>(f * cs.x - g * sn);
        y.v[e] = from_f<T>(g * cs.x + f * sn);
      }
      *reinterpret_cast<Pk*>(dst + c) = x;
      *reinterpret_cast<Pk*>(dst + c + a.R / 2) = y;
    }
  }
}

template <typename T, int V, bool IL>
int launch(const void* q, const void* k, void* oq, void* ok, const Args& a, cudaStream_t stream) {
  const int turn = IL ? a.R / (V == 1 ? 2 : V) : a.R / 2 / V;
  const int units = turn + (a.D - a.R) / V;
  const long long items = (long long)a.B * a.T * (a.H + a.HK) * units;
  const long long grid = (items + kThreads * kItems - 1) / (kThreads * kItems);
  if (grid > 0x7fffffffll) return GD_ERR_SHAPE;
  rotary_kernel<T, V, IL><<<(unsigned)grid, kThreads, 0, stream>>>(static_cast<const T*>(q), static_cast<const T*>(k),
                                                                  static_cast<T*>(oq), static_cast<T*>(ok), a, turn,
                                                                  units, items);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, bool IL>
int by_width(int v, const void* q, const void* k, void* oq, void* ok, const Args& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  if (v >= E) return launch<T, E, IL>(q, k, oq, ok, a, s);
  if (E == 8 && v == 4) return launch<T, 4, IL>(q, k, oq, ok, a, s);
  if (v == 2) return launch<T, 2, IL>(q, k, oq, ok, a, s);
  return launch<T, 1, IL>(q, k, oq, ok, a, s);
}
template <typename T>
int by_layout(int il, int v, const void* q, const void* k, void* oq, void* ok, const Args& a, cudaStream_t s) {
  return il ? by_width<T, true>(v, q, k, oq, ok, a, s) : by_width<T, false>(v, q, k, oq, ok, a, s);
}

}  // namespace

extern "C" int gd_rotary(const void* q, const void* k, void* oq, void* ok, const float* table, const void* positions,
                         int positions64, long long pos_stride_b, long long table_rows, int dtype, int B, int T, int H,
                         int HK, int D, int R, long long q_stride_b, long long q_stride_t, long long q_stride_h,
                         long long k_stride_b, long long k_stride_t, long long k_stride_h, int interleaved, int inverse,
                         void* stream) {
  if (dtype != GD_FLOAT32 && dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) return GD_ERR_ARG;
  if (B < 0 || T < 0 || H < 0 || HK < 0 || D <= 0 || R <= 0 || R % 2 != 0 || R > D || table_rows < 0) return GD_ERR_SHAPE;
  if ((long long)B * T == 0 || H + HK == 0) return GD_OK;
  if (table_rows == 0 || (long long)(H + HK) * D > 0x3fffffff) return GD_ERR_SHAPE;
  if (table == nullptr || (H > 0 && (q == nullptr || oq == nullptr)) || (HK > 0 && (k == nullptr || ok == nullptr)))
    return GD_ERR_ARG;
  const int size = dtype == GD_FLOAT32 ? 4 : 2;
  // the widest V that divides every width, stride and address
  unsigned long long all = 16 / size | (unsigned)D | (unsigned)(interleaved ? R : R / 2) | (unsigned)(D - R);
  auto add = [&](const void* in, const void* out, long long sb, long long st, long long sh, bool bb, bool tt, bool hh) {
    all |= (reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) / size;
    if (bb) all |= (unsigned long long)sb;
    if (tt) all |= (unsigned long long)st;
    if (hh) all |= (unsigned long long)sh;
  };
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(oq) |
        reinterpret_cast<uintptr_t>(ok)) % size) != 0 || reinterpret_cast<uintptr_t>(table) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(positions) % (positions64 ? 8 : 4) != 0)
    return GD_ERR_ALIGN;
  if (H > 0) add(q, oq, q_stride_b, q_stride_t, q_stride_h, B > 1, T > 1, H > 1);
  if (HK > 0) add(k, ok, k_stride_b, k_stride_t, k_stride_h, B > 1, T > 1, HK > 1);
  const int v = (int)(all & (~all + 1));
  Args a;
  a.q = {q_stride_b, q_stride_t, q_stride_h};
  a.k = {k_stride_b, k_stride_t, k_stride_h};
  a.table = reinterpret_cast<const float2*>(table);
  a.positions = positions;
  a.pos_b = pos_stride_b;
  a.pos64 = positions64;
  a.P = table_rows;
  a.B = B, a.T = T, a.H = H, a.HK = HK, a.D = D, a.R = R;
  a.sign = inverse ? -1.f : 1.f;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GD_FLOAT32) return by_layout<float>(interleaved, v, q, k, oq, ok, a, s);
  if (dtype == GD_FLOAT16) return by_layout<__half>(interleaved, v, q, k, oq, ok, a, s);
  return by_layout<__nv_bfloat16>(interleaved, v, q, k, oq, ok, a, s);
}
