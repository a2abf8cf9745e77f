// Rotary positions of the queries and keys of a softmax-attention layer, both in one pass. The first R channels of a
// head are pairs turned by the token's angles, the others pass through:
//   a' = a cos - b sin,  b' = b cos + a sin       (fp32, one rounding)
// with pairs (i, i + R/2) (half layout) or (2 i, 2 i + 1) (interleaved), cos and sin from a table [P, R/2, 2] in fp32
// indexed by the token's position. The backward is the turn by the opposite angle (sign = -1).
//
// Bound by HBM: every channel of q and k is read and written once; a token's R/2 angles serve all its heads (through shared memory). q and k may be views of a fused projection (any batch, token and head stride);
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
constexpr int kItems = 2;  // units a thread has in flight: with 48 warps an SM, enough; more registers cost more warps

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
  bool table16;           // every row of the table starts on 16 bytes
};

// n / d for n < 2^16 and d <= 2^16, by m = ceil(2^32 / d): n m is off n 2^32 / d by less than n d <= 2^32
__device__ __forceinline__ unsigned div16(unsigned n, unsigned m) { return m == 0u ? n : __umulhi(n, m); }

// How a CTA's items are numbered: first the turned units of its tokens, (token, head, unit), then the copied ones, so that
// a warp does one or the other.
struct Items {
  int tokens;                       // of a CTA
  int turn, copy;                   // units of a head
  unsigned m_turn, m_copy;          // div16's numbers: of turn, copy
  unsigned m_hturn, m_hcopy;        // of heads * turn, heads * copy
};

// A CTA takes `tokens` consecutive tokens of a batch row. A thread's items lie kThreads apart; their loads are in flight
// before any arithmetic.
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                             T* __restrict__ oq, T* __restrict__ ok, const Args a,
                                                             const Items n) {
  constexpr int N = IL && V == 1 ? 2 : V;  // channels of a turned unit (of each half of its pairs in the half layout)
  constexpr int L = N / V;                 // packs of it
  constexpr int A = IL ? N / 2 : V;        // angles of it
  using Pk = Pack<T, V>;
  const unsigned heads = a.H + a.HK;
  const int b = blockIdx.y, t0 = blockIdx.x * n.tokens, here = a.T - t0 < n.tokens ? a.T - t0 : n.tokens;
  const unsigned turned = (unsigned)here * heads * n.turn, items = turned + (unsigned)here * heads * n.copy;
  const bool small = items <= 65536u;  // (a CTA of one token may have more: it divides)
  for (unsigned first = threadIdx.x; first < items; first += kThreads * kItems) {
    Pk x[kItems][L], y[kItems];
    T* dst[kItems];
    const float2* cs[kItems];  // a turned item's angles
    bool live[kItems];
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
      unsigned i = first + it * kThreads;
      live[it] = i < items;
      cs[it] = nullptr;
      if (!live[it]) continue;
      const bool turn = i < turned;
      if (!turn) i -= turned;
      const unsigned units = turn ? n.turn : n.copy, per_token = heads * units;
      const unsigned tt = small ? div16(i, turn ? n.m_hturn : n.m_hcopy) : i / per_token, rest = i - tt * per_token;
      const unsigned hh = small ? div16(rest, turn ? n.m_turn : n.m_copy) : rest / units, u = rest - hh * units;
      const int t = t0 + (int)tt;
      const bool is_q = hh < (unsigned)a.H;
      const long long h = is_q ? hh : hh - a.H, token = (long long)b * a.T + t;
      const int c = turn ? (int)u * N : a.R + (int)u * V;
      const T* src = (is_q ? q + b * a.q.b + t * a.q.t + h * a.q.h : k + b * a.k.b + t * a.k.t + h * a.k.h) + c;
      dst[it] = (is_q ? oq + (token * a.H + h) * a.D : ok + (token * a.HK + h) * a.D) + c;
      x[it][0] = *reinterpret_cast<const Pk*>(src);
      if (turn) {
#pragma unroll
        for (int l = 1; l < L; ++l) x[it][l] = *reinterpret_cast<const Pk*>(src + l * V);
        if (!IL) y[it] = *reinterpret_cast<const Pk*>(src + a.R / 2);
        long long p = t;
        if (a.positions != nullptr) {
          const long long w = b * a.pos_b + t;
          p = a.pos64 ? __ldg(static_cast<const long long*>(a.positions) + w)
                      : (long long)__ldg(static_cast<const int*>(a.positions) + w);
        }
        p = p < 0 ? 0 : p >= a.P ? a.P - 1 : p;  // never outside the table
        cs[it] = a.table + p * (a.R / 2) + (IL ? c / 2 : c);
      }
    }
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
      if (!live[it]) continue;
      if (cs[it] != nullptr) {
        float2 t[A];
        if constexpr (A % 2 == 0) {  // an even number of angles starts on 16 bytes when the table does
          if (a.table16) {
#pragma unroll
            for (int i = 0; i < A; i += 2) {
              const float4 v = __ldg(reinterpret_cast<const float4*>(cs[it] + i));
              t[i] = make_float2(v.x, v.y);
              t[i + 1] = make_float2(v.z, v.w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < A; ++i) t[i] = __ldg(cs[it] + i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < A; ++i) t[i] = __ldg(cs[it] + i);
        }
        if constexpr (IL) {
          T* v = reinterpret_cast<T*>(x[it]);
#pragma unroll
          for (int i = 0; i < A; ++i) {
            const float f = to_f<T>(v[2 * i]), g = to_f<T>(v[2 * i + 1]), sn = t[i].y * a.sign;
            v[2 * i] = from_f<T>(f * t[i].x - g * sn);
            v[2 * i + 1] = from_f<T>(g * t[i].x + f * sn);
          }
#pragma unroll
          for (int l = 1; l < L; ++l) *reinterpret_cast<Pk*>(dst[it] + l * V) = x[it][l];
        } else {
#pragma unroll
          for (int e = 0; e < A; ++e) {
            const float f = to_f<T>(x[it][0].v[e]), g = to_f<T>(y[it].v[e]), sn = t[e].y * a.sign;
            x[it][0].v[e] = from_f<T>(f * t[e].x - g * sn);
            y[it].v[e] = from_f<T>(g * t[e].x + f * sn);
          }
          *reinterpret_cast<Pk*>(dst[it] + a.R / 2) = y[it];
        }
      }
      *reinterpret_cast<Pk*>(dst[it]) = x[it][0];
    }
  }
}

unsigned magic(unsigned d) { return d <= 1 ? 0u : (unsigned)(((1ull << 32) + d - 1) / d); }

template <typename T, int V, bool IL>
int launch(const void* q, const void* k, void* oq, void* ok, const Args& a, cudaStream_t stream) {
  Items n;
  n.turn = IL ? a.R / (V == 1 ? 2 : V) : a.R / 2 / V;
  n.copy = (a.D - a.R) / V;
  const unsigned heads = (unsigned)(a.H + a.HK), per_token = heads * (unsigned)(n.turn + n.copy);
  // as many tokens as give each thread twice kItems units; one where a token has more, or where that leaves SMs idle
  int tokens = (int)(kThreads * 2 * kItems / per_token);
  while (tokens > 1 && (long long)a.B * ((a.T + tokens - 1) / tokens) < 148) tokens /= 2;
  if (tokens < 1) tokens = 1;
  n.tokens = tokens;
  n.m_turn = magic(n.turn), n.m_copy = magic(n.copy);
  n.m_hturn = magic(heads * n.turn), n.m_hcopy = magic(heads * n.copy);
  rotary_kernel<T, V, IL>
      <<<dim3((unsigned)((a.T + tokens - 1) / tokens), (unsigned)a.B), kThreads, 0, stream>>>(
          static_cast<const T*>(q), static_cast<const T*>(k), static_cast<T*>(oq), static_cast<T*>(ok), a, n);
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
  if (B < 0 || B > 65535 || T < 0 || H < 0 || HK < 0 || D <= 0 || R <= 0 || R % 2 != 0 || R > D || table_rows < 0) return GD_ERR_SHAPE;
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
  a.table16 = reinterpret_cast<uintptr_t>(table) % 16 == 0 && R % 4 == 0;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == GD_FLOAT32) return by_layout<float>(interleaved, v, q, k, oq, ok, a, s);
  if (dtype == GD_FLOAT16) return by_layout<__half>(interleaved, v, q, k, oq, ok, a, s);
  return by_layout<__nv_bfloat16>(interleaved, v, q, k, oq, ok, a, s);
}
