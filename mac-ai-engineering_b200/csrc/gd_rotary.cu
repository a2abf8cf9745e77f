// Rotary positions of the queries and keys of a softmax-attention layer, both in one pass. The first R channels of a
// head are pairs turned by the token's angles, the others pass through:
//   a' = a cos - b sin,  b' = b cos + a sin       (fp32, one rounding)
// with pairs (i, i + R/2) (half layout) or (2 i, 2 i + 1) (interleaved), cos and sin from a table [P, R/2, 2] in fp32
// indexed by the token's position. The backward is the turn by the opposite angle (sign = -1).
//
// Bound by HBM: every channel of q and k is read and written once; a token's R/2 angles serve all its heads (they come
// from L1 and L2 after the first). q and k may be views of a fused projection (any batch, token and head stride); outputs
// are contiguous. A unit of work is V channels of a head that pass through or are turned among themselves (interleaved),
// or the two V-channel halves of V pairs; V is the widest that divides widths, strides and addresses.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gated_delta_b200.h"

namespace {

constexpr int kMaxThreads = 512;
constexpr int kTokens = 4;  // of a CTA

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

// A thread has one unit of one head (the turned units first, so that a warp turns or copies) and walks the CTA's tokens:
// the address arithmetic of an item is done once, not once per token. Warps, not loads per thread, keep memory busy: with
// one token's loads in flight a thread needs 40 registers, and q, k of 4 x 4096 tokens (16 + 4 heads of 128, 32 turned,
// bf16, views of a fused projection) take 33 us (5.1 TB/s); with two tokens ahead 49 us, with four 65 us.
template <typename T, int V, bool IL>
__global__ void __launch_bounds__(kMaxThreads, 3) rotary_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                             T* __restrict__ oq, T* __restrict__ ok, const Args a,
                                                             const int turn_units, const int copy_units, const int tokens) {
  constexpr int N = IL && V == 1 ? 2 : V;  // channels of a turned unit (of each half of its pairs in the half layout)
  constexpr int L = N / V;                 // packs of it
  constexpr int A = IL ? N / 2 : V;        // angles of it
  using Pk = Pack<T, V>;
  const unsigned heads = a.H + a.HK, turned = heads * turn_units;
  unsigned i = blockIdx.z * blockDim.x + threadIdx.x;
  if (i >= turned + heads * copy_units) return;
  const bool turn = i < turned;
  if (!turn) i -= turned;
  const unsigned units = turn ? turn_units : copy_units, hh = i / units, u = i - hh * units;
  const int b = blockIdx.y, t0 = blockIdx.x * tokens, t1 = a.T - t0 < tokens ? a.T : t0 + tokens;
  const bool is_q = hh < (unsigned)a.H;
  const Rows in = is_q ? a.q : a.k;
  const long long h = is_q ? hh : hh - a.H, nh = is_q ? a.H : a.HK;
  const int c = turn ? (int)u * N : a.R + (int)u * V;
  const T* src = (is_q ? q : k) + b * in.b + t0 * in.t + h * in.h + c;
  T* dst = (is_q ? oq : ok) + (((long long)b * a.T + t0) * nh + h) * a.D + c;
  const long long sstep = in.t, dstep = nh * a.D;
  if (!turn) {
    for (int t = t0; t < t1; ++t, src += sstep, dst += dstep) *reinterpret_cast<Pk*>(dst) = *reinterpret_cast<const Pk*>(src);
    return;
  }
  for (int t = t0; t < t1; ++t, src += sstep, dst += dstep) {
    Pk x[L], y;
    float2 an[A];
#pragma unroll
    for (int l = 0; l < L; ++l) x[l] = *reinterpret_cast<const Pk*>(src + l * V);
    if (!IL) y = *reinterpret_cast<const Pk*>(src + a.R / 2);
    long long p = t;
    if (a.positions != nullptr) {
      const long long w = b * a.pos_b + t;
      p = a.pos64 ? __ldg(static_cast<const long long*>(a.positions) + w)
                  : (long long)__ldg(static_cast<const int*>(a.positions) + w);
    }
    p = p < 0 ? 0 : p >= a.P ? a.P - 1 : p;  // never outside the table
    const float2* cs = a.table + p * (a.R / 2) + (IL ? c / 2 : c);
    if (A % 2 == 0 && a.table16) {  // an even number of angles starts on 16 bytes when the table's rows do
#pragma unroll
      for (int e = 0; e + 1 < A; e += 2) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(cs + e));
        an[e] = make_float2(v.x, v.y);
        an[e + 1] = make_float2(v.z, v.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < A; ++e) an[e] = __ldg(cs + e);
    }
    if constexpr (IL) {
      T* v = reinterpret_cast<T*>(x);
#pragma unroll
      for (int e = 0; e < A; ++e) {
        const float f = to_f<T>(v[2 * e]), g = to_f<T>(v[2 * e + 1]), sn = an[e].y * a.sign;
        v[2 * e] = from_f<T>(f * an[e].x - g * sn);
        v[2 * e + 1] = from_f<T>(g * an[e].x + f * sn);
      }
    } else {
#pragma unroll
      for (int e = 0; e < A; ++e) {
        const float f = to_f<T>(x[0].v[e]), g = to_f<T>(y.v[e]), sn = an[e].y * a.sign;
        x[0].v[e] = from_f<T>(f * an[e].x - g * sn);
        y.v[e] = from_f<T>(g * an[e].x + f * sn);
      }
      *reinterpret_cast<Pk*>(dst + a.R / 2) = y;
    }
#pragma unroll
    for (int l = 0; l < L; ++l) *reinterpret_cast<Pk*>(dst + l * V) = x[l];
  }
}

template <typename T, int V, bool IL>
int launch(const void* q, const void* k, void* oq, void* ok, const Args& a, cudaStream_t stream) {
  const int turn = IL ? a.R / (V == 1 ? 2 : V) : a.R / 2 / V, copy = (a.D - a.R) / V;
  const long long items = (long long)(a.H + a.HK) * (turn + copy);
  const long long passes = (items + kMaxThreads - 1) / kMaxThreads;
  if (passes > 65535) return GD_ERR_SHAPE;
  const int threads = (int)((items + passes * 32 - 1) / (passes * 32)) * 32;
  // fewer tokens a CTA where that many leave SMs with less than 1,024 threads
  int tokens = kTokens;
  while (tokens > 1 && (long long)a.B * ((a.T + tokens - 1) / tokens) * passes * threads < 148 * 1024) tokens /= 2;
  rotary_kernel<T, V, IL><<<dim3((unsigned)((a.T + tokens - 1) / tokens), (unsigned)a.B, (unsigned)passes), threads, 0,
                            stream>>>(static_cast<const T*>(q), static_cast<const T*>(k), static_cast<T*>(oq),
                                      static_cast<T*>(ok), a, turn, copy, tokens);
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
  if (B < 0 || B > 65535 || T < 0 || H < 0 || HK < 0 || D <= 0 || R <= 0 || R % 2 != 0 || R > D || table_rows < 0)
    return GD_ERR_SHAPE;
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
