// The residual addition with its RMS norm (the step that opens every layer of the decoder), one pass each way, and the
// form whose output is e4m3 with scales (the input of an 8-bit projection).
//   s = (x + res).to(T)                         the residual stream carried on (s = x without a residual)
//   r = rsqrt(mean(s^2) + eps),  xh = s r       (fp32)
//   y = (xh w').to(T)                           w' = w, or 1 + w for a zero-centred weight; one rounding
//   backward: h = dy w',  dx = (ds + r (h - xh mean(h xh))).to(T)  (the gradient of x and of res),
//             dw = sum over rows of dy xh       (only when asked: fixed-order partial rows, then a sum)
//   8 bits:   a = max |y| over a group of channels, scale = max(a / 448, 2^-126) (1 where a = 0), q = e4m3(y / scale),
//             from the fp32 y: the only rounding is the one to e4m3
//
// Bound by HBM, the backward and the 8-bit form nearly as much by issue slots: the forward moves 4 elements per channel
// (x, res in; s, y out), the backward 4 (s, dy, ds in; dx out), the 8-bit form 3 and a byte. So a row is read once: a team
// of TPR threads holds it in registers as 16-byte chunks.
// Chunks are those of the flat [rows * D] array, which start on 16-byte boundaries whatever D is; where D is not a
// multiple of the chunk a row's first and last chunk are shared with its neighbours: their foreign
// elements are read with them, count as zero, and are not written. So odd widths run on 16-byte loads too.
// Measured (bf16): 32,771 rows of 2,048 forward 83.6 us (6.4 TB/s), backward with dw 102.3 + 3.5 us (5.2 TB/s); 16,384
// rows of 4,096 to e4m3 in groups of 128 90.5 us (5.2 TB/s). A plain copy runs at 6.5 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gated_delta_b200.h"

namespace {

constexpr int kMaxChunks = 2048;    // 16-byte chunks of a row: two for each of 1024 threads
constexpr int kMaxD = kMaxChunks * 8;
constexpr int kThreads = 256;       // a CTA, unless a row needs more
constexpr int kMaxPartials = 1024;  // CTAs of the backward with dw (its fixed-order partial rows)
constexpr float kE4m3Max = 448.f;
constexpr float kLeastTop = kE4m3Max * 1.17549435e-38f;  // of a group: its scale is the smallest normal number

// Resident CTAs of an SM, which the register limits are set for. The backward holds more of a row: 80 registers a thread at
// one chunk (three CTAs of 256; at four its sums spill and it takes 160 us instead of 111 us for 32,771 rows of 2,048, bf16),
// 128 at two.
constexpr int per_sm(int threads, int nv, bool bwd) {
  return threads == 1024 ? 1 : threads == 512 ? 1 : nv == 1 ? (bwd ? 3 : 4) : bwd ? 2 : 3;
}

// ---- E = 16 / sizeof(T) consecutive elements as floats
template <typename T>
struct Vec {
  static constexpr int E = 16 / sizeof(T);
  __device__ __forceinline__ static void unpack(const uint4 r, float (&f)[E]) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        f[i] = __uint_as_float(u[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(u + i));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      } else {
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(u + i));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ static uint4 pack(const float (&f)[E]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        u[i] = __float_as_uint(f[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
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

// ---- two fp32 values at once (the packed instructions take an issue slot for two operations: these kernels move a chunk of
// 8 elements for every hundred instructions or so, and an SM issues about that many in the time its share of HBM takes)
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unf2(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float sum2(F2 v) {
  float a, b;
  unf2(v, a, b);
  return a + b;
}
// a 16-byte chunk as E / 2 pairs, and back (rounded)
template <typename T>
__device__ __forceinline__ void unpack2(const uint4 r, F2 (&f)[Vec<T>::E / 2]) {
  float v[Vec<T>::E];
  Vec<T>::unpack(r, v);
#pragma unroll
  for (int i = 0; i < Vec<T>::E / 2; ++i) f[i] = f2(v[2 * i], v[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ uint4 pack2(const F2 (&f)[Vec<T>::E / 2]) {
  float v[Vec<T>::E];
#pragma unroll
  for (int i = 0; i < Vec<T>::E / 2; ++i) unf2(f[i], v[2 * i], v[2 * i + 1]);
  return Vec<T>::pack(v);
}
// w' of the chunk that starts at column c, in pairs
template <typename T>
__device__ __forceinline__ void weights2(const void* w, int wdtype, float bias, int c, F2 (&f)[Vec<T>::E / 2]) {
  if (wdtype == GD_FLOAT32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + c);
#pragma unroll
    for (int i = 0; i < Vec<T>::E / 4; ++i) {
      const float4 v = __ldg(p + i);
      f[2 * i] = f2(v.x, v.y);
      f[2 * i + 1] = f2(v.z, v.w);
    }
  } else {
    unpack2<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c)), f);
  }
#pragma unroll
  for (int i = 0; i < Vec<T>::E / 2; ++i) f[i] = add2(f[i], f2(bias, bias));
}

// A thread's view of its row: chunk j of the thread starts at flat element `at(j)`; elements [lo, hi) are the row's.
template <typename T>
struct Row {
  static constexpr int E = Vec<T>::E;
  long long lo, hi, total;  // flat: the row's elements, the array's end
  long long first;          // flat start of the thread's chunk 0
  int step;                 // elements between the thread's chunks
  __device__ __forceinline__ Row(long long row, long long rows, int D, int sub, int tpr)
      : lo(row * D), hi(row < rows ? row * D + D : row * D), total(rows * D), step(tpr * E) {
    first = lo / E * E + (long long)sub * E;
  }
  __device__ __forceinline__ long long at(int j) const { return first + (long long)j * step; }
  __device__ __forceinline__ bool live(int j) const { return at(j) < hi; }
  __device__ __forceinline__ bool whole(long long a) const { return a >= lo && a + E <= hi; }
  __device__ __forceinline__ bool mine(long long e) const { return e >= lo && e < hi; }
  // chunk a of p as it stands in memory; foreign elements as zero
  __device__ __forceinline__ uint4 load(const T* p, long long a) const {
    float f[E];
    if (a + E <= total) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + a));
      if (whole(a)) return u;
      Vec<T>::unpack(u, f);
    } else {  // the array's last, partial chunk
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = a + e < total ? to_f<T>(p[a + e]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = mine(a + e) ? f[e] : 0.f;
    return Vec<T>::pack(f);
  }
  __device__ __forceinline__ void store(T* p, long long a, const float (&f)[E]) const {
    if (whole(a)) {
      *reinterpret_cast<uint4*>(p + a) = Vec<T>::pack(f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (mine(a + e)) p[a + e] = from_f<T>(f[e]);
    }
  }
  // the weights w' of chunk a from shared memory (load_weights); of foreign elements, any
  __device__ __forceinline__ void weights(const float* w, int stride, int D, long long a, float (&f)[E]) const {
    const int c = (int)(a - lo);
    if (whole(a)) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = w[((c + e) & 7) * stride + ((c + e) >> 3)];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int k = c + e < 0 ? 0 : c + e >= D ? D - 1 : c + e;
        f[e] = w[(k & 7) * stride + (k >> 3)];
      }
    }
  }
};

// w' in shared memory, element e at (e mod 8, e / 8) of [8][stride]: a warp's lanes read consecutive words whatever a row's
// start is. Returns the first float past it (a multiple of 16 bytes on).
__host__ __device__ __forceinline__ int weight_stride(int D) { return (D + 7) / 8 + 1; }
__host__ __device__ __forceinline__ int weight_floats(int D) { return (8 * weight_stride(D) + 3) / 4 * 4; }
template <typename T>
__device__ __forceinline__ float* load_weights(float* sm, const void* w, int wdtype, float bias, int D) {
  const int stride = weight_stride(D);
  for (int e = threadIdx.x; e < D; e += blockDim.x)
    sm[(e & 7) * stride + (e >> 3)] =
        bias + (wdtype == GD_FLOAT32 ? __ldg(static_cast<const float*>(w) + e) : to_f<T>(static_cast<const T*>(w)[e]));
  return sm + weight_floats(D);
}

// n floats from shared memory (16-byte aligned; those up to the next multiple of four are zero), in the same order in every
// thread
__device__ __forceinline__ float sum_parts(const float* p, int n) {
  float s = 0.f;
  for (int i = 0; i < n; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    s += (v.x + v.y) + (v.z + v.w);
  }
  return s;
}
// Where a team's warps leave their parts: n floats from `at` on, this thread's warp's at `mine`
struct Parts {
  int n, at, mine;
  __device__ __forceinline__ explicit Parts(int tpr) {
    const int warp = threadIdx.x >> 5;
    n = tpr >> 5;
    const int team = n > 0 ? warp / n : 0;
    at = team * ((n + 3) & ~3);
    mine = at + warp - team * n;
  }
};

// The sum over a team (a power of two up to 32 of consecutive threads, or whole warps); every thread of the CTA calls. red:
// a float per warp, zero before the first call; two buffers in turn, so that one barrier a row is enough.
__device__ __forceinline__ float team_sum(float v, int tpr, const Parts& p, float* red) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
    if (o < tpr) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  if ((threadIdx.x & 31) == 0) red[p.mine] = v;
  __syncthreads();
  return sum_parts(red + p.at, p.n);
}

// 1 / sqrt(mean + eps): the approximate reciprocal root is within 2 units in the last place
__device__ __forceinline__ float inv_rms(float ss, float inv_D, float eps) { return rsqrtf(fmaf(ss, inv_D, eps)); }

// The scale of a group whose largest |y| is `top`, and 1 / scale to 2 units in the last place (any number where all are
// zero). Below kLeastTop the scale stays 2^-126: a smaller one would have lost bits (or be 0), and its reciprocal would
// overflow. The eighths keep the divisor inside __fdividef's range, up to 2^126.
__device__ __forceinline__ float group_scale(float top) { return top > 0.f ? fmaxf(top, kLeastTop) / kE4m3Max : 1.f; }
__device__ __forceinline__ float group_factor(float top) {
  return __fdividef(0.125f * kE4m3Max, 0.125f * fmaxf(top, kLeastTop));
}

// ---- forward, plain (FP8 = 0) or with the 8-bit output. Persistent CTAs: a team walks the rows, with the next row's
// loads in flight while this one is reduced and written, and keeps its columns' weights in registers.
//
// 8 bits: group g of a row is channels [g G, (g + 1) G). FP8 = 1: a group is the chunks of `lanes` consecutive lanes (a power
// of two of 32 chunks at most) and its maximum a shuffle. FP8 = 2: any G of 8 channels or more, a maximum per group in shared
// memory (integer maxima of non-negative floats: the order does not matter); a chunk of a row whose width is no multiple of
// the chunk touches two groups at most. A NaN counts in no maximum and comes out as e4m3's NaN.
//
// The widths that are whole chunks (the others below):
template <typename T, int NV, int FP8, int THREADS>
__global__ void __launch_bounds__(THREADS, per_sm(THREADS, NV, false))
    rnorm_fwd_flat(const T* __restrict__ x, const T* __restrict__ res,
                   const void* __restrict__ w, T* __restrict__ s, T* __restrict__ y,
                   uint8_t* __restrict__ q, float* __restrict__ scale, int wdtype,
                   float bias, long long rows, int D, int G, int lanes, int tpr,
                   float eps) {
  constexpr int E = Vec<T>::E, H = E / 2;
  __shared__ __align__(16) float red[2][32];
  const Parts parts(tpr);
  for (int i = threadIdx.x; i < 64; i += blockDim.x) (&red[0][0])[i] = 0.f;
  __syncthreads();
  extern __shared__ unsigned int tops[];  // FP8 = 2: [teams][groups] bit patterns
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const int groups = FP8 ? (D + G - 1) / G : 0;
  const long long step = (long long)gridDim.x * teams, hop = step * D;
  const float inv_D = 1.f / (float)D;
  int col[NV];
  F2 wv[NV][H];
  uint4 a[NV], b[NV];
  long long r0 = (long long)blockIdx.x * teams + team, off = r0 * D;  // the team's row, its first element
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (sub + j * tpr) * E;
    if (col[j] >= D) {
      col[j] = -1;  // no chunk of the row
#pragma unroll
      for (int i = 0; i < H; ++i) wv[j][i] = 0;
    } else {
      weights2<T>(w, wdtype, bias, col[j], wv[j]);
    }
    a[j] = b[j] = make_uint4(0, 0, 0, 0);
  }
  auto fetch = [&](long long at) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col[j] >= 0) {
        a[j] = __ldg(reinterpret_cast<const uint4*>(x + at + col[j]));
        if (res != nullptr) b[j] = __ldg(reinterpret_cast<const uint4*>(res + at + col[j]));
      }
  };
  if (r0 < rows) fetch(off);
  for (int parity = 0; r0 - team < rows; r0 += step, off += hop, parity ^= 1) {
    const bool live = r0 < rows;
    F2 v[NV][H], ss2 = 0;
    if constexpr (FP8 == 2) {
      __syncthreads();  // the last row's maxima are read
      for (int i = threadIdx.x; i < groups * teams; i += blockDim.x) tops[i] = 0u;
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack2<T>(a[j], v[j]);
      if (res != nullptr) {
        F2 f[H];
        unpack2<T>(b[j], f);
#pragma unroll
        for (int i = 0; i < H; ++i) v[j][i] = add2(v[j][i], f[i]);
        const uint4 packed = pack2<T>(v[j]);
        if constexpr (!std::is_same<T, float>::value) unpack2<T>(packed, v[j]);  // rounded to T
        if (live && col[j] >= 0) *reinterpret_cast<uint4*>(s + off + col[j]) = packed;
      }
    }
    if (r0 + step < rows) fetch(off + hop);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < H; ++i) ss2 = fma2(v[j][i], v[j][i], ss2);
    const float r = inv_rms(team_sum(sum2(ss2), tpr, parts, red[parity]), inv_D, eps);
    const F2 rr = f2(r, r);
    float top[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < H; ++i) v[j][i] = mul2(mul2(v[j][i], rr), wv[j][i]);
      if constexpr (FP8 == 0) {
        if (live && col[j] >= 0) *reinterpret_cast<uint4*>(y + off + col[j]) = pack2<T>(v[j]);
      } else {
        top[j] = 0.f;
#pragma unroll
        for (int i = 0; i < H; ++i) {
          float f, g;
          unf2(v[j][i], f, g);
          top[j] = fmaxf(top[j], fmaxf(fabsf(f), fabsf(g)));
        }
        if constexpr (FP8 == 1) {
          for (int o = lanes >> 1; o >= 1; o >>= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
        } else {
          if (col[j] >= 0) atomicMax(&tops[team * groups + col[j] / G], __float_as_uint(top[j]));
        }
      }
    }
    if constexpr (FP8 == 2) __syncthreads();
    if constexpr (FP8 != 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!live || col[j] < 0) continue;
        const int g = col[j] / G;
        if constexpr (FP8 == 2) top[j] = __uint_as_float(tops[team * groups + g]);
        const float sc = group_factor(top[j]);
        if (FP8 == 1 ? (sub & (lanes - 1)) == 0 : col[j] == g * G)
          scale[r0 * groups + g] = group_scale(top[j]);
        uint32_t packed[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          float f[4];
          unf2(mul2(v[j][2 * i], f2(sc, sc)), f[0], f[1]);
          unf2(mul2(v[j][2 * i + 1], f2(sc, sc)), f[2], f[3]);
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
          packed[i] = lo | hi << 16;
        }
        if constexpr (E == 8) *reinterpret_cast<uint2*>(q + off + col[j]) = make_uint2(packed[0], packed[1]);
        else *reinterpret_cast<uint32_t*>(q + off + col[j]) = packed[0];
      }
    }
  }
}

// Widths that are no whole number of chunks (FP8 = 0 or 2): the same walk, a row's chunks cut out of the flat array.
template <typename T, int NV, int FP8, int THREADS>
__global__ void __launch_bounds__(THREADS, per_sm(THREADS, NV, false))
    rnorm_fwd_odd(const T* __restrict__ x, const T* __restrict__ res,
                  const void* __restrict__ w, T* __restrict__ s, T* __restrict__ y,
                  uint8_t* __restrict__ q, float* __restrict__ scale, int wdtype,
                  float bias, long long rows, int D, int G, int tpr, float eps) {
  constexpr int E = Vec<T>::E;
  __shared__ __align__(16) float red[2][32];
  const Parts parts(tpr);
  for (int i = threadIdx.x; i < 64; i += blockDim.x) (&red[0][0])[i] = 0.f;
  __syncthreads();
  extern __shared__ __align__(16) float wsm[];  // the weights; FP8 = 2: then [teams][groups] bit patterns of maxima
  unsigned int* tops = reinterpret_cast<unsigned int*>(load_weights<T>(wsm, w, wdtype, bias, D));
  const int wstride = weight_stride(D);
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const int groups = FP8 ? (D + G - 1) / G : 0;
  const long long step = (long long)gridDim.x * teams;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 a[NV], b[NV];
  auto fetch = [&](long long r) {
    const Row<T> row(r, rows, D, sub, tpr);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      a[j] = row.live(j) ? row.load(x, row.at(j)) : zero;
      b[j] = res != nullptr && row.live(j) ? row.load(res, row.at(j)) : zero;
    }
  };
  long long base = (long long)blockIdx.x * teams;
  fetch(base + team);
  const float inv_D = 1.f / (float)D;
  for (int parity = 0; base < rows; base += step, parity ^= 1) {
    const long long r0 = base + team;
    const Row<T> row(r0, rows, D, sub, tpr);
    float v[NV][E];
    float ss = 0.f;
    if constexpr (FP8 == 2) {
      __syncthreads();  // the last row's maxima are read
      for (int i = threadIdx.x; i < groups * teams; i += blockDim.x) tops[i] = 0u;
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Vec<T>::unpack(a[j], v[j]);
      if (res != nullptr && row.live(j)) {
        float f[E];
        Vec<T>::unpack(b[j], f);
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][e] += f[e];
        const uint4 packed = Vec<T>::pack(v[j]);
        Vec<T>::unpack(packed, v[j]);  // rounded to T
        row.store(s, row.at(j), v[j]);
      }
    }
    if (base + step < rows) fetch(r0 + step);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(v[j][e], v[j][e], ss);
    const float r = inv_rms(team_sum(ss, tpr, parts, red[parity]), inv_D, eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!row.live(j)) continue;
      float wv[E];
      row.weights(wsm, wstride, D, row.at(j), wv);
#pragma unroll
      for (int e = 0; e < E; ++e) v[j][e] = v[j][e] * r * wv[e];
      if constexpr (FP8 == 0) row.store(y, row.at(j), v[j]);
      if constexpr (FP8 == 2) {
        const int c0 = (int)(row.at(j) - row.lo);  // may be negative: the chunk starts in the row before
        const int g0 = c0 > 0 ? c0 / G : 0, split = (g0 + 1) * G;
        float f = 0.f, g = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float m = row.mine(row.at(j) + e) ? fabsf(v[j][e]) : 0.f;
          if (c0 + e < split) f = fmaxf(f, m);
          else g = fmaxf(g, m);
        }
        atomicMax(&tops[team * groups + g0], __float_as_uint(f));
        if (g > 0.f) atomicMax(&tops[team * groups + g0 + 1], __float_as_uint(g));
      }
    }
    if constexpr (FP8 != 0) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!row.live(j)) continue;
        const long long at = row.at(j);
        const int c0 = (int)(at - row.lo), g0 = c0 > 0 ? c0 / G : 0, split = (g0 + 1) * G;
        uint32_t packed[E / 4];
        const float t1 = __uint_as_float(tops[team * groups + g0]);
        const float t2 = g0 + 1 < groups ? __uint_as_float(tops[team * groups + g0 + 1]) : 0.f;
        const float sc = group_factor(t1), sc2 = group_factor(t2);
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = v[j][4 * i + e] * (c0 + 4 * i + e < split ? sc : sc2);
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
          packed[i] = lo | hi << 16;
        }
        if (row.whole(at)) {
          if constexpr (E == 8) *reinterpret_cast<uint2*>(q + at) = make_uint2(packed[0], packed[1]);
          else *reinterpret_cast<uint32_t*>(q + at) = packed[0];
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (row.mine(at + e)) q[at + e] = (uint8_t)(packed[e / 4] >> (8 * (e % 4)));
        }
      }
      if (r0 < rows)
        for (int g = sub; g < groups; g += tpr) {
          const float t = __uint_as_float(tops[team * groups + g]);
          scale[r0 * groups + g] = group_scale(t);
        }
    }
  }
}

// ---- backward. CTA p takes the blocks of R rows (R teams) p, p + grid, ...: every CTA has work to the end, the next row's
// loads in flight. With dw, where widths are whole chunks, a thread keeps its columns' sums in registers (the columns stay
// its own over the rows) and the CTA's teams are added in team order; else the columns move with the row, so the sums stand
// in shared memory, where one thread adds to an element at a time, in the rows' order (one team a CTA).
template <typename T, int NV, bool DW, int THREADS>
__global__ void __launch_bounds__(THREADS, per_sm(THREADS, NV, true))
    rnorm_bwd_flat(const T* __restrict__ s, const void* __restrict__ w,
                   const T* __restrict__ dy, const T* __restrict__ ds,
                   T* __restrict__ dx, float* __restrict__ part, int wdtype,
                   float bias, long long rows, int D, int tpr, float eps) {
  constexpr int E = Vec<T>::E, H = E / 2;
  __shared__ __align__(16) float red[2][2][32];
  const Parts parts(tpr);
  for (int i = threadIdx.x; i < 128; i += blockDim.x) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  extern __shared__ __align__(16) float sums[];  // DW: [teams][D], at the end
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const long long step = (long long)gridDim.x * teams, hop = step * D;
  const float inv_D = 1.f / (float)D;
  int col[NV];
  F2 wv[NV][H], acc[DW ? NV : 1][H];
  uint4 nv[NV], ng[NV], nc[NV];  // the next row's s, dy, ds as they stand in memory
  long long r0 = (long long)blockIdx.x * teams + team, off = r0 * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    col[j] = (sub + j * tpr) * E;
    if (col[j] >= D) {
      col[j] = -1;
#pragma unroll
      for (int i = 0; i < H; ++i) wv[j][i] = 0;
    } else {
      weights2<T>(w, wdtype, bias, col[j], wv[j]);
    }
    nv[j] = ng[j] = nc[j] = make_uint4(0, 0, 0, 0);
    if constexpr (DW)
#pragma unroll
      for (int i = 0; i < H; ++i) acc[j][i] = 0;
  }
  auto fetch = [&](long long at) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col[j] >= 0) {
        nv[j] = __ldg(reinterpret_cast<const uint4*>(s + at + col[j]));
        if (dy != nullptr) ng[j] = __ldg(reinterpret_cast<const uint4*>(dy + at + col[j]));
        if (ds != nullptr) nc[j] = __ldg(reinterpret_cast<const uint4*>(ds + at + col[j]));
      }
  };
  if (r0 < rows) fetch(off);
  for (int parity = 0; r0 - team < rows; r0 += step, off += hop, parity ^= 1) {
    const bool live = r0 < rows;
    F2 v[NV][H], g[NV][H], ss2 = 0, dot2 = 0;  // sums of s^2, and of h s: the mean of h xh is dot r / D
    uint4 c[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack2<T>(nv[j], v[j]);
      unpack2<T>(ng[j], g[j]);
      c[j] = nc[j];
    }
    if (r0 + step < rows) fetch(off + hop);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < H; ++i) {
        ss2 = fma2(v[j][i], v[j][i], ss2);
        dot2 = fma2(mul2(g[j][i], wv[j][i]), v[j][i], dot2);
      }
    float ss = sum2(ss2), dot = sum2(dot2);
    // two sums at once: their warp parts side by side, one barrier a row (two buffers in turn)
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
      if (o < tpr) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
    if (tpr > 32) {
      if ((threadIdx.x & 31) == 0) {
        red[parity][0][parts.mine] = ss;
        red[parity][1][parts.mine] = dot;
      }
      __syncthreads();
      ss = sum_parts(red[parity][0] + parts.at, parts.n);
      dot = sum_parts(red[parity][1] + parts.at, parts.n);
    }
    const float r = inv_rms(ss, inv_D, eps), m = -dot * r * inv_D;
    const F2 rr = f2(r, r), mm = f2(m, m);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      F2 out[H];
      unpack2<T>(c[j], out);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const F2 xh = mul2(v[j][i], rr);
        out[i] = fma2(rr, fma2(xh, mm, mul2(g[j][i], wv[j][i])), out[i]);
        if constexpr (DW)
          if (live) acc[j][i] = fma2(g[j][i], xh, acc[j][i]);
      }
      if (live && col[j] >= 0) *reinterpret_cast<uint4*>(dx + off + col[j]) = pack2<T>(out);
    }
  }
  if constexpr (DW) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col[j] >= 0)
#pragma unroll
        for (int i = 0; i < H; ++i) *reinterpret_cast<F2*>(sums + (size_t)team * D + col[j] + 2 * i) = acc[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      float t = sums[i];
      for (int x = 1; x < teams; ++x) t += sums[(size_t)x * D + i];
      part[(size_t)blockIdx.x * D + i] = t;
    }
  }
}

// Widths that are no whole number of chunks, or more than 1,024 of them.
template <typename T, int NV, bool DW, int THREADS>
__global__ void __launch_bounds__(THREADS, per_sm(THREADS, NV, true))
    rnorm_bwd_odd(const T* __restrict__ s, const void* __restrict__ w,
                  const T* __restrict__ dy, const T* __restrict__ ds,
                  T* __restrict__ dx, float* __restrict__ part, int wdtype, float bias,
                  long long rows, int D, int tpr, float eps) {
  constexpr int E = Vec<T>::E;
  __shared__ __align__(16) float red[2][2][32];
  const Parts parts(tpr);
  for (int i = threadIdx.x; i < 128; i += blockDim.x) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  extern __shared__ __align__(16) float wsm[];  // the weights; DW: then the sums [D]
  float* sums = load_weights<T>(wsm, w, wdtype, bias, D);
  const int wstride = weight_stride(D);
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const long long step = (long long)gridDim.x * teams;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 nv[NV], ng[NV], nc[NV];  // the next row's s, dy, ds as they stand in memory
  auto fetch = [&](long long r) {
    const Row<T> row(r, rows, D, sub, tpr);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool live = row.live(j);
      nv[j] = live ? row.load(s, row.at(j)) : zero;
      ng[j] = live && dy != nullptr ? row.load(dy, row.at(j)) : zero;
      nc[j] = live && ds != nullptr ? row.load(ds, row.at(j)) : zero;
    }
  };
  long long base = (long long)blockIdx.x * teams;
  fetch(base + team);
  float wv[NV][E];
  const float inv_D = 1.f / (float)D;
  if constexpr (DW) {
    for (int i = threadIdx.x; i < D; i += blockDim.x) sums[i] = 0.f;
    __syncthreads();
  }
  for (int parity = 0; base < rows; base += step, parity ^= 1) {
    const Row<T> row(base + team, rows, D, sub, tpr);
    uint4 v[NV], g[NV], c[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = nv[j];
      g[j] = ng[j];
      c[j] = nc[j];
    }
    if (base + step < rows) fetch(base + step + team);
    float ss = 0.f, dot = 0.f;  // sum of s^2, and of h s: the mean of h xh is dot r / D
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!row.live(j)) continue;
      float vf[E], gf[E];
      row.weights(wsm, wstride, D, row.at(j), wv[j]);
      Vec<T>::unpack(v[j], vf);
      Vec<T>::unpack(g[j], gf);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        ss = fmaf(vf[e], vf[e], ss);
        dot = fmaf(gf[e] * wv[j][e], vf[e], dot);
      }
    }
    // two sums at once: their warp parts side by side, one barrier a row (two buffers in turn)
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
      if (o < tpr) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
    if (tpr > 32) {
      if ((threadIdx.x & 31) == 0) {
        red[parity][0][parts.mine] = ss;
        red[parity][1][parts.mine] = dot;
      }
      __syncthreads();
      ss = sum_parts(red[parity][0] + parts.at, parts.n);
      dot = sum_parts(red[parity][1] + parts.at, parts.n);
    } else if constexpr (DW) {
      __syncthreads();  // the last row's sums are in place (one team: an element's adders take turns)
    }
    const float r = inv_rms(ss, inv_D, eps);
    const float m = dot * r * inv_D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!row.live(j)) continue;
      const long long a = row.at(j);
      float vf[E], gf[E], out[E];
      Vec<T>::unpack(v[j], vf);
      Vec<T>::unpack(g[j], gf);
      Vec<T>::unpack(c[j], out);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float xh = vf[e] * r;
        out[e] += r * (gf[e] * wv[j][e] - xh * m);
        if constexpr (DW) gf[e] *= xh;
      }
      row.store(dx, a, out);
      if constexpr (DW) {
        float* p = sums + (a - row.lo);
        if (row.whole(a)) {
#pragma unroll
          for (int e = 0; e < E; ++e) p[e] += gf[e];
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (row.mine(a + e)) p[e] += gf[e];
        }
      }
    }
  }
  if constexpr (DW) {
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += blockDim.x) part[(size_t)blockIdx.x * D + i] = sums[i];
  }
}

// dw[i] = the partial rows' sum: 32 columns a CTA, 32 runs of rows, then the runs in order
template <typename TW>
__global__ void __launch_bounds__(1024) rnorm_dw(const float* __restrict__ part, TW* __restrict__ dw, int n, int D) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < D)
    for (int p = run; p < n; p += 32) t += part[(size_t)p * D + col];
  red[run][lane] = t;
  __syncthreads();
  if (run == 0 && col < D) {
    float u = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) u += red[k][lane];
    dw[col] = from_f<TW>(u);
  }
}

// ---- host
struct Shape {
  bool flat;
  int tpr, nv, threads, teams;
};

constexpr int kSms = 148;  // of a B200

int chunks_of(int D, int E) { return D % E == 0 ? D / E : D / E + 2; }  // with the two shared with the neighbours

// The team: one chunk a thread up to 256 chunks, CTAs of 256 threads then hold several teams of narrow rows (fewer where rows
// are too few to give every SM a CTA so). Two chunks a thread from there on, in as many whole warps as that takes: CTAs of up
// to 256 threads, of which an SM holds several that cover each other's barriers.
Shape shape_of(long long rows, int D, int E, bool one_team) {
  Shape s;
  s.flat = D % E == 0;
  const int chunks = chunks_of(D, E);
  s.nv = chunks <= 256 ? 1 : 2;
  if (s.nv == 1) {
    s.tpr = 4;
    while (s.tpr < chunks) s.tpr *= 2;
    s.threads = one_team ? s.tpr : kThreads;
    while (!one_team && s.threads > s.tpr && s.threads > 32 && rows * s.tpr / s.threads < kSms) s.threads /= 2;
    if (s.threads < 32) s.threads = s.tpr = 32;
  } else {
    s.tpr = s.threads = ((chunks + 1) / 2 + 31) / 32 * 32;
  }
  s.teams = s.threads / s.tpr;
  return s;
}
int launch_class(int threads) { return threads <= 256 ? 256 : threads <= 512 ? 512 : 1024; }
// persistent CTAs: as many as are resident
int grid_of(long long rows, const Shape& s, bool bwd, int most = 1 << 30) {
  const int cls = launch_class(s.threads);
  const long long blocks = (rows + s.teams - 1) / s.teams;
  const long long resident = (long long)kSms * per_sm(cls, s.nv, bwd) * (cls / s.threads > 0 ? cls / s.threads : 1);
  const long long g = blocks < resident ? blocks : resident;
  return (int)(g < most ? g : most);
}

int chunk_elems(int dtype) { return dtype == GD_FLOAT32 ? 4 : 8; }
bool dtype_ok(int d) { return d == GD_FLOAT32 || d == GD_FLOAT16 || d == GD_BFLOAT16; }
bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int check_common(const void* w, int dtype, int wdtype, long long rows, int D) {
  if (!dtype_ok(dtype) || !(wdtype == dtype || wdtype == GD_FLOAT32)) return GD_ERR_ARG;
  if (D <= 0 || D > kMaxD || chunks_of(D, chunk_elems(dtype)) > kMaxChunks || rows < 0 || rows > (1ll << 40))
    return GD_ERR_SHAPE;
  if (rows > 0 && w == nullptr) return GD_ERR_ARG;
  return GD_OK;
}

template <typename F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case GD_FLOAT32: return f(float{});
    case GD_FLOAT16: return f(__half{});
    default: return f(__nv_bfloat16{});
  }
}
int launched() { return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH); }


template <typename K>
bool enough_smem(K k, size_t bytes) {
  return bytes <= 48 * 1024 ||
         cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess ||
         (cudaGetLastError(), false);
}

// f(integral_constant NV, integral_constant THREADS)
template <typename F>
int with_shape(const Shape& s, F&& f) {
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (s.nv == 1) return f(One{}, std::integral_constant<int, 256>{});
  switch (launch_class(s.threads)) {
    case 256: return f(Two{}, std::integral_constant<int, 256>{});
    case 512: return f(Two{}, std::integral_constant<int, 512>{});
    default: return f(Two{}, std::integral_constant<int, 1024>{});
  }
}

template <int FP8>
int forward(const void* x, const void* res, const void* w, void* s, void* y, void* q, float* scale, int dtype, int wdtype,
            int zero_centered, long long rows, int D, int G, int lanes, const Shape& sh, size_t smem, float eps,
            void* stream) {
  const int grid = grid_of(rows, sh, false);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_shape(sh, [&](auto nv, auto threads) {
      constexpr int NV = decltype(nv)::value, TH = decltype(threads)::value;
      const cudaStream_t cs = static_cast<cudaStream_t>(stream);
      const float bias = zero_centered ? 1.f : 0.f;
      if (sh.flat)
        rnorm_fwd_flat<T, NV, FP8, TH><<<grid, sh.threads, smem, cs>>>(
            static_cast<const T*>(x), static_cast<const T*>(res), w, static_cast<T*>(s), static_cast<T*>(y),
            static_cast<uint8_t*>(q), scale, wdtype, bias, rows, D, G, lanes, sh.tpr, eps);
      else if constexpr (FP8 != 1) {
        auto k = rnorm_fwd_odd<T, NV, FP8, TH>;
        const size_t bytes = smem + weight_floats(D) * sizeof(float);
        if (!enough_smem(k, bytes)) return GD_ERR_LAUNCH;
        k<<<grid, sh.threads, bytes, cs>>>(static_cast<const T*>(x), static_cast<const T*>(res), w, static_cast<T*>(s),
                                           static_cast<T*>(y), static_cast<uint8_t*>(q), scale, wdtype, bias, rows, D, G,
                                           sh.tpr, eps);
      }
      return launched();
    });
  });
}

}  // namespace

extern "C" int gd_rnorm_fwd(const void* x, const void* res, const void* w, void* s, void* y, int dtype, int wdtype,
                            int zero_centered, long long rows, int D, float eps, void* stream) {
  if (const int st = check_common(w, dtype, wdtype, rows, D)) return st;
  if (rows == 0) return GD_OK;
  if (x == nullptr || y == nullptr || (res != nullptr && s == nullptr)) return GD_ERR_ARG;
  if (misaligned(x) || misaligned(res) || misaligned(w) || misaligned(s) || misaligned(y)) return GD_ERR_ALIGN;
  const Shape sh = shape_of(rows, D, chunk_elems(dtype), false);
  return forward<0>(x, res, w, s, y, nullptr, nullptr, dtype, wdtype, zero_centered, rows, D, 1, 1, sh, 0, eps, stream);
}

extern "C" int gd_rnorm_fp8(const void* x, const void* res, const void* w, void* s, void* q, float* scale, int dtype,
                            int wdtype, int zero_centered, long long rows, int D, int group, float eps, void* stream) {
  if (const int st = check_common(w, dtype, wdtype, rows, D)) return st;
  if (group < 0 || group % 8 != 0) return GD_ERR_SHAPE;
  if (rows == 0) return GD_OK;
  if (x == nullptr || q == nullptr || scale == nullptr || (res != nullptr && s == nullptr)) return GD_ERR_ARG;
  if (misaligned(x) || misaligned(res) || misaligned(w) || misaligned(s) || misaligned(q)) return GD_ERR_ALIGN;
  const int E = chunk_elems(dtype);
  const int G = group == 0 || group > D ? (D + 7) / 8 * 8 : group;  // 0: the whole row
  const Shape sh = shape_of(rows, D, E, false);
  // groups that are the chunks of a power of two of lanes of one warp; a row of one group: of the whole team
  const int groups = (D + G - 1) / G, lanes = groups == 1 && sh.nv == 1 ? sh.tpr : G / E;
  if (sh.flat && lanes <= 32 && lanes <= sh.tpr && (lanes & (lanes - 1)) == 0)
    return forward<1>(x, res, w, s, nullptr, q, scale, dtype, wdtype, zero_centered, rows, D, G, lanes, sh, 0, eps, stream);
  return forward<2>(x, res, w, s, nullptr, q, scale, dtype, wdtype, zero_centered, rows, D, G, 1, sh,
                    (size_t)sh.teams * groups * sizeof(unsigned int), eps, stream);
}

extern "C" size_t gd_rnorm_workspace_bytes(long long rows, int D) {
  if (rows <= 0 || D <= 0 || D > kMaxD) return 0;
  const long long n = rows < kMaxPartials ? rows : kMaxPartials;
  return (size_t)n * D * sizeof(float);
}

extern "C" int gd_rnorm_bwd(const void* s, const void* w, const void* dy, const void* ds, void* dx, void* dw, int dtype,
                            int wdtype, int zero_centered, long long rows, int D, float eps, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int st = check_common(w, dtype, wdtype, rows, D)) return st;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dw != nullptr &&
        cudaMemsetAsync(dw, 0, (size_t)D * (wdtype == GD_FLOAT32 ? 4 : 2), cs) != cudaSuccess)
      return (cudaGetLastError(), GD_ERR_LAUNCH);
    return GD_OK;
  }
  if (s == nullptr || dx == nullptr) return GD_ERR_ARG;
  if (misaligned(s) || misaligned(w) || misaligned(dy) || misaligned(ds) || misaligned(dx) || misaligned(workspace))
    return GD_ERR_ALIGN;
  if (dw != nullptr && (workspace == nullptr || workspace_bytes < gd_rnorm_workspace_bytes(rows, D)))
    return GD_ERR_WORKSPACE;
  const int E = chunk_elems(dtype);
  const Shape sh = shape_of(rows, D, E, dw != nullptr && D % E != 0);
  const int grid = grid_of(rows, sh, true, dw != nullptr ? kMaxPartials : 1 << 30);
  const float bias = zero_centered ? 1.f : 0.f;
  float* part = static_cast<float*>(workspace);
  int st = with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_shape(sh, [&](auto nv, auto threads) {
      constexpr int NV = decltype(nv)::value, TH = decltype(threads)::value;
      auto k = dw != nullptr ? rnorm_bwd_odd<T, NV, true, TH> : rnorm_bwd_odd<T, NV, false, TH>;
      if constexpr (TH <= 512)  // two chunks of each of 1,024 threads would not fit the registers
        if (sh.flat) k = dw != nullptr ? rnorm_bwd_flat<T, NV, true, TH> : rnorm_bwd_flat<T, NV, false, TH>;
      // the sums of dw, and the weights of the kernel that cuts rows out of the flat array
      const size_t smem = ((dw == nullptr ? 0 : (size_t)(sh.flat ? sh.teams : 1) * D) +
                           (TH <= 512 && sh.flat ? 0 : weight_floats(D))) * sizeof(float);
      if (!enough_smem(k, smem)) return GD_ERR_LAUNCH;
      k<<<grid, sh.threads, smem, cs>>>(static_cast<const T*>(s), w, static_cast<const T*>(dy), static_cast<const T*>(ds),
                                        static_cast<T*>(dx), part, wdtype, bias, rows, D, sh.tpr, eps);
      return launched();
    });
  });
  if (st != GD_OK || dw == nullptr) return st;
  return with_type(wdtype, [&](auto t) {
    using TW = decltype(t);
    rnorm_dw<TW><<<(D + 31) / 32, 1024, 0, cs>>>(part, static_cast<TW*>(dw), grid, D);
    return launched();
  });
}
