// The residual addition with its RMS norm (the step that opens every layer of the decoder), one pass each way, and the
// form whose output is e4m3 with scales (the input of an 8-bit projection).
//   s = (x + res).to(T)                         the residual stream carried on (s = x without a residual)
//   r = rsqrt(mean(s^2) + eps),  xh = s r       (fp32)
//   y = (xh w').to(T)                           w' = w, or 1 + w for a zero-centred weight; one rounding
//   backward: h = dy w',  dx = (ds + r (h - xh mean(h xh))).to(T)  (the gradient of x and of res),
//             dw = sum over rows of dy xh       (only when asked: fixed-order partial rows, then a sum)
//   8 bits:   a = max |y| over a group of channels, scale = a / 448 (1 where a = 0), q = e4m3(y / scale), from the
//             fp32 y: the only rounding is the one to e4m3
//
// Bound by HBM: the forward moves 4 elements per channel (x, res in; s, y out), the backward 4 (s, dy, ds in; dx out),
// the 8-bit form 3 and a byte. So a row is read once: a team of TPR threads holds it in registers as 16-byte chunks.
// Chunks are those of the flat [rows * D] array, which start on 16-byte boundaries whatever D is; where D is not a
// multiple of the chunk (FLAT = false) a row's first and last chunk are shared with its neighbours: their foreign
// elements are read with them, count as zero, and are not written. So odd widths run on 16-byte loads too.
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

// A thread's view of its row: chunk j of the thread starts at flat element `at(j)`; elements [lo, hi) are the row's.
template <typename T, bool FLAT>
struct Row {
  static constexpr int E = Vec<T>::E;
  long long lo, hi, total;  // flat: the row's elements, the array's end
  long long first;          // flat start of the thread's chunk 0
  int step;                 // elements between the thread's chunks
  __device__ __forceinline__ Row(long long row, long long rows, int D, int sub, int tpr)
      : lo(row * D), hi(row < rows ? row * D + D : row * D), total(rows * D), step(tpr * E) {
    first = (FLAT ? lo : lo / E * E) + (long long)sub * E;
  }
  __device__ __forceinline__ long long at(int j) const { return first + (long long)j * step; }
  __device__ __forceinline__ bool live(int j) const { return at(j) < hi; }
  __device__ __forceinline__ bool whole(long long a) const { return FLAT || (a >= lo && a + E <= hi); }
  __device__ __forceinline__ bool mine(long long e) const { return FLAT || (e >= lo && e < hi); }
  // chunk a of p as it stands in memory; foreign elements as zero
  __device__ __forceinline__ uint4 load(const T* p, long long a) const {
    if (FLAT) return __ldg(reinterpret_cast<const uint4*>(p + a));
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
  // the weights w' of chunk a (zero at foreign elements); wdtype as the ABI's
  __device__ __forceinline__ void weights(const void* w, int wdtype, float bias, long long a, float (&f)[E]) const {
    const int c = (int)(a - lo);
    if (FLAT) {
      if (wdtype == GD_FLOAT32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(w) + c);
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          const float4 v = __ldg(p + i);
          f[4 * i] = v.x;
          f[4 * i + 1] = v.y;
          f[4 * i + 2] = v.z;
          f[4 * i + 3] = v.w;
        }
      } else {  // x's own type
        Vec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(w) + c)), f);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] += bias;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[e] = 0.f;
        if (mine(a + e))
          f[e] = bias + (wdtype == GD_FLOAT32 ? __ldg(static_cast<const float*>(w) + c + e)
                                              : to_f<T>(static_cast<const T*>(w)[c + e]));
      }
    }
  }
};

// The sum over a team of TPR threads (a power of two, 4 or more consecutive threads of the CTA); every thread of the CTA
// calls. red: one float per warp; two buffers in turn, so that one barrier a row is enough.
__device__ __forceinline__ float team_sum(float v, int tpr, float* red) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1)
    if (o < tpr) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (tpr <= 32) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  __syncthreads();
  const int n = tpr >> 5, w0 = warp / n * n;
  float s = 0.f;
  for (int i = 0; i < n; ++i) s += red[w0 + i];  // the same order in every thread
  return s;
}

// 1 / sqrt(mean + eps), correctly rounded root and division
__device__ __forceinline__ float inv_rms(float ss, int D, float eps) { return 1.f / sqrtf(ss / (float)D + eps); }

// ---- forward, plain (FP8 = 0) or with the 8-bit output. Persistent CTAs: a team walks the rows, with the next row's
// loads in flight while this one is reduced and written, and keeps its columns' weights in registers (FLAT: the columns
// stay its own).
//
// 8 bits: group g of a row is channels [g G, (g + 1) G). FP8 = 1: a group is the chunks of `lanes` consecutive lanes (FLAT
// rows, a power of two of 32 chunks at most) and its maximum a shuffle. FP8 = 2: any G of 8 channels or more, a maximum per
// group in shared memory (integer maxima of non-negative floats: the order does not matter); a chunk touches two groups at
// most. A NaN counts in no maximum and comes out as e4m3's NaN.
template <typename T, int NV, bool FLAT, int FP8, int THREADS>
__global__ void __launch_bounds__(THREADS) rnorm_fwd(const T* __restrict__ x, const T* __restrict__ res,
                                                     const void* __restrict__ w, T* __restrict__ s, T* __restrict__ y,
                                                     uint8_t* __restrict__ q, float* __restrict__ scale, int wdtype,
                                                     float bias, long long rows, int D, int G, int lanes, int tpr,
                                                     float eps) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[2][32];
  extern __shared__ unsigned int tops[];  // FP8 = 2: [teams][groups] bit patterns
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const int groups = FP8 ? (D + G - 1) / G : 0;
  const long long step = (long long)gridDim.x * teams;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 a[NV], b[NV];
  auto fetch = [&](long long r) {
    const Row<T, FLAT> row(r, rows, D, sub, tpr);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      a[j] = row.live(j) ? row.load(x, row.at(j)) : zero;
      b[j] = res != nullptr && row.live(j) ? row.load(res, row.at(j)) : zero;
    }
  };
  long long base = (long long)blockIdx.x * teams;
  fetch(base + team);
  float wv[NV][E];
  if constexpr (FLAT) {
    const Row<T, FLAT> row(0, 1, D, sub, tpr);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (row.live(j)) row.weights(w, wdtype, bias, row.at(j), wv[j]);
  }
  for (int parity = 0; base < rows; base += step, parity ^= 1) {
    const long long r0 = base + team;
    const Row<T, FLAT> row(r0, rows, D, sub, tpr);
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
    const float r = inv_rms(team_sum(ss, tpr, red[parity]), D, eps);
    float top[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      top[j] = 0.f;
      if (!row.live(j)) continue;
      if constexpr (!FLAT) row.weights(w, wdtype, bias, row.at(j), wv[j]);
#pragma unroll
      for (int e = 0; e < E; ++e) v[j][e] = v[j][e] * r * wv[j][e];
      if constexpr (FP8 == 0) row.store(y, row.at(j), v[j]);
      if constexpr (FP8 == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) top[j] = fmaxf(top[j], fabsf(v[j][e]));
      }
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
      if constexpr (FP8 == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          for (int o = lanes >> 1; o >= 1; o >>= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
      }
      if constexpr (FP8 == 2) __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!row.live(j)) continue;
        const long long at = row.at(j);
        const int c0 = (int)(at - row.lo);
        uint32_t packed[E / 4];
        float sc = 1.f, sc2 = 1.f;  // 1 / scale: the product is within 2 units in the last place of y / scale
        int split = 1 << 30;
        if constexpr (FP8 == 1) {
          sc = top[j] > 0.f ? kE4m3Max / top[j] : 1.f;
          if ((sub & (lanes - 1)) == 0) scale[r0 * groups + c0 / G] = top[j] > 0.f ? top[j] / kE4m3Max : 1.f;
        } else {
          const int g0 = c0 > 0 ? c0 / G : 0;
          split = (g0 + 1) * G;
          const float t1 = __uint_as_float(tops[team * groups + g0]);
          sc = t1 > 0.f ? kE4m3Max / t1 : 1.f;
          if (g0 + 1 < groups) {
            const float t2 = __uint_as_float(tops[team * groups + g0 + 1]);
            sc2 = t2 > 0.f ? kE4m3Max / t2 : 1.f;
          }
        }
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] = v[j][4 * i + e] * (FP8 == 1 || c0 + 4 * i + e < split ? sc : sc2);
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
      if constexpr (FP8 == 2) {
        if (r0 < rows)
          for (int g = sub; g < groups; g += tpr) {
            const float t = __uint_as_float(tops[team * groups + g]);
            scale[r0 * groups + g] = t > 0.f ? t / kE4m3Max : 1.f;
          }
      }
    }
  }
}

// ---- backward. CTA p takes the blocks of R rows (R teams) p, p + grid, ...: every CTA has work to the end. With dw a
// FLAT thread keeps its columns' sums in registers (the columns stay its own over the rows) and the CTA's teams are
// added in team order; without FLAT the columns move with the row, so the sums stand in shared memory, where one thread
// adds to an element at a time, in the rows' order (one team a CTA).
template <typename T, int NV, bool FLAT, bool DW, int THREADS>
__global__ void __launch_bounds__(THREADS) rnorm_bwd(const T* __restrict__ s, const void* __restrict__ w,
                                                     const T* __restrict__ dy, const T* __restrict__ ds,
                                                     T* __restrict__ dx, float* __restrict__ part, int wdtype, float bias,
                                                     long long rows, int D, int tpr, float eps) {
  constexpr int E = Vec<T>::E;
  __shared__ float red[2][2][32];
  extern __shared__ __align__(16) float sums[];  // DW: [teams][D] (FLAT, at the end), or [D]
  const int teams = blockDim.x / tpr, team = threadIdx.x / tpr, sub = threadIdx.x % tpr;
  const long long step = (long long)gridDim.x * teams;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 nv[NV], ng[NV], nc[NV];  // the next row's s, dy, ds as they stand in memory
  auto fetch = [&](long long r) {
    const Row<T, FLAT> row(r, rows, D, sub, tpr);
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
  float acc[DW && FLAT ? NV : 1][E], wv[NV][E];
  if constexpr (FLAT) {
    const Row<T, FLAT> row(0, 1, D, sub, tpr);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) wv[j][e] = 0.f;
      if (row.live(j)) row.weights(w, wdtype, bias, row.at(j), wv[j]);
    }
  }
  if constexpr (DW) {
    if constexpr (FLAT) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[j][e] = 0.f;
    } else {
      for (int i = threadIdx.x; i < D; i += blockDim.x) sums[i] = 0.f;
      __syncthreads();
    }
  }
  for (int parity = 0; base < rows; base += step, parity ^= 1) {
    const Row<T, FLAT> row(base + team, rows, D, sub, tpr);
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
      if constexpr (!FLAT) row.weights(w, wdtype, bias, row.at(j), wv[j]);
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
      const int warp = threadIdx.x >> 5, n = tpr >> 5, w0 = warp / n * n;
      if ((threadIdx.x & 31) == 0) {
        red[parity][0][warp] = ss;
        red[parity][1][warp] = dot;
      }
      __syncthreads();
      ss = dot = 0.f;
      for (int i = 0; i < n; ++i) {
        ss += red[parity][0][w0 + i];
        dot += red[parity][1][w0 + i];
      }
    } else if constexpr (DW && !FLAT) {
      __syncthreads();  // the last row's sums are in place (one team: an element's adders take turns)
    }
    const float r = inv_rms(ss, D, eps);
    const float m = dot * r / (float)D;
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
        if constexpr (DW) {
          if constexpr (FLAT) acc[j][e] = fmaf(gf[e], xh, acc[j][e]);
          else if (row.mine(a + e)) sums[a - row.lo + e] += gf[e] * xh;
        }
      }
      row.store(dx, a, out);
    }
  }
  if constexpr (DW) {
    if constexpr (FLAT) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c0 = (sub + j * tpr) * E;
        if (c0 < D)
#pragma unroll
          for (int e = 0; e < E; ++e) sums[(size_t)team * D + c0 + e] = acc[j][e];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
      float t = sums[i];
      if constexpr (FLAT)
        for (int k = 1; k < teams; ++k) t += sums[(size_t)k * D + i];
      part[(size_t)blockIdx.x * D + i] = t;
    }
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

// The team: one chunk a thread (two past 1,024 threads): the next row's loads already double what is in flight. CTAs of
// 256 threads hold several teams of narrow rows, except where rows are too few to give every SM a CTA so.
Shape shape_of(long long rows, int D, int E, bool one_team) {
  Shape s;
  s.flat = D % E == 0;
  const int chunks = chunks_of(D, E);
  s.tpr = 4;
  while (s.tpr < 1024 && s.tpr < chunks) s.tpr *= 2;
  s.nv = s.tpr < chunks ? 2 : 1;
  s.threads = s.tpr > kThreads ? s.tpr : kThreads;
  if (one_team) s.threads = s.tpr;
  while (!one_team && s.threads > s.tpr && s.threads > 32 && rows * s.tpr / s.threads < kSms) s.threads /= 2;
  if (s.threads < 32) s.threads = s.tpr = 32;
  s.teams = s.threads / s.tpr;
  return s;
}
// persistent CTAs: as many as are resident at 64 registers a thread
int grid_of(long long rows, const Shape& s, int most = 1 << 30) {
  const long long blocks = (rows + s.teams - 1) / s.teams, resident = (long long)kSms * (1024 / s.threads);
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


// f(integral_constant NV, integral_constant THREADS): kernels of up to 256 threads get more registers each
template <typename F>
int with_shape(const Shape& s, F&& f) {
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (s.nv == 2) return f(Two{}, std::integral_constant<int, 1024>{});
  return s.threads <= 256 ? f(One{}, std::integral_constant<int, 256>{}) : f(One{}, std::integral_constant<int, 1024>{});
}

template <int FP8>
int forward(const void* x, const void* res, const void* w, void* s, void* y, void* q, float* scale, int dtype, int wdtype,
            int zero_centered, long long rows, int D, int G, int lanes, const Shape& sh, size_t smem, float eps,
            void* stream) {
  const int grid = grid_of(rows, sh);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_shape(sh, [&](auto nv, auto threads) {
      constexpr int NV = decltype(nv)::value, TH = decltype(threads)::value;
      auto k = rnorm_fwd<T, NV, true, FP8, TH>;
      if constexpr (FP8 != 1)
        if (!sh.flat) k = rnorm_fwd<T, NV, false, FP8, TH>;
      k<<<grid, sh.threads, smem, static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(x), static_cast<const T*>(res), w, static_cast<T*>(s), static_cast<T*>(y),
          static_cast<uint8_t*>(q), scale, wdtype, zero_centered ? 1.f : 0.f, rows, D, G, lanes, sh.tpr, eps);
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
  const int groups = (D + G - 1) / G, lanes = groups == 1 ? sh.tpr : G / E;
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
  const int grid = grid_of(rows, sh, dw != nullptr ? kMaxPartials : 1 << 30);
  const float bias = zero_centered ? 1.f : 0.f;
  float* part = static_cast<float*>(workspace);
  const size_t smem = dw == nullptr ? 0 : (size_t)(sh.flat ? sh.teams : 1) * D * sizeof(float);
  int st = with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_shape(sh, [&](auto nv, auto threads) {
      constexpr int NV = decltype(nv)::value, TH = decltype(threads)::value;
      auto k = dw != nullptr ? (sh.flat ? rnorm_bwd<T, NV, true, true, TH> : rnorm_bwd<T, NV, false, true, TH>)
                             : (sh.flat ? rnorm_bwd<T, NV, true, false, TH> : rnorm_bwd<T, NV, false, false, TH>);
      if (smem > 48 * 1024 &&
          cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return (cudaGetLastError(), GD_ERR_LAUNCH);
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
