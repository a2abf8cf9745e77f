// The gated delta rule's recurrent form, for single tokens and short runs over kept states. For each request and value head,
// with the state S [DK, DV] in fp32, token after token:
//   S <- exp(g) S,   d = beta (v - S^T k),   S <- S + k d^T,   o = S^T q
// (q and k l2-normalised where asked, q scaled by DK^-1/2). Both products with the state are taken before d is known:
//   o = exp(g) (S^T q) + (q . k) d,
// so a token costs one pass over S in registers and one join over the rows.
//
// Bound by memory: 8 DK DV bytes of a head's state for about 7 DK DV operations a token. The state is read once into registers,
// run through all tokens of the call, and written once. The recurrence never mixes value columns, so a warp has 2,048 / ROWS
// columns of a head with all their rows (ROWS: 64, 128 or 256, at least DK; a lane four adjacent columns of every RG-th row, 16 in
// all), and its sums need no other warp. The order of the sums goes by DK alone: a token has the same bits in a run or alone,
// whatever the other requests are. What decides is how many bytes are on their way, that is, how many warps with 64 registers of
// state an SM holds: 16 of up to 128 registers. The compiler would keep the k of all rows from the sums for the update (16 registers
// more; with spills a single token of 128 requests took 91 to 125 us); read again through a volatile pointer they cost nothing.
// Square heads have their strides as constants (128 requests: 83 us, else 87; 64 requests x 32 heads, 4 tokens: 64, else 71).
//   token_kernel: single tokens. 125 live of 128 requests x 32 heads of 128 x 128: 83 us, 6.35 TB/s (a plain copy of the states:
// 81 us); 8 requests: 7.5 us; 1 request: 3.4 us. (Persistent warps with the next states on their way by TMA took 99 us: 96 KB an SM
// under way where this one has 128; a persistent form of this one took 91, five CTAs an SM, which spill, 86.)
//   run_kernel: runs of tokens. The four warps of a CTA prepare the tokens' q and k together, up to eight at a time, while the state
// is on its way; the token loop has no barrier. 24 requests x 16 heads of 128 x 128, 6 tokens: 19 us: 10 us of memory, then the
// packed multiply-adds, about 1.5 us a token; 768 CTAs are 1.3 turns of the 592 that run at once.
#include <cstdint>

#include "gd_common.cuh"
#include "gd_wattn.cuh"

namespace gd {
namespace rule_step {
namespace {

using wattn::F2;
using wattn::f2;
using wattn::fma2;
using wattn::mul2;
using wattn::unf2;

constexpr int kMaxWidth = 256;  // DK, DV
constexpr int kWarps = 4;       // of a CTA, at most
constexpr int kThreads = 32 * kWarps;
constexpr int kCtas = 4;        // an SM
constexpr int kRun = 8;         // tokens prepared at a time

struct Args {
  const void *q, *k, *v;  // [B, T, HK, DK], [B, T, HK, DK], [B, T, H, DV]
  const float *g, *beta;  // [B, T, H]
  const float* s_in;      // [S, H, DK, DV] (NULL: zeros)
  float* s_out;           // the same (NULL: not kept)
  const int *in, *out;    // [B] slots read and written (NULL: b)
  void* o;                // [B, T, H, DV]
  int B, T, H, HK, DK, DV, slots;
  bool l2norm;
};

// Four adjacent values as loaded.
template <typename T>
struct Four {
  uint2 u;
  Four() = default;
  __device__ __forceinline__ explicit Four(const T* p) { load(p); }
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void get(float (&v)[4]) const {
    const float2 a = wattn::unpack16<T>(u.x), b = wattn::unpack16<T>(u.y);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
};
template <>
struct Four<float> {
  float4 u;
  Four() = default;
  __device__ __forceinline__ explicit Four(const float* p) { load(p); }
  __device__ __forceinline__ void load(const float* p) { u = __ldg(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w; }
};
template <typename T>
__device__ __forceinline__ void put4(T* p, float a, float b, float c, float d) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
  else *reinterpret_cast<uint2*>(p) = make_uint2(wattn::pack16<T>(a, b), wattn::pack16<T>(c, d));
}

template <typename T, typename TV, int ROWS, bool SQUARE>
__global__ void __launch_bounds__(kThreads, kCtas) run_kernel(const Args a) {
  constexpr int COLS = 2048 / ROWS, LC = COLS / 4, RG = 32 / LC, R = 16;  // a warp's columns, lanes across them, row groups, rows a lane
  constexpr int kParts = (ROWS + 127) / 128;                              // of a row of q or k, 128 values each
  // a token's k and q, normalised, each twice (operands of the packed arithmetic), and its decay, beta, q k
  __shared__ __align__(16) float4 kq[kRun][ROWS];
  __shared__ float scalars[kRun][4];
  const int DK = SQUARE ? ROWS : a.DK, DV = SQUARE ? ROWS : a.DV;
  const int warps = SQUARE ? (ROWS / COLS < kWarps ? ROWS / COLS : kWarps) : blockDim.x >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = lane % LC, rg = lane / LC;
  const int per = DV / (COLS * warps), b = blockIdx.y, h = blockIdx.x / per;
  const int col = ((blockIdx.x - h * per) * warps + warp) * COLS + cl * 4;
  const int hk = h / (a.H / a.HK);
  const int from = a.in == nullptr ? b : __ldg(a.in + b), to = a.out == nullptr ? b : __ldg(a.out + b);
  T* const o = static_cast<T*>(a.o) + ((long long)b * a.T * a.H + h) * DV + col;
  const long long o_step = (long long)a.H * DV;
  auto fill = [&](float x) {
    for (int t = rg; t < a.T; t += RG) put4<T>(o + t * o_step, x, x, x, x);
  };
  // an idle request gives zeros; one whose slot does not exist, or that another request writes or reads, gives NaN; neither
  // touches the states
  if (from < 0 || to < 0) return fill(0.f);
  if (from >= a.slots || to >= a.slots) return fill(NAN);

  F2 s[R][2];
  const long long step = (long long)RG * DV;
  const float* src = a.s_in + (((long long)a.H * from + h) * DK + rg) * DV + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.s_in != nullptr && (SQUARE || i * RG + rg < DK)) x = __ldcs(reinterpret_cast<const float4*>(src));
    src += step;
    s[i][0] = f2(x.x, x.y);
    s[i][1] = f2(x.z, x.w);
  }
  // (while the state is on its way) does another request read or write the slot that this one writes?
  bool hit = false;
  if (a.out != nullptr)
    for (int j = threadIdx.x; j < a.B; j += blockDim.x)
      if (j != b) {
        const int x = __ldg(a.in + j), y = __ldg(a.out + j);
        // (an idle request does neither, nor does one whose slot does not exist)
        hit |= (unsigned)x < (unsigned)a.slots && (unsigned)y < (unsigned)a.slots && (x == to || y == to);
      }

  const float scale = rsqrtf((float)DK);
  for (int t0 = 0; t0 < a.T; t0 += kRun) {
    const int n = a.T - t0 < kRun ? a.T - t0 : kRun;
    if (t0 > 0) __syncthreads();  // the tokens before are read
    for (int j = warp; j < n; j += warps) {
      const long long row = (long long)b * a.T + t0 + j, key = (row * a.HK + hk) * DK + lane * 4;
      float q[kParts][4], k[kParts][4], kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
      for (int x = 0; x < kParts; ++x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[x][i] = k[x][i] = 0.f;
        if (lane * 4 + 128 * x < DK) {
          Four<T>(static_cast<const T*>(a.q) + key + 128 * x).get(q[x]);
          Four<T>(static_cast<const T*>(a.k) + key + 128 * x).get(k[x]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kk = fmaf(k[x][i], k[x][i], kk);
          qq = fmaf(q[x][i], q[x][i], qq);
          qk = fmaf(q[x][i], k[x][i], qk);
        }
      }
      qk = warp_sum(qk);
      float fk = 1.f, fq = scale;
      if (a.l2norm) {
        fk = rsqrtf(warp_sum(kk) + 1e-6f);
        fq *= rsqrtf(warp_sum(qq) + 1e-6f);
      }
#pragma unroll
      for (int x = 0; x < kParts; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane * 4 + i + 128 * x < ROWS)
            kq[j][lane * 4 + i + 128 * x] = make_float4(k[x][i] * fk, k[x][i] * fk, q[x][i] * fq, q[x][i] * fq);
      if (lane == 0) {
        scalars[j][0] = expf(__ldg(a.g + row * a.H + h));
        scalars[j][1] = __ldg(a.beta + row * a.H + h);
        scalars[j][2] = qk * fk * fq;
      }
    }
    const TV* const vp = static_cast<const TV*>(a.v) + (((long long)b * a.T + t0) * a.H + h) * DV + col;
    Four<TV> v_next(vp);
    if (__syncthreads_or(hit)) return fill(NAN);
    for (int j = 0; j < n; ++j) {
      float v[4];
      v_next.get(v);
      if (j + 1 < n) v_next.load(vp + (j + 1) * o_step);
      F2 pk0 = f2(0.f, 0.f), pk1 = pk0, pq0 = pk0, pq1 = pk0;
#pragma unroll
      for (int i = 0; i < R; ++i) {  // (zeros past DK)
        const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&kq[j][i * RG + rg]);
        pk0 = fma2(w.x, s[i][0], pk0);
        pk1 = fma2(w.x, s[i][1], pk1);
        pq0 = fma2(w.y, s[i][0], pq0);
        pq1 = fma2(w.y, s[i][1], pq1);
      }
      float pk[4], pq[4];
      unf2(pk0, pk[0], pk[1]);
      unf2(pk1, pk[2], pk[3]);
      unf2(pq0, pq[0], pq[1]);
      unf2(pq1, pq[2], pq[3]);
#pragma unroll
      for (int m = LC; m < 32; m *= 2) {  // the row groups
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pk[i] += __shfl_xor_sync(0xffffffffu, pk[i], m);
          pq[i] += __shfl_xor_sync(0xffffffffu, pq[i], m);
        }
      }
      const float decay = scalars[j][0], beta = scalars[j][1];
      float d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = beta * (v[i] - decay * pk[i]);
      if (rg == 0) {
        const float f = scalars[j][2];
        put4<T>(o + (t0 + j) * o_step, fmaf(f, d[0], decay * pq[0]), fmaf(f, d[1], decay * pq[1]), fmaf(f, d[2], decay * pq[2]),
                fmaf(f, d[3], decay * pq[3]));
      }
      const F2 d0 = f2(d[0], d[1]), d1 = f2(d[2], d[3]), e = f2(decay, decay);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const F2 w = *reinterpret_cast<const volatile F2*>(&kq[j][i * RG + rg]);
        s[i][0] = fma2(w, d0, mul2(e, s[i][0]));
        s[i][1] = fma2(w, d1, mul2(e, s[i][1]));
      }
    }
  }
  if (a.T == 0 && __syncthreads_or(hit)) return;
  if (a.s_out == nullptr) return;
  float* dst = a.s_out + (((long long)a.H * to + h) * DK + rg) * DV + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float4 x;
    unf2(s[i][0], x.x, x.y);
    unf2(s[i][1], x.z, x.w);
    if (SQUARE || i * RG + rg < DK) __stcs(reinterpret_cast<float4*>(dst), x);
    dst += step;
  }
}

template <typename T, typename TV, int ROWS, bool SQUARE>
__global__ void __launch_bounds__(kThreads, kCtas) token_kernel(const Args a) {
  constexpr int COLS = 2048 / ROWS, LC = COLS / 4, RG = 32 / LC, R = 16;
  constexpr int kParts = (ROWS + 127) / 128;
  __shared__ __align__(16) float2 kq[ROWS];                               // the token's k and q, normalised
  const int DK = SQUARE ? ROWS : a.DK, DV = SQUARE ? ROWS : a.DV;
  const int warps = SQUARE ? (ROWS / COLS < kWarps ? ROWS / COLS : kWarps) : blockDim.x >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = lane % LC, rg = lane / LC;
  const int per = DV / (COLS * warps), b = blockIdx.y, h = blockIdx.x / per;
  const int col = ((blockIdx.x - h * per) * warps + warp) * COLS + cl * 4;
  const int from = a.in == nullptr ? b : __ldg(a.in + b), to = a.out == nullptr ? b : __ldg(a.out + b);
  const long long row = (long long)b * a.H + h, step = (long long)RG * DV;
  T* const o = static_cast<T*>(a.o) + row * DV + col;
  // an idle request gives zeros; one whose slot does not exist, or that another request writes or reads, gives NaN
  if (from < 0 || to < 0 || from >= a.slots || to >= a.slots) {
    const float x = from < 0 || to < 0 ? 0.f : NAN;
    if (rg == 0) put4<T>(o, x, x, x, x);
    return;
  }
  float4 s[R];
  const float* src = a.s_in + (((long long)a.H * from + h) * DK + rg) * DV + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.s_in != nullptr && (SQUARE || i * RG + rg < DK)) s[i] = __ldcs(reinterpret_cast<const float4*>(src));
    src += step;
  }
  // (while the state is on its way)
  const long long key = ((long long)b * a.HK + h / (a.H / a.HK)) * DK + lane * 4;
  float q[kParts][4], k[kParts][4], kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
  for (int x = 0; x < kParts; ++x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[x][i] = k[x][i] = 0.f;
    if (lane * 4 + 128 * x < DK) {
      Four<T>(static_cast<const T*>(a.q) + key + 128 * x).get(q[x]);
      Four<T>(static_cast<const T*>(a.k) + key + 128 * x).get(k[x]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kk = fmaf(k[x][i], k[x][i], kk);
      qq = fmaf(q[x][i], q[x][i], qq);
      qk = fmaf(q[x][i], k[x][i], qk);
    }
  }
  const Four<TV> v4(static_cast<const TV*>(a.v) + row * DV + col);
  const float decay = expf(__ldg(a.g + row)), beta = __ldg(a.beta + row);
  qk = warp_sum(qk);
  float fk = 1.f, fq = rsqrtf((float)DK);
  if (a.l2norm) {
    fk = rsqrtf(warp_sum(kk) + 1e-6f);
    fq *= rsqrtf(warp_sum(qq) + 1e-6f);
  }
  // (all warps have the sums; each writes its share of the lanes)
#pragma unroll
  for (int x = 0; x < kParts; ++x)
    if (lane % warps == warp && lane * 4 + 128 * x < ROWS) {
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        *reinterpret_cast<float4*>(kq + lane * 4 + 128 * x + i) =
            make_float4(k[x][i] * fk, q[x][i] * fq, k[x][i + 1] * fk, q[x][i + 1] * fq);
    }
  bool hit = false;  // does another request read or write the slot that this one writes?
  if (a.out != nullptr)
    for (int j = threadIdx.x; j < a.B; j += blockDim.x)
      if (j != b) {
        const int x = __ldg(a.in + j), y = __ldg(a.out + j);
        // (an idle request does neither, nor does one whose slot does not exist)
        hit |= (unsigned)x < (unsigned)a.slots && (unsigned)y < (unsigned)a.slots && (x == to || y == to);
      }
  if (__syncthreads_or(hit)) {
    if (rg == 0) put4<T>(o, NAN, NAN, NAN, NAN);
    return;
  }
  float pk[4] = {0.f, 0.f, 0.f, 0.f}, pq[4] = {0.f, 0.f, 0.f, 0.f}, v[4], d[4];
#pragma unroll
  for (int i = 0; i < R; ++i) {  // (zeros past DK)
    const float2 w = kq[i * RG + rg];
    const float x[4] = {s[i].x, s[i].y, s[i].z, s[i].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      pk[c] = fmaf(w.x, x[c], pk[c]);
      pq[c] = fmaf(w.y, x[c], pq[c]);
    }
  }
#pragma unroll
  for (int m = LC; m < 32; m *= 2) {  // the row groups
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pk[i] += __shfl_xor_sync(0xffffffffu, pk[i], m);
      pq[i] += __shfl_xor_sync(0xffffffffu, pq[i], m);
    }
  }
  v4.get(v);
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = beta * (v[i] - decay * pk[i]);
  if (rg == 0) {
    const float f = qk * fk * fq;
    put4<T>(o, fmaf(f, d[0], decay * pq[0]), fmaf(f, d[1], decay * pq[1]), fmaf(f, d[2], decay * pq[2]),
            fmaf(f, d[3], decay * pq[3]));
  }
  if (a.s_out == nullptr) return;
  float* dst = a.s_out + (((long long)a.H * to + h) * DK + rg) * DV + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    // (read again: kept from above, the k of all rows would cost 16 registers, and a CTA an SM)
    const float w = *const_cast<const volatile float*>(&kq[i * RG + rg].x);
    if (SQUARE || i * RG + rg < DK)
      __stcs(reinterpret_cast<float4*>(dst),
             make_float4(fmaf(w, d[0], decay * s[i].x), fmaf(w, d[1], decay * s[i].y), fmaf(w, d[2], decay * s[i].z),
                         fmaf(w, d[3], decay * s[i].w)));
    dst += step;
  }
}

template <typename T, typename TV, int ROWS>
int launch_rows(const Args& a, cudaStream_t stream) {
  const int parts = a.DV * ROWS / 2048;  // a head's warps; its CTAs, all of one size
  int ctas = (parts + kWarps - 1) / kWarps;
  while (parts % ctas) ++ctas;
  const dim3 grid((unsigned)(a.H * ctas), (unsigned)a.B);
  const int threads = 32 * (parts / ctas);
  const bool square = a.DK == ROWS && a.DV == ROWS;
  if (a.T == 1)
    square ? token_kernel<T, TV, ROWS, true><<<grid, threads, 0, stream>>>(a)
           : token_kernel<T, TV, ROWS, false><<<grid, threads, 0, stream>>>(a);
  else
    square ? run_kernel<T, TV, ROWS, true><<<grid, threads, 0, stream>>>(a)
           : run_kernel<T, TV, ROWS, false><<<grid, threads, 0, stream>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, typename TV>
int launch(const Args& a, cudaStream_t stream) {
  return a.DK <= 64    ? launch_rows<T, TV, 64>(a, stream)
         : a.DK <= 128 ? launch_rows<T, TV, 128>(a, stream)
                       : launch_rows<T, TV, 256>(a, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace rule_step
}  // namespace gd

extern "C" int gd_rule_step(const void* q, const void* k, const void* v, const float* g, const float* beta,
                            const float* s_in, float* s_out, const int* slots, const int* out_slots, void* o, int dtype,
                            int vdtype, int B, int T, int H, int HK, int DK, int DV, int n_slots, int flags, void* stream) {
  using namespace gd::rule_step;
  if ((dtype != GD_FLOAT32 && dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) || (vdtype != dtype && vdtype != GD_FLOAT32) ||
      (flags & ~GD_L2NORM))
    return GD_ERR_ARG;
  if (B < 0 || B > 65535 || T < 0 || H <= 0 || HK <= 0 || H % HK != 0 || H > (1 << 24) || n_slots < 0 ||
      (long long)n_slots * H >= (1ll << 31) || DK <= 0 || DK % 32 != 0 || DK > kMaxWidth || DV <= 0 || DV % 32 != 0 ||
      DV > kMaxWidth || (slots == nullptr && n_slots < B))
    return GD_ERR_SHAPE;
  if (B == 0) return GD_OK;
  if ((slots == nullptr) != (out_slots == nullptr)) return GD_ERR_ARG;
  if (T > 0 && (q == nullptr || k == nullptr || v == nullptr || g == nullptr || beta == nullptr || o == nullptr))
    return GD_ERR_ARG;
  for (const void* p : {q, k, v, (const void*)s_in, (const void*)s_out, (const void*)o})
    if (!aligned16(p)) return GD_ERR_ALIGN;
  Args a;
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.s_in = s_in, a.s_out = s_out, a.in = slots, a.out = out_slots;
  a.o = o, a.B = B, a.T = T, a.H = H, a.HK = HK, a.DK = DK, a.DV = DV, a.slots = n_slots;
  a.l2norm = (flags & GD_L2NORM) != 0;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (dtype == GD_FLOAT32) return launch<float, float>(a, cs);
  if (dtype == GD_FLOAT16) return vdtype == dtype ? launch<__half, __half>(a, cs) : launch<__half, float>(a, cs);
  return vdtype == dtype ? launch<__nv_bfloat16, __nv_bfloat16>(a, cs) : launch<__nv_bfloat16, float>(a, cs);
}
