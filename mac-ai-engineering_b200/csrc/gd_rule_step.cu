// The gated delta rule's recurrent form, for single tokens and short runs over kept states. For each request and value head,
// with the state S [DK, DV] in fp32, token after token:
//   S <- exp(g) S,   d = beta (v - S^T k),   S <- S + k d^T,   o = S^T q
// (q and k l2-normalised where asked, q scaled by DK^-1/2). Both products with the state are taken before d is known:
//   o = exp(g) (S^T q) + (q . k) d,
// so a token costs one pass over S in registers and one join over the rows.
//
// Bound by memory: 8 DK DV bytes of a head's state for about 7 DK DV operations a token. The state is read once into registers,
// run through all tokens of the call, and written once. The recurrence never mixes value columns, so a warp has COLS columns of a
// head with all their rows (a lane four adjacent columns of every 128 / COLS-th row), and its sums need no other warp. Two kernels:
//   run_kernel: runs of tokens, and few heads. The four warps of a CTA prepare the tokens' q and k together, up to eight at a time,
// while the state is on its way; the token loop has no barrier. 24 requests x 16 heads of 128 x 128, 6 tokens: 22 us (bound by the
// packed multiply-adds and their operands from shared memory: about 2 us a token, after 10 us of memory); 1 request x 32 heads, 1
// token: 4.2 us with 8 columns a warp (16: 4.8, 32: 6.9), latency.
//   token_kernel: one token of many heads. Persistent warps walk the (request, head, columns) items; while a warp works on one in
// registers, TMA brings the next one's columns into the warp's stage of shared memory, and its rows of q, k, v into registers.
// 125 live of 128 requests x 32 heads of 128 x 128: 99 us, 5.3 TB/s (run_kernel: 122 us; a plain copy of the states: 83 us; this
// kernel without its arithmetic: 96 us, so that the memory's order of reads and writes is what is left). 8 requests: 10.3 us
// (run_kernel 11.6).
#include <cstdint>

#include "gd_common.cuh"
#include "gd_wattn.cuh"

namespace gd {
namespace rule_step {
namespace {

using wattn::F2;
using wattn::add2;
using wattn::f2;
using wattn::fma2;
using wattn::mul2;
using wattn::unf2;

constexpr int kMaxWidth = 256;  // DK, DV
constexpr int kRunWarps = 4;
constexpr int kRunThreads = 32 * kRunWarps;
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

// ROWS: 64, 128 or 256, at least DK; COLS: columns of a warp.
template <typename T, typename TV, int ROWS, int COLS>
__global__ void __launch_bounds__(kRunThreads, ROWS > 128 ? 2 : 3) run_kernel(const Args a) {
  constexpr int LC = COLS / 4, RG = 32 / LC, R = ROWS / RG;  // lanes across the columns, row groups, rows a lane has
  constexpr int kParts = (ROWS + 127) / 128;                 // of a row of q or k, 128 values each
  // a token's k and q, normalised, each twice (operands of the packed arithmetic), and its decay, beta, q k
  __shared__ __align__(16) float4 kq[kRun][ROWS];
  __shared__ float scalars[kRun][4];
  const int slices = (a.DV + kRunWarps * COLS - 1) / (kRunWarps * COLS);
  const int b = blockIdx.y, h = blockIdx.x / slices;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = lane % LC, rg = lane / LC;
  const int c0 = ((blockIdx.x - h * slices) * kRunWarps + warp) * COLS, col = c0 + cl * 4;
  const bool mine = c0 < a.DV;  // (DV is a multiple of 32)
  const int hk = h / (a.H / a.HK);
  const int from = a.in == nullptr ? b : __ldg(a.in + b), to = a.out == nullptr ? b : __ldg(a.out + b);
  T* const o = static_cast<T*>(a.o) + ((long long)b * a.T * a.H + h) * a.DV + col;
  const long long o_step = (long long)a.H * a.DV;
  auto fill = [&](float x) {
    if (mine)
      for (int t = rg; t < a.T; t += RG) put4<T>(o + t * o_step, x, x, x, x);
  };
  // an idle request gives zeros; one whose slot does not exist, or that another request writes or reads, gives NaN; neither
  // touches the states
  if (from < 0 || to < 0) return fill(0.f);
  if (from >= a.slots || to >= a.slots) return fill(NAN);

  F2 s[R][2];
  const long long head = ((long long)a.H * from + h) * a.DK;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = i * RG + rg;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.s_in != nullptr && mine && r < a.DK) x = __ldcs(reinterpret_cast<const float4*>(a.s_in + (head + r) * a.DV + col));
    s[i][0] = f2(x.x, x.y);
    s[i][1] = f2(x.z, x.w);
  }
  // (while the state is on its way) does another request read or write the slot that this one writes?
  bool hit = false;
  if (a.out != nullptr)
    for (int j = threadIdx.x; j < a.B; j += kRunThreads)
      if (j != b) {
        const int x = __ldg(a.in + j), y = __ldg(a.out + j);
        hit |= x >= 0 && y >= 0 && (x == to || y == to);  // (an idle request does neither)
      }

  const float scale = rsqrtf((float)a.DK);
  for (int t0 = 0; t0 < a.T; t0 += kRun) {
    const int n = a.T - t0 < kRun ? a.T - t0 : kRun;
    if (t0 > 0) __syncthreads();  // the tokens before are read
    for (int j = warp; j < n; j += kRunWarps) {
      const long long row = (long long)b * a.T + t0 + j, key = (row * a.HK + hk) * a.DK + lane * 4;
      float q[kParts][4], k[kParts][4], kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
      for (int x = 0; x < kParts; ++x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[x][i] = k[x][i] = 0.f;
        if (lane * 4 + 128 * x < a.DK) {
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
    const TV* const vp = static_cast<const TV*>(a.v) + (((long long)b * a.T + t0) * a.H + h) * a.DV + col;
    Four<TV> v_next;
    if (mine) v_next.load(vp);
    if (__syncthreads_or(hit)) return fill(NAN);
    if (!mine) continue;
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
        const F2 w = *reinterpret_cast<const F2*>(&kq[j][i * RG + rg]);
        s[i][0] = fma2(w, d0, mul2(e, s[i][0]));
        s[i][1] = fma2(w, d1, mul2(e, s[i][1]));
      }
    }
  }
  if (a.T == 0 && __syncthreads_or(hit)) return;
  if (a.s_out == nullptr || !mine) return;
  float* const dst = a.s_out + (((long long)a.H * to + h) * a.DK + rg) * a.DV + col;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float4 x;
    unf2(s[i][0], x.x, x.y);
    unf2(s[i][1], x.z, x.w);
    if (i * RG + rg < a.DK) __stcs(reinterpret_cast<float4*>(dst + (long long)i * RG * a.DV), x);
  }
}

// ROWS: 64, 128 or 256, at least DK; COLS: columns of an item.
template <int ROWS, int COLS>
struct Cfg {
  static constexpr int LC = COLS / 4, RG = 32 / LC, R = ROWS / RG;  // lanes across the columns, row groups, rows a lane has
  static constexpr int kParts = (ROWS + 127) / 128;                 // of a row of q or k, 128 values each
  static constexpr int kStage = ROWS * COLS * 4, kWarp = kStage + ROWS * 8;
  static constexpr int kFit = 220 * 1024 / kWarp, kMost = R <= 16 ? 12 : 8, kWarps = kFit > kMost ? kMost : kFit;
  static constexpr size_t kSmem = 128 + (size_t)kWarps * kWarp;
};

enum Kind { kLive, kIdle, kBad };
struct Item {
  int b, h, c0, from, to, kind;
};

template <typename T, typename TV, int ROWS, int COLS>
__global__ void __launch_bounds__(32 * Cfg<ROWS, COLS>::kWarps, 1)
    token_kernel(const __grid_constant__ CUtensorMap map, const Args a) {
  using C = Cfg<ROWS, COLS>;
  constexpr int LC = C::LC, RG = C::RG, R = C::R, kWarps = C::kWarps;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cl = lane % LC, rg = lane / LC;
  uint8_t* const own =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)) + warp * C::kWarp;
  float4* const stage = reinterpret_cast<float4*>(own) + rg * LC + cl;  // the lane's first row
  float2* const kq = reinterpret_cast<float2*>(own + C::kStage);        // a token's k and q, normalised
  uint64_t* const bar = bars + warp;
  if (lane == 0) {
    mbar_init(bar, 1);
    fence_mbar_init();
  }
  for (int i = lane; i < ROWS * COLS / 4; i += 32) reinterpret_cast<float4*>(own)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = lane; i < ROWS; i += 32) kq[i] = make_float2(0.f, 0.f);
  __syncwarp();

  const int slices = a.DV / COLS;
  const long long items = (long long)a.B * a.H * slices;
  // a CTA's items lie together and its warps take them in turn: neighbours read and write the same rows at about the same time
  const long long end = items * (blockIdx.x + 1) / gridDim.x;
  long long at = items * blockIdx.x / gridDim.x + warp;
  if (at >= end) return;

  int checked = -1, from = 0, to = 0, kind = kLive;  // the request whose slots these are
  auto plan = [&](long long i) {
    const long long r = i / slices;
    Item it;
    it.c0 = (int)(i - r * slices) * COLS;
    it.b = (int)(r / a.H);
    it.h = (int)(r - (long long)it.b * a.H);
    if (it.b != checked) {
      checked = it.b;
      from = a.in == nullptr ? it.b : __ldg(a.in + it.b);
      to = a.out == nullptr ? it.b : __ldg(a.out + it.b);
      kind = from < 0 || to < 0 ? kIdle : from >= a.slots || to >= a.slots ? kBad : kLive;
      if (kind == kLive && a.out != nullptr) {  // does another request read or write the slot that this one writes?
        bool hit = false;
        for (int j = lane; j < a.B; j += 32)
          if (j != it.b) {
            const int x = __ldg(a.in + j), y = __ldg(a.out + j);
            hit |= x >= 0 && y >= 0 && (x == to || y == to);  // (an idle request does neither)
          }
        if (__any_sync(0xffffffffu, hit)) kind = kBad;
      }
    }
    it.from = from, it.to = to, it.kind = kind;
    return it;
  };
  const bool reads = a.s_in != nullptr, writes = a.s_out != nullptr;
  auto fetch = [&](const Item& it) {  // when the stage is read
    if (it.kind != kLive || !reads) return;
    fence_async_smem();
    __syncwarp();
    if (lane != 0) return;
    mbar_arrive_expect_tx(bar, a.DK * COLS * 4);
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(own)),
        "l"(reinterpret_cast<uint64_t>(&map)), "r"(it.c0), "r"(0), "r"(it.from * a.H + it.h), "r"(smem_u32(bar))
        : "memory");
  };
  // the next item's rows: values of q and k a lane, v for the lane's columns
  Four<T> q4[C::kParts], k4[C::kParts];
  Four<TV> v4;
  float g1 = 0.f, b1 = 0.f;
  auto rows = [&](const Item& it) {
    const long long row = it.b, key = (row * a.HK + it.h / (a.H / a.HK)) * a.DK + lane * 4;
#pragma unroll
    for (int j = 0; j < C::kParts; ++j)
      if (lane * 4 + 128 * j < a.DK) {
        q4[j].load(static_cast<const T*>(a.q) + key + 128 * j);
        k4[j].load(static_cast<const T*>(a.k) + key + 128 * j);
      }
    v4.load(static_cast<const TV*>(a.v) + (row * a.H + it.h) * a.DV + it.c0 + cl * 4);
    g1 = __ldg(a.g + row * a.H + it.h);
    b1 = __ldg(a.beta + row * a.H + it.h);
  };

  const float scale = rsqrtf((float)a.DK);
  uint32_t phase = 0;
  Item next = plan(at);
  fetch(next);
  rows(next);
  for (; at < end; at += kWarps) {
    const Item it = next;
    const bool more = at + kWarps < end;
    if (more) next = plan(at + kWarps);
    T* const o = static_cast<T*>(a.o) + ((long long)it.b * a.H + it.h) * a.DV + it.c0 + cl * 4;
    if (it.kind != kLive) {
      // an idle request gives zeros; one whose slot does not exist, or that another request writes or reads, gives NaN
      const float x = it.kind == kIdle ? 0.f : NAN;
      if (rg == 0) put4<T>(o, x, x, x, x);
      if (more) fetch(next);
      if (more) rows(next);
    } else {
      F2 s[R][2];
#pragma unroll
      for (int i = 0; i < R; ++i) s[i][0] = s[i][1] = f2(0.f, 0.f);
      if (reads) {
        const bool ok = mbar_wait(bar, phase, nullptr, 0);
        phase ^= 1;
#pragma unroll
        for (int i = 0; i < R; ++i) {  // (zeros past DK)
          const float4 x = stage[i * RG * LC];
          s[i][0] = f2(x.x, x.y);
          s[i][1] = f2(x.z, x.w);
        }
        if (!ok) s[0][0] = s[0][1] = f2(NAN, NAN);  // a wait that gave up leaves NaN
      }
      if (more) fetch(next);
      float q[C::kParts][4], k[C::kParts][4], v[4];
      float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
      for (int j = 0; j < C::kParts; ++j) {
        q4[j].get(q[j]);
        k4[j].get(k[j]);
        const bool in = lane * 4 + 128 * j < a.DK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          k[j][i] = in ? k[j][i] : 0.f;
          q[j][i] = in ? q[j][i] : 0.f;
          kk = fmaf(k[j][i], k[j][i], kk);
          qq = fmaf(q[j][i], q[j][i], qq);
          qk = fmaf(q[j][i], k[j][i], qk);
        }
      }
      v4.get(v);
      const float decay = expf(g1), beta = b1;
      if (more) rows(next);
      qk = warp_sum(qk);
      float fk = 1.f, fq = scale;
      if (a.l2norm) {
        fk = rsqrtf(warp_sum(kk) + 1e-6f);
        fq *= rsqrtf(warp_sum(qq) + 1e-6f);
      }
      __syncwarp();  // the rows of the item before are read
#pragma unroll
      for (int j = 0; j < C::kParts; ++j)
        if (lane * 4 + 128 * j < a.DK) {
#pragma unroll
          for (int i = 0; i < 4; i += 2)
            *reinterpret_cast<float4*>(kq + lane * 4 + 128 * j + i) =
                make_float4(k[j][i] * fk, q[j][i] * fq, k[j][i + 1] * fk, q[j][i + 1] * fq);
        }
      __syncwarp();
      F2 pk0 = f2(0.f, 0.f), pk1 = pk0, pq0 = pk0, pq1 = pk0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float2 w = kq[i * RG + rg];
        const F2 kx = f2(w.x, w.x), qx = f2(w.y, w.y);
        pk0 = fma2(kx, s[i][0], pk0);
        pk1 = fma2(kx, s[i][1], pk1);
        pq0 = fma2(qx, s[i][0], pq0);
        pq1 = fma2(qx, s[i][1], pq1);
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
      float d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = beta * (v[i] - decay * pk[i]);
      if (rg == 0) {
        const float f = qk * fq * fk;
        put4<T>(o, fmaf(f, d[0], decay * pq[0]), fmaf(f, d[1], decay * pq[1]), fmaf(f, d[2], decay * pq[2]),
                fmaf(f, d[3], decay * pq[3]));
      }
      const F2 d0 = f2(d[0], d[1]), d1 = f2(d[2], d[3]), e = f2(decay, decay);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = kq[i * RG + rg].x;
        const F2 kx = f2(w, w);
        s[i][0] = fma2(kx, d0, mul2(e, s[i][0]));
        s[i][1] = fma2(kx, d1, mul2(e, s[i][1]));
      }
      if (writes) {
        float* const dst = a.s_out + (((long long)it.to * a.H + it.h) * a.DK + rg) * a.DV + it.c0 + cl * 4;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          float4 x;
          unf2(s[i][0], x.x, x.y);
          unf2(s[i][1], x.z, x.w);
          if (i * RG + rg < a.DK) __stcs(reinterpret_cast<float4*>(dst + (long long)i * RG * a.DV), x);
        }
      }
    }
  }
}

// [slots * H, DK, DV] float32 as boxes of `cols` columns x DK rows
bool state_map(CUtensorMap* m, const Args& a, int cols) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.DV, (cuuint64_t)a.DK, (cuuint64_t)a.slots * a.H};
  const cuuint64_t strides[2] = {(cuuint64_t)a.DV * 4, (cuuint64_t)a.DK * a.DV * 4};
  const cuuint32_t box[3] = {(cuuint32_t)cols, (cuuint32_t)a.DK, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<float*>(a.s_in), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename TV, int ROWS, int COLS>
int launch_run(const Args& a, cudaStream_t stream) {
  const int slices = (a.DV + kRunWarps * COLS - 1) / (kRunWarps * COLS);
  run_kernel<T, TV, ROWS, COLS><<<dim3((unsigned)(a.H * slices), (unsigned)a.B), kRunThreads, 0, stream>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, typename TV, int ROWS, int COLS>
int launch_token(const Args& a, int sms, cudaStream_t stream) {
  using C = Cfg<ROWS, COLS>;
  CUtensorMap m = {};
  if (a.s_in != nullptr && !state_map(&m, a, COLS)) return GD_ERR_LAUNCH;
  static bool done[kMaxDevices];
  auto kern = token_kernel<T, TV, ROWS, COLS>;
  if (set_smem_once(kern, C::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const long long items = (long long)a.B * a.H * (a.DV / COLS);
  kern<<<(unsigned)(items < sms ? items : sms), 32 * C::kWarps, C::kSmem, stream>>>(m, a);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, typename TV>
int launch(const Args& a, cudaStream_t stream) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  const long long heads = (long long)a.B * a.H;
  if (a.T == 1 && heads > sms && a.slots > 0) {  // (up to as many heads run_kernel has work for every SM at once)
    return a.DK <= 64    ? launch_token<T, TV, 64, 32>(a, sms, stream)
           : a.DK <= 128 ? launch_token<T, TV, 128, 16>(a, sms, stream)
                         : launch_token<T, TV, 256, 16>(a, sms, stream);
  }
  return a.DK > 128       ? launch_run<T, TV, 256, 16>(a, stream)
         : a.DK <= 64     ? launch_run<T, TV, 64, 32>(a, stream)
         : heads * 2 <= sms ? launch_run<T, TV, 128, 8>(a, stream)
                          : launch_run<T, TV, 128, 16>(a, stream);
}

// Tensor maps are encoded by the driver, which wants the device's context bound to the calling thread.
bool bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
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
  if (!bind_context()) return (cudaGetLastError(), GD_ERR_LAUNCH);
  Args a;
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.s_in = s_in, a.s_out = s_out, a.in = slots, a.out = out_slots;
  a.o = o, a.B = B, a.T = T, a.H = H, a.HK = HK, a.DK = DK, a.DV = DV, a.slots = n_slots;
  a.l2norm = (flags & GD_L2NORM) != 0;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (dtype == GD_FLOAT32) return launch<float, float>(a, cs);
  if (dtype == GD_FLOAT16) return vdtype == dtype ? launch<__half, __half>(a, cs) : launch<__half, float>(a, cs);
  return vdtype == dtype ? launch<__nv_bfloat16, __nv_bfloat16>(a, cs) : launch<__nv_bfloat16, float>(a, cs);
}
