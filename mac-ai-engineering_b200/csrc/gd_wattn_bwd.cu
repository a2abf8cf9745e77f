// Backward of the causal softmax attention with a sliding window and first tokens that stay visible. With P = softmax,
// L the forward's log2-sum and delta = rowsum(dO O):
//   P = exp2(scale log2(e) S - L),  dP = dO V^T,  dS = P (dP - delta)
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q       (dK, dV summed over the query heads of a key head)
// Bound by the chain product, elementwise work, product within a tile (tensor pipe 60 % busy). Measured at 1 x 8192 x 16
// heads (4 key heads), D 128, window 2048, bf16: delta 21 us (4.7 TB/s), dq 171 us, dk dv 300 us (1,060 and 810 TFLOP/s of 6 and 8 D operations a visible pair); at
// 2 x 2048 x 8 (2), D 256, causal: 10, 73 and 145 us.
// Three kernels, none of which waits on another CTA and none with atomics on results (the same bits every run):
//   delta_kernel  delta, and for float16 the largest ||dO|| and ||v|| (the scale below)
//   dq_kernel     one CTA per 128 queries of a head, over the key tiles they see
//   dkv_kernel    one CTA per 128 keys of a key head, over the group's query heads and the query tiles that see them
// S and dP are formed twice (7 products of 128 x 128 x D a tile pair instead of 5): with the queries on the rows in the
// first kernel and the keys on the rows in the second, so that every accumulator stays in TMEM for the whole loop and
// dS, P are the A operands of the products that follow straight from TMEM; nothing is exchanged between CTAs.
//
// P and dS are rounded to the inputs' 16-bit type (the operand type of the matrix instruction); exponentials, sums and
// accumulators are fp32. float16 has normal numbers from 2^-14 to 2^16 only, so both are scaled by powers of two before their
// rounding and the results scaled back:
//   P by 2^15 (P <= 1): all 11 bits down to P = 2^-29, as rows of millions of keys have
//   dS by F = 2^e, one for the call, with 2 F max ||dO|| max ||v|| in [2^14, 2^15]. That bounds F |dS| (dP is a product of two
//   rows, delta an average of dP), so nothing overflows whatever the sizes of dO and v, and |dS| keeps 11 bits down to 2^-29
//   of its bound; below, it is off by 2^-40 of the bound at most.
#include "gd_wattn.cuh"

namespace gd {
namespace wattn {
namespace {

constexpr int kWarpsEw = 16;                     // elementwise work: four threads a row, 32 columns each
constexpr int kThreads = 32 * (kWarpsEw + 2);    // + loads, + products (dK, dV: one more, for L and delta)

constexpr float kPScale = 32768.f, kPLog2 = 15.f;  // float16's P in dV and dK

// F. The error word's first spare fields hold the bits of the largest ||dO||^2 and ||v||^2 (float16; 0 or 2^-48 .. 2^41 each).
__device__ __forceinline__ float ds_scale(const ErrorWord* err) {
  const volatile int* p = &err->pad[0];
  const float c = __int_as_float(p[0]) * __int_as_float(p[1]);
  if (!(c > 0.f)) return 1.f;  // dS is 0
  const int e = ((__float_as_int(c) >> 23) & 0xff) - 127;  // sqrt(c) in [2^(k - 1), 2^k] with k = (e + 2) >> 1
  return __int_as_float((127 + 14 - ((e + 2) >> 1)) << 23);
}

// ---- delta = rowsum(dO O), O as its 16-bit value and what its rounding took away (delta and dP nearly cancel in rows
// that see few keys: O's rounding alone would cost dS half a bit there). 16 lanes a row of [B, Tq, H], kRowsEach rows in
// flight. HBM-bound: three reads of [B, Tq, H, D]. float16: also the largest ||dO||^2, and in the CTAs from `first_v` on the
// largest ||v||^2 (a row with an infinity or NaN does not count: what it reaches is infinite or NaN under any scale).
constexpr int kRowsEach = 4;

struct ValueRows {  // v [B, Tk, HK, D], strides in elements
  const void* v;
  long long b, t, h, rows;  // rows: Tk HK
  int HK;
  unsigned first;           // the CTAs from here on
};

// the largest of the warp's non-negative values, infinities and NaN aside -> word `to` (a maximum: any order)
__device__ __forceinline__ void put_max(float top, int* to) {
#pragma unroll
  for (int w = 16; w >= 1; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  if ((threadIdx.x & 31) == 0 && top > 0.f) atomicMax(to, __float_as_int(top));
}
__device__ __forceinline__ float finite_or_0(float x) { return x <= 3e38f ? x : 0.f; }

template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(const T* __restrict__ o, const T* __restrict__ low,
                                                    const T* __restrict__ g, long long gb, long long gt, long long gh,
                                                    float* __restrict__ delta, int Tq, int H, int D, const ValueRows vr,
                                                    ErrorWord* err) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  const int sub = threadIdx.x & 15;
  if constexpr (kHalf) {
    if (blockIdx.x >= vr.first) {
      const long long row0 = (long long)(blockIdx.x - vr.first) * (16 * kRowsEach) + (threadIdx.x >> 4);
      float top = 0.f;
#pragma unroll
      for (int r = 0; r < kRowsEach; ++r) {
        const long long row = row0 + r * 16, t = row / vr.HK;
        float n = 0.f;
        if (row < vr.rows) {
          const T* v = static_cast<const T*>(vr.v) + blockIdx.y * vr.b + t * vr.t + (row - t * vr.HK) * vr.h;
          for (int c = sub * 8; c < D; c += 128) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(v + c));
            const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 y = unpack16<T>(uu[i]);
              n = fmaf(y.x, y.x, n);
              n = fmaf(y.y, y.y, n);
            }
          }
        }
#pragma unroll
        for (int w = 8; w >= 1; w >>= 1) n += __shfl_xor_sync(0xffffffffu, n, w);
        top = fmaxf(top, finite_or_0(n));
      }
      put_max(top, &err->pad[1]);
      return;
    }
  }
  const unsigned rows = (unsigned)Tq * (unsigned)H;  // of batch row blockIdx.y
  if (!kHalf && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < sizeof(ErrorWord) / 4)
    reinterpret_cast<int*>(err)[threadIdx.x] = 0;  // (this kernel waits for nothing; the next ones record)
  const unsigned row0 = blockIdx.x * (16 * kRowsEach) + (threadIdx.x >> 4);
  o += (long long)blockIdx.y * rows * D;
  low += (long long)blockIdx.y * rows * D;
  g += blockIdx.y * gb;
  delta += (long long)blockIdx.y * rows;
  float s[kRowsEach], n[kRowsEach];  // n: ||dO||^2
  unsigned h[kRowsEach], t[kRowsEach];
#pragma unroll
  for (int r = 0; r < kRowsEach; ++r) {
    s[r] = n[r] = 0.f;
    t[r] = (row0 + r * 16) / (unsigned)H;
    h[r] = row0 + r * 16 - t[r] * (unsigned)H;
  }
  for (int c = sub * 8; c < D; c += 128) {
    uint4 a[kRowsEach], l[kRowsEach], d[kRowsEach];
#pragma unroll
    for (int r = 0; r < kRowsEach; ++r) {
      const unsigned row = row0 + r * 16;
      a[r] = l[r] = d[r] = make_uint4(0, 0, 0, 0);
      if (row < rows) {
        a[r] = __ldg(reinterpret_cast<const uint4*>(o + (long long)row * D + c));
        l[r] = __ldg(reinterpret_cast<const uint4*>(low + (long long)row * D + c));
        d[r] = __ldg(reinterpret_cast<const uint4*>(g + t[r] * gt + h[r] * gh + c));
      }
    }
#pragma unroll
    for (int r = 0; r < kRowsEach; ++r) {
      const uint32_t ua[4] = {a[r].x, a[r].y, a[r].z, a[r].w}, ul[4] = {l[r].x, l[r].y, l[r].z, l[r].w},
                     ud[4] = {d[r].x, d[r].y, d[r].z, d[r].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = unpack16<T>(ua[i]), z = unpack16<T>(ul[i]), y = unpack16<T>(ud[i]);
        if constexpr (kHalf) n[r] = fmaf(y.x, y.x, fmaf(y.y, y.y, n[r]));
        s[r] = fmaf(x.x + z.x, y.x, s[r]);
        s[r] = fmaf(x.y + z.y, y.y, s[r]);
      }
    }
  }
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < kRowsEach; ++r) {
#pragma unroll
    for (int w = 8; w >= 1; w >>= 1) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], w);
      if constexpr (kHalf) n[r] += __shfl_xor_sync(0xffffffffu, n[r], w);
    }
    if (row0 + r * 16 < rows && sub == 0) delta[(long long)h[r] * Tq + t[r]] = s[r];
    top = fmaxf(top, finite_or_0(n[r]));
  }
  if constexpr (kHalf) put_max(top, &err->pad[0]);
}

// 16 fp32 columns (from channel c) of an accumulator times f -> row `row` of a swizzled tile in shared memory, rounded
template <typename T>
__device__ __forceinline__ void stage16(uint32_t smem, int row, int c, const float (&v)[16], float f) {
#pragma unroll
  for (int k = 0; k < 16; k += 8) {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = pack16<T>(v[k + 2 * e] * f, v[k + 2 * e + 1] * f);
    st_shared16(smem + tile_at(row, (c + k) >> 3), u);
  }
}
// between the staging of a tile and its store: the elementwise warps (each gets here in bounded time, failed waits or not)
__device__ __forceinline__ void staged() {
  fence_async_smem();
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarpsEw) : "memory");
}

// dS of two columns: p (dp - delta) f, packed
template <typename T>
__device__ __forceinline__ uint32_t ds2(F2 p, F2 d, F2 minus_delta, float f) {
  F2 x = add2(d, minus_delta);
  if constexpr (std::is_same<T, __half>::value) x = mul2(x, f2(f, f));
  x = mul2(p, x);
  float a, b;
  unf2(x, a, b);
  return pack16<T>(a, b);
}

// ------------------------------------------------------------------------------------------------------------------
// dQ. TMEM: S | dP | dQ | dS (NS = 4: dS over dP). The products of the next key tile run under the elementwise work of
// this one as soon as its S and dP are in registers. Shared memory: Q, dO, a ring of key tiles (used twice: S, dQ) and
// one of value tiles; NS = 4: one ring of half tiles (128 channels) in the order of their use, keys loaded twice.
template <int NS>
struct DqCfg {
  static constexpr bool kHalves = NS == 4;
  static constexpr int kUnit = (kHalves ? 2 : NS) * kSlabBytes;
  static constexpr int kKs = kHalves ? 3 : NS == 1 ? 4 : 3, kVs = kHalves ? 0 : NS == 1 ? 4 : 2;
  static constexpr int kDp = 128, kDq = 256, kDs = kHalves ? 128 : 256 + NS * 64;
  static constexpr int kBarriers = 1 + 2 * (kKs + kVs) + 7;
  static constexpr size_t kSmem = 1024 + 2 * NS * kSlabBytes + (size_t)kUnit * (kKs + kVs) + 8 * kBarriers + 64;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <typename T, int NS>
__global__ void __launch_bounds__(kThreads, 1)
    dq_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
              const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mo,
              const __grid_constant__ CUtensorMap mdq, const Problem pr, const float* __restrict__ lse,
              const float* __restrict__ delta, T* __restrict__ dq, ErrorWord* err) {
  using C = DqCfg<NS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + 2 * NS * kSlabBytes + C::kUnit * (C::kKs + C::kVs));
  uint64_t* in_full = bars;  // Q and dO
  uint64_t* full = bars + 1;  // key ring, then value ring
  uint64_t* empty = full + C::kKs + C::kVs;
  uint64_t* s_full = empty + C::kKs + C::kVs;
  uint64_t* dp_full = s_full + 1;
  uint64_t* s_read = s_full + 2;
  uint64_t* dp_read = s_full + 3;
  uint64_t* ds_full = s_full + 4;
  uint64_t* dq_done = s_full + 5;
  uint64_t* fin = s_full + 6;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + C::kBarriers);
  int* info = reinterpret_cast<int*>(tslot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform

  if (threadIdx.x == 0) {
    mbar_init(in_full, 1);
    for (int i = 0; i < C::kKs + C::kVs; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(s_read, kWarpsEw);
    mbar_init(dp_read, kWarpsEw);
    mbar_init(ds_full, kWarpsEw);
    mbar_init(dq_done, 1);
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == kWarpsEw + 1) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  const int item = gridDim.x - 1 - blockIdx.x, h = blockIdx.y;  // later tiles see more keys: first
  Seq sq;
  int tile = item;
  bool gap = false;
  if (pr.cu != nullptr && warp == 0) {
    tile = find_item(pr.cu, pr.N, pr.Tq, item, [](int n) { return (n + kTile - 1) / kTile; }, sq, gap);
    if (lane == 0) {
      info[0] = tile;
      info[1] = sq.q0;
      info[2] = sq.Tq;
      info[3] = gap;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (pr.cu != nullptr) {
    tile = info[0];
    sq.b = 0;
    sq.q0 = sq.k0 = info[1];
    sq.Tq = sq.Tk = info[2];
    gap = info[3] != 0;
  } else {
    sq = {(int)blockIdx.z, 0, pr.Tq, 0, pr.Tk};
  }
  const uint32_t tm = __shfl_sync(0xffffffffu, *tslot, 0);  // uniform
  const int i0 = tile * kTile;
  const int i1 = i0 + kTile - 1 < sq.Tq - 1 ? i0 + kTile - 1 : sq.Tq - 1;
  const int p0 = i0 + sq.offset(), p1 = i1 + sq.offset();
  const bool idle = tile < 0 || gap;
  const KeyRange kr(idle ? -1 : p0, idle ? -1 : p1, pr.window, pr.sinks);
  const uint32_t s_q = smem_u32(base), s_o = s_q + NS * kSlabBytes, s_k = s_o + NS * kSlabBytes,
                 s_v = s_k + C::kKs * C::kUnit;

  if (warp == kWarpsEw) {
    if (lane == 0 && kr.n > 0) {
      const int hk = h / (pr.H / pr.HK);
      mbar_arrive_expect_tx(in_full, 2 * NS * kSlabBytes);
      load_tile<NS>(s_q, &mq, h, sq.q0 + i0, sq.b, in_full);
      load_tile<NS>(s_o, &mo, h, sq.q0 + i0, sq.b, in_full);
      bool ok = true;
      int nk = 0, nv = 0;  // units loaded into each ring
      if constexpr (!C::kHalves) {
        for (int j = 0; ok && j < kr.n; ++j) {
          const int t = sq.k0 + kr.key(j);
          const int a = nk % C::kKs, b = nv % C::kVs;
          if (nk >= C::kKs && !(ok = mbar_wait(empty + a, (nk / C::kKs - 1) & 1, err, 80))) break;
          mbar_arrive_expect_tx(full + a, C::kUnit);
          load_tile<NS>(s_k + a * C::kUnit, &mk, hk, t, sq.b, full + a);
          ++nk;
          if (nv >= C::kVs && !(ok = mbar_wait(empty + C::kKs + b, (nv / C::kVs - 1) & 1, err, 81))) break;
          mbar_arrive_expect_tx(full + C::kKs + b, C::kUnit);
          load_tile<NS>(s_v + b * C::kUnit, &mv, hk, t, sq.b, full + C::kKs + b);
          ++nv;
        }
      } else {
        auto halves = [&](const CUtensorMap* m, int j) {  // the two halves of tile j
#pragma unroll 1
          for (int x = 0; ok && x < 2; ++x) {
            const int a = nk % C::kKs;
            if (nk >= C::kKs && !(ok = mbar_wait(empty + a, (nk / C::kKs - 1) & 1, err, 82))) return;
            mbar_arrive_expect_tx(full + a, C::kUnit);
            load_half(s_k + a * C::kUnit, m, x, hk, sq.k0 + kr.key(j), sq.b, full + a);
            ++nk;
          }
        };
        halves(&mk, 0);
        if (ok) halves(&mv, 0);
        for (int j = 0; ok && j < kr.n; ++j) {
          if (j + 1 < kr.n) halves(&mk, j + 1);
          if (ok) halves(&mk, j);
          if (ok && j + 1 < kr.n) halves(&mv, j + 1);
        }
      }
      mbar_wait(in_full, 0, err, 83);  // the copies in flight land before the CTA ends
      for (int l = nk > C::kKs ? nk - C::kKs : 0; l < nk; ++l) mbar_wait(full + l % C::kKs, (l / C::kKs) & 1, err, 83);
      if constexpr (C::kVs > 0)
        for (int l = nv > C::kVs ? nv - C::kVs : 0; l < nv; ++l)
          mbar_wait(full + C::kKs + l % C::kVs, (l / C::kVs) & 1, err, 83);
    }
  } else if (warp == kWarpsEw + 1) {
    if (kr.n > 0) {
      const uint32_t lead = elect();
      bool ok = warp_wait(in_full, 0, err, 84);
      if constexpr (!C::kHalves) {
        auto first = [&](int j) {  // S and dP of tile j
          const int a = j % C::kKs, b = C::kKs + j % C::kVs;
          if (!warp_wait(full + a, (j / C::kKs) & 1, err, 85)) return false;
          if (j > 0 && !warp_wait(s_read, (j - 1) & 1, err, 86)) return false;
          tc_fence_after();
          mma_xyt<T, NS>(lead, tm, s_q, s_k + a * C::kUnit);
          mma_commit(lead, s_full);
          if (!warp_wait(full + b, (j / C::kVs) & 1, err, 87)) return false;
          if (j > 0 && !warp_wait(dp_read, (j - 1) & 1, err, 88)) return false;
          tc_fence_after();
          mma_xyt<T, NS>(lead, tm + C::kDp, s_o, s_v + (j % C::kVs) * C::kUnit);
          mma_commit(lead, dp_full);
          mma_commit(lead, empty + b);
          return true;
        };
        ok = ok && first(0);
        for (int j = 0; ok && j < kr.n; ++j) {
          if (j + 1 < kr.n) ok = first(j + 1);
          if (!(ok = ok && warp_wait(ds_full, j & 1, err, 89))) break;
          tc_fence_after();
          mma_py<T, NS>(lead, tm + C::kDq, tm + C::kDs, s_k + (j % C::kKs) * C::kUnit, j > 0, 16);
          mma_commit(lead, empty + j % C::kKs);
          mma_commit(lead, dq_done);
        }
      } else {
        int n = 0;  // units used
        auto pair = [&](uint32_t d, uint32_t x) {  // D = X Y^T over the ring's next two halves
          for (int y = 0; y < 2; ++y, ++n) {
            const int a = n % C::kKs;
            if (!warp_wait(full + a, (n / C::kKs) & 1, err, 85)) return false;
            tc_fence_after();
            mma_xyt<T, 2>(lead, d, x + y * 2 * kSlabBytes, s_k + a * C::kUnit, y > 0);
            mma_commit(lead, empty + a);
          }
          return true;
        };
        ok = ok && pair(tm, s_q);
        if (ok) mma_commit(lead, s_full);
        ok = ok && pair(tm + C::kDp, s_o);
        if (ok) mma_commit(lead, dp_full);
        for (int j = 0; ok && j < kr.n; ++j) {
          if (j + 1 < kr.n) {
            ok = warp_wait(s_read, j & 1, err, 86) && pair(tm, s_q);
            if (ok) mma_commit(lead, s_full);
          }
          if (!(ok = ok && warp_wait(ds_full, j & 1, err, 89))) break;
          tc_fence_after();
          for (int y = 0; ok && y < 2; ++y, ++n) {
            const int a = n % C::kKs;
            if (!(ok = warp_wait(full + a, (n / C::kKs) & 1, err, 85))) break;
            if (pr.cu != nullptr) zero_rows<2>(s_k + a * C::kUnit, sq.Tk - kr.key(j));
            tc_fence_after();
            mma_py<T, 2>(lead, tm + C::kDq + y * 128, tm + C::kDs, s_k + a * C::kUnit, j > 0, 16);
            mma_commit(lead, empty + a);
          }
          if (!ok) break;
          mma_commit(lead, dq_done);
          if (j + 1 < kr.n) {  // dP over dS, once its products have read it
            ok = warp_wait(dq_done, j & 1, err, 88);
            tc_fence_after();
            ok = ok && pair(tm + C::kDp, s_o);
            if (ok) mma_commit(lead, dp_full);
          }
        }
      }
      mma_commit(lead, fin);
      warp_wait(fin, 0, err, 90);
    }
  } else if (tile >= 0) {
    const int row = (warp & 3) * 32 + lane, part = warp >> 2;  // TMEM lane, which 32 columns
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int i = i0 + row, p = p0 + row;
    const bool live = i < sq.Tq;
    const long long at = ((long long)sq.b * pr.H + h) * pr.Tq + sq.q0 + i;
    const float L = live ? lse[at] : INFINITY, de = live ? delta[at] : 0.f;
    const F2 sc = f2(pr.scale_log2, pr.scale_log2), mL = f2(-L, -L), mde = f2(-de, -de);
    float f = 1.f;
    if constexpr (std::is_same<T, __half>::value) f = ds_scale(err);
    bool ok = true;
    for (int j = 0; j < kr.n; ++j) {
      const int c0 = kr.key(j) + part * 32;
      const bool whole = all_visible(kr.key(j), p0, p1, pr.window, pr.sinks);
      const uint32_t vis = whole ? 0xffffffffu : visible_keys(c0, p, pr.window, pr.sinks);
      float s[32], d[32];
      if (!(ok = warp_wait(s_full, j & 1, err, 91))) break;
      tc_fence_after();
      if (!C::kHalves && pr.cu != nullptr && kr.key(j) + kTile > sq.Tk)  // K's rows past the sequence (S has read them)
        zero_rows<NS>(s_k + j % C::kKs * C::kUnit, sq.Tk - kr.key(j), kTile, threadIdx.x, 32 * kWarpsEw);
      tmem_ld32(tm + lanes + part * 32, s);
      tc_fence_before();
      mbar_arrive_warp(s_read);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        ex2_pair(fma2(f2(s[c], s[c + 1]), sc, mL), s[c], s[c + 1]);
      }
      if (!(ok = warp_wait(dp_full, j & 1, err, 92))) break;
      tc_fence_after();
      tmem_ld32(tm + lanes + C::kDp + part * 32, d);
      tc_fence_before();
      mbar_arrive_warp(dp_read);
      if (!whole) {  // nothing of a masked key reaches dS, infinities and NaN included
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          s[c] = (vis >> c) & 1 ? s[c] : 0.f;
          d[c] = (vis >> c) & 1 ? d[c] : de;
        }
      }
      uint32_t u[16];
#pragma unroll
      for (int c = 0; c < 32; c += 2) u[c / 2] = ds2<T>(f2(s[c], s[c + 1]), f2(d[c], d[c + 1]), mde, f);
      // dS's columns: free once the last dQ product has read them. NS = 4: over dP, where all of a row's dP must be in
      // registers first
      if (C::kHalves) {
        if (!(ok = warp_wait(dp_read, j & 1, err, 93))) break;
      } else if (j > 0) {
        if (!(ok = warp_wait(dq_done, (j - 1) & 1, err, 93))) break;
      }
      tc_fence_after();
      tmem_st16(tm + lanes + C::kDs + part * 16, u);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(ds_full);
    }
    if (ok && kr.n > 0) {
      ok = warp_wait(dq_done, (kr.n - 1) & 1, err, 94);
      tc_fence_after();
    }
    const float g = ok ? pr.scale / f : NAN;
#pragma unroll
    for (int c = part * NS * 16; c < (part + 1) * NS * 16; c += 16) {
      float v[16];
      if (kr.n > 0) {
        tmem_ld16(tm + lanes + C::kDq + c, v);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = 0.f;
      }
      stage16<T>(s_q, row, c, v, g);  // Q's place
    }
    staged();
    if (warp < 4) store_rows<T, NS>(&mdq, dq, s_q, warp * 32, sq.b, sq.q0 + i0, sq.Tq - i0, pr.Tq, h, pr.H, pr.D);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpsEw + 1) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// dK, dV. S^T = K Q^T and dP^T = V dO^T with the keys on the rows. TMEM: S^T | dP^T | dV | dK, P^T over S^T and dS^T over
// dP^T (each thread's 32 columns over its own). The elementwise warps are two groups of eight, one for each 64 of a tile's
// queries, with signals of their own; the products alternate between the groups, so that each waits for what the other
// group's product covers: dV(i) on P^T(i), S^T(i + 1) once dV(i) has read P^T, dK(i) on dS^T(i), dP^T(i + 1) once dK(i) has
// read dS^T. (One signal for all sixteen warps left the tensor pipe idle for every one of those four latencies: 316 us
// against 296 us at 1 x 8192 x 16, 4 key heads, D 128, window 2048.) The sums are formed in this order in every run. NS = 4: a
// CTA accumulates one half of the channels (S^T and dP^T over all of them), Q and dO pass through a ring of half tiles in the
// order of their use, and the groups stay in step.
// parts > 1 (the first `heavy` key tiles): the tile's list of (query head, query tile) is cut into `parts` pieces, a CTA
// each, whose sums go to fp32 partial tiles that sum_parts adds in order.
template <int NS>
struct DkvCfg {
  static constexpr bool kHalves = NS == 4;
  static constexpr int kAcc = NS == 1 ? 64 : 128;  // channels a CTA accumulates
  static constexpr int kUnit = (kHalves ? 2 : NS) * kSlabBytes;
  static constexpr int kQs = kHalves ? 3 : 2, kOs = kHalves ? 0 : 2;
  static constexpr int kDp = 128, kDv = 256, kDk = 256 + kAcc;
  static constexpr int kStats = kHalves ? 1 : 2;   // buffers of L and delta of a query tile
  static constexpr int kBarriers = 1 + 2 * (kQs + kOs) + 13 + 2 * kStats;
  static constexpr size_t kSmem =
      1024 + 2 * NS * kSlabBytes + (size_t)kUnit * (kQs + kOs) + 8 * kBarriers + 64 + kStats * 2 * 4 * kTile;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct Split {
  int heavy, parts;
  float* part;  // [b, key head, heavy tile, part][dK, dV][128][D]
};

template <typename T, int NS>
__global__ void __launch_bounds__(kThreads + 32, 1)
    dkv_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
               const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mo,
               const __grid_constant__ CUtensorMap mdk, const __grid_constant__ CUtensorMap mdv, const Problem pr,
               const Split sp, const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dk,
               T* __restrict__ dv, ErrorWord* err) {
  using C = DkvCfg<NS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // [kStats][L, delta][128]
  float* stats = reinterpret_cast<float*>(base + 2 * NS * kSlabBytes + C::kUnit * (C::kQs + C::kOs));
  uint64_t* bars = reinterpret_cast<uint64_t*>(stats + C::kStats * 2 * kTile);
  uint64_t* in_full = bars;   // K and V
  uint64_t* full = bars + 1;  // Q ring, then dO ring
  uint64_t* empty = full + C::kQs + C::kOs;
  uint64_t* s_full = empty + C::kQs + C::kOs;
  uint64_t* dp_full = s_full + 2;             // of each group, as the next four
  uint64_t* p_full = s_full + 4;
  uint64_t* ds_full = s_full + 6;
  uint64_t* dv_done = s_full + 8;
  uint64_t* dk_done = s_full + 10;
  uint64_t* st_full = s_full + 12;
  uint64_t* st_empty = st_full + C::kStats;
  uint64_t* fin = st_empty + C::kStats;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + C::kBarriers);
  int* info = reinterpret_cast<int*>(tslot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform

  if (threadIdx.x == 0) {
    mbar_init(in_full, 1);
    for (int i = 0; i < C::kQs + C::kOs; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, C::kHalves ? 1 : 2);  // both groups' products have read the tile
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_full + g, 1);
      mbar_init(dp_full + g, 1);
      mbar_init(p_full + g, kWarpsEw / 2);
      mbar_init(ds_full + g, kWarpsEw / 2);
      mbar_init(dv_done + g, 1);
      mbar_init(dk_done + g, 1);
    }
    for (int i = 0; i < C::kStats; ++i) {
      mbar_init(st_full + i, 1);
      mbar_init(st_empty + i, kWarpsEw);
    }
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == kWarpsEw + 1) {
    tmem_alloc(tslot, 512);
    tmem_relinquish();
  }
  const int xh = C::kHalves ? (int)(blockIdx.y & 1) : 0;  // which half of the channels is accumulated
  const int hk = C::kHalves ? (int)(blockIdx.y >> 1) : (int)blockIdx.y;
  const int G = pr.H / pr.HK;
  Seq sq;
  // the first key tiles are seen by most queries: they start first, cut into parts where that pays
  int tile = blockIdx.x, part = 0, parts = 1;
  bool gap = false;
  if (tile < sp.heavy * sp.parts) {
    parts = sp.parts;
    part = tile % parts;
    tile /= parts;
  } else {
    tile -= sp.heavy * (sp.parts - 1);
  }
  if (pr.cu != nullptr && warp == 0) {
    tile = find_item(pr.cu, pr.N, pr.Tk, blockIdx.x, [](int n) { return (n + kTile - 1) / kTile; }, sq, gap);
    if (lane == 0) {
      info[0] = tile;
      info[1] = sq.q0;
      info[2] = sq.Tq;
      info[3] = gap;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (pr.cu != nullptr) {
    tile = info[0];
    sq.b = 0;
    sq.q0 = sq.k0 = info[1];
    sq.Tq = sq.Tk = info[2];
    gap = info[3] != 0;
  } else {
    sq = {(int)blockIdx.z, 0, pr.Tq, 0, pr.Tk};
  }
  const uint32_t tm = __shfl_sync(0xffffffffu, *tslot, 0);  // uniform
  const int c0 = tile * kTile, off = sq.offset();
  // the query tiles that see some of these keys
  int lo = 0, nq = 0;
  if (tile >= 0 && !gap) {
    const int from = c0 - off > 0 ? c0 - off : 0;
    int last = sq.Tq - 1;
    if (c0 >= pr.sinks && pr.window < kNoWindow) {
      const long long w = (long long)c0 + kTile - 1 + pr.window - 1 - off;
      if (w < last) last = (int)w;
    }
    lo = from / kTile;
    if (last >= from) nq = last / kTile - lo + 1;
  }
  const int all = nq * G;
  const int it0 = (int)((long long)all * part / parts), n = (int)((long long)all * (part + 1) / parts) - it0;
  const uint32_t s_k = smem_u32(base), s_v = s_k + NS * kSlabBytes, s_q = s_v + NS * kSlabBytes,
                 s_o = s_q + C::kQs * C::kUnit;

  if (warp == kWarpsEw + 2) {
    // -L (float16: + 15, P's scale) and -delta of each iteration's queries, a step ahead of the elementwise warps; dead
    // queries get -inf and 0
    const long long at = (long long)sq.b * pr.H * pr.Tq + sq.q0;
    int h = hk * G + (n > 0 ? it0 / nq : 0), qt = lo + (n > 0 ? it0 % nq : 0);
    for (int i = 0; i < n; ++i) {
      float L[4], de[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int t = qt * kTile + x * 32 + lane;
        const bool live = t < sq.Tq;
        constexpr float up = std::is_same<T, __half>::value ? kPLog2 : 0.f;
        L[x] = live ? up - __ldg(lse + at + (long long)h * pr.Tq + t) : -INFINITY;
        de[x] = live ? -__ldg(delta + at + (long long)h * pr.Tq + t) : 0.f;
      }
      if (++qt == lo + nq) {
        qt = lo;
        ++h;
      }
      float* st = stats + (i % C::kStats) * 256;
      if (i >= C::kStats && !warp_wait(st_empty + i % C::kStats, (i / C::kStats - 1) & 1, err, 115)) break;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        st[x * 32 + lane] = L[x];
        st[128 + x * 32 + lane] = de[x];
      }
      mbar_arrive_warp(st_full + i % C::kStats);
    }
  } else if (warp == kWarpsEw) {
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(in_full, 2 * NS * kSlabBytes);
      load_tile<NS>(s_k, &mk, hk, sq.k0 + c0, sq.b, in_full);
      load_tile<NS>(s_v, &mv, hk, sq.k0 + c0, sq.b, in_full);
      bool ok = true;
      int a_n = 0, b_n = 0;
      if constexpr (!C::kHalves) {
        for (int i = 0; ok && i < n; ++i) {
          const int h = hk * G + (it0 + i) / nq, t = sq.q0 + (lo + (it0 + i) % nq) * kTile;
          const int a = i % C::kQs, b = C::kQs + i % C::kOs;
          if (i >= C::kQs && !(ok = mbar_wait(empty + a, (i / C::kQs - 1) & 1, err, 100))) break;
          mbar_arrive_expect_tx(full + a, C::kUnit);
          load_tile<NS>(s_q + a * C::kUnit, &mq, h, t, sq.b, full + a);
          ++a_n;
          if (i >= C::kOs && !(ok = mbar_wait(empty + b, (i / C::kOs - 1) & 1, err, 101))) break;
          mbar_arrive_expect_tx(full + b, C::kUnit);
          load_tile<NS>(s_o + (i % C::kOs) * C::kUnit, &mo, h, t, sq.b, full + b);
          ++b_n;
        }
      } else {
        auto unit = [&](const CUtensorMap* m, int x, int i) {
          const int h = hk * G + (it0 + i) / nq, t = sq.q0 + (lo + (it0 + i) % nq) * kTile;
          const int a = a_n % C::kQs;
          if (a_n >= C::kQs && !(ok = ok && mbar_wait(empty + a, (a_n / C::kQs - 1) & 1, err, 102))) return;
          mbar_arrive_expect_tx(full + a, C::kUnit);
          load_half(s_q + a * C::kUnit, m, x, h, t, sq.b, full + a);
          ++a_n;
        };
        unit(&mq, 0, 0);
        unit(&mq, 1, 0);
        unit(&mo, 0, 0);
        if (ok) unit(&mo, 1, 0);
        for (int i = 0; ok && i < n; ++i) {
          unit(&mo, xh, i);
          if (ok && i + 1 < n) unit(&mq, 0, i + 1);
          if (ok && i + 1 < n) unit(&mq, 1, i + 1);
          if (ok) unit(&mq, xh, i);
          if (ok && i + 1 < n) unit(&mo, 0, i + 1);
          if (ok && i + 1 < n) unit(&mo, 1, i + 1);
        }
      }
      mbar_wait(in_full, 0, err, 103);  // the copies in flight land before the CTA ends
      for (int l = a_n > C::kQs ? a_n - C::kQs : 0; l < a_n; ++l) mbar_wait(full + l % C::kQs, (l / C::kQs) & 1, err, 103);
      if constexpr (C::kOs > 0)
        for (int l = b_n > C::kOs ? b_n - C::kOs : 0; l < b_n; ++l)
          mbar_wait(full + C::kQs + l % C::kOs, (l / C::kOs) & 1, err, 103);
    }
  } else if (warp == kWarpsEw + 1) {
    if (n > 0) {
      const uint32_t lead = elect();
      bool ok = warp_wait(in_full, 0, err, 104);
      if constexpr (!C::kHalves) {
        constexpr int kRows64 = 64 * 128;  // bytes of 64 rows of a slab
        auto scores = [&](int i, int g) {
          tc_fence_after();
          mma_xyt<T, NS, 64>(lead, tm + 64 * g, s_k, s_q + i % C::kQs * C::kUnit + g * kRows64);
          mma_commit(lead, s_full + g);
        };
        auto dps = [&](int i, int g) {
          tc_fence_after();
          mma_xyt<T, NS, 64>(lead, tm + C::kDp + 64 * g, s_v, s_o + i % C::kOs * C::kUnit + g * kRows64);
          mma_commit(lead, dp_full + g);
        };
        if ((ok = ok && warp_wait(full, 0, err, 105) && warp_wait(full + C::kQs, 0, err, 107))) {
          scores(0, 0);
          scores(0, 1);
          dps(0, 0);
          dps(0, 1);
        }
        for (int i = 0; ok && i < n; ++i) {
          const uint32_t qa = s_q + i % C::kQs * C::kUnit, oa = s_o + i % C::kOs * C::kUnit;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!(ok = ok && warp_wait(p_full + g, i & 1, err, 109))) break;
            tc_fence_after();
            mma_py<T, NS, 4>(lead, tm + C::kDv, tm + 64 * g, oa + g * kRows64, i > 0 || g > 0, 32);
            mma_commit(lead, dv_done + g);
            mma_commit(lead, empty + C::kQs + i % C::kOs);
          }
          if (i + 1 < n) {  // S over P, once that is read
            ok = ok && warp_wait(full + (i + 1) % C::kQs, ((i + 1) / C::kQs) & 1, err, 105);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (!(ok = ok && warp_wait(dv_done + g, i & 1, err, 106))) break;
              scores(i + 1, g);
            }
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!(ok = ok && warp_wait(ds_full + g, i & 1, err, 110))) break;
            tc_fence_after();
            mma_py<T, NS, 4>(lead, tm + C::kDk, tm + C::kDp + 64 * g, qa + g * kRows64, i > 0 || g > 0, 32);
            mma_commit(lead, dk_done + g);
            mma_commit(lead, empty + i % C::kQs);
          }
          if (i + 1 < n) {  // dP over dS, once that is read
            ok = ok && warp_wait(full + C::kQs + (i + 1) % C::kOs, ((i + 1) / C::kOs) & 1, err, 107);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              if (!(ok = ok && warp_wait(dk_done + g, i & 1, err, 108))) break;
              dps(i + 1, g);
            }
          }
        }
      } else {
        int u = 0;  // units used
        auto next = [&]() { return warp_wait(full + u % C::kQs, (u / C::kQs) & 1, err, 105); };
        auto pair = [&](uint32_t d, uint32_t x) {
          for (int y = 0; y < 2; ++y, ++u) {
            if (!next()) return false;
            tc_fence_after();
            mma_xyt<T, 2>(lead, d, x + y * 2 * kSlabBytes, s_q + u % C::kQs * C::kUnit, y > 0);
            mma_commit(lead, empty + u % C::kQs);
          }
          return true;
        };
        ok = ok && pair(tm, s_k);
        auto live = [&](int i) { return sq.Tq - (lo + (it0 + i) % nq) * kTile; };  // rows of the iteration's tile
        auto both = [&](uint64_t* bar) {
          mma_commit(lead, bar);
          mma_commit(lead, bar + 1);
        };
        auto wait2 = [&](uint64_t* bar, int i, int where) {
          return warp_wait(bar, i & 1, err, where) && warp_wait(bar + 1, i & 1, err, where);
        };
        if (ok) both(s_full);
        ok = ok && pair(tm + C::kDp, s_v);
        if (ok) both(dp_full);
        for (int i = 0; ok && i < n; ++i) {
          if (!(ok = wait2(p_full, i, 109) && next())) break;
          if (pr.cu != nullptr) zero_rows<2>(s_q + u % C::kQs * C::kUnit, live(i));
          tc_fence_after();
          mma_py<T, 2>(lead, tm + C::kDv, tm, s_q + u % C::kQs * C::kUnit, i > 0, 32);
          mma_commit(lead, empty + u % C::kQs);
          mma_commit(lead, dv_done);
          ++u;
          if (i + 1 < n) {
            ok = warp_wait(dv_done, i & 1, err, 106);
            tc_fence_after();
            ok = ok && pair(tm, s_k);
            if (ok) both(s_full);
          }
          if (!(ok = ok && wait2(ds_full, i, 110) && next())) break;
          if (pr.cu != nullptr) zero_rows<2>(s_q + u % C::kQs * C::kUnit, live(i));
          tc_fence_after();
          mma_py<T, 2>(lead, tm + C::kDk, tm + C::kDp, s_q + u % C::kQs * C::kUnit, i > 0, 32);
          mma_commit(lead, empty + u % C::kQs);
          mma_commit(lead, dk_done);
          ++u;
          if (i + 1 < n) {
            ok = warp_wait(dk_done, i & 1, err, 108);
            tc_fence_after();
            ok = ok && pair(tm + C::kDp, s_v);
            if (ok) both(dp_full);
          }
        }
      }
      mma_commit(lead, fin);
      warp_wait(fin, 0, err, 111);
    }
  } else if (tile >= 0) {
    const int row = (warp & 3) * 32 + lane, quarter = warp >> 2, gr = quarter >> 1;  // TMEM lane, which 32 columns, group
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int key = c0 + row;
    const F2 sc = f2(pr.scale_log2, pr.scale_log2);
    constexpr bool kHalf = std::is_same<T, __half>::value;
    float f = 1.f;
    if constexpr (kHalf) f = ds_scale(err);
    const float fp = kHalf ? f / kPScale : f;  // dS from a P that carries 2^15
    bool ok = true;
    int qt = lo + (n > 0 ? it0 % nq : 0);  // the iteration's query tile
    for (int i = 0; i < n; ++i) {
      const float* st = stats + (i % C::kStats) * 256;  // -L and -delta of the tile's queries
      const ulonglong2* L4 = reinterpret_cast<const ulonglong2*>(st + quarter * 32);
      const ulonglong2* D4 = reinterpret_cast<const ulonglong2*>(st + 128 + quarter * 32);
      const int i0 = qt * kTile, q0 = i0 + off;  // the tile's first query and its position
      const bool whole = i0 + kTile <= sq.Tq && all_visible(c0, q0, q0 + kTile - 1, pr.window, pr.sinks);
      uint32_t vis = 0xffffffffu;
      if (!whole) {
        // query column c (position q0 + 32 quarter + c) sees the key: key <= position, key > position - window or key < sinks
        const long long to = key < pr.sinks ? (1ll << 40) : (long long)key + pr.window - q0 - quarter * 32;
        int end = sq.Tq - i0 - quarter * 32;
        if (to < end) end = (int)to;
        vis = bits(key - q0 - quarter * 32, end);
      }
      if (++qt == lo + nq) qt = lo;
      if (!(ok = warp_wait(st_full + i % C::kStats, (i / C::kStats) & 1, err, 116) &&
            warp_wait(s_full + gr, i & 1, err, 112))) break;
      if constexpr (!C::kHalves) {
        if (pr.cu != nullptr && i0 + (gr + 1) * 64 > sq.Tq) {
          // rows past the sequence of the group's 64 of Q and dO, once S and dP have read them (the warp that issues the
          // products, doing this, took 10 us more of 45 at 4,093 packed rows of seven sequences, 12 heads of 96)
          if (!(ok = warp_wait(dp_full + gr, i & 1, err, 113))) break;
          const int from = sq.Tq - i0 > gr * 64 ? sq.Tq - i0 : gr * 64, id = threadIdx.x & 255;
          zero_rows<NS>(s_q + i % C::kQs * C::kUnit, from, (gr + 1) * 64, id, 256);
          zero_rows<NS>(s_o + i % C::kOs * C::kUnit, from, (gr + 1) * 64, id, 256);
        }
      }
      tc_fence_after();
      float s[32], d[32];
      tmem_ld32(tm + lanes + quarter * 32, s);
      uint32_t u[16];
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const ulonglong2 L = L4[c / 4];
        ex2_pair(fma2(f2(s[c], s[c + 1]), sc, L.x), s[c], s[c + 1]);
        ex2_pair(fma2(f2(s[c + 2], s[c + 3]), sc, L.y), s[c + 2], s[c + 3]);
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 32; ++c) s[c] = (vis >> c) & 1 ? s[c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 32; c += 2) u[c / 2] = pack16<T>(s[c], s[c + 1]);
      tmem_st16(tm + lanes + quarter * 32, u);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(p_full + gr);
      if (!(ok = warp_wait(dp_full + gr, i & 1, err, 113))) break;
      tc_fence_after();
      tmem_ld32(tm + lanes + C::kDp + quarter * 32, d);
      if (!whole) {  // nothing of a masked pair reaches dS, infinities and NaN included
#pragma unroll
        for (int c = 0; c < 32; ++c) d[c] = (vis >> c) & 1 ? d[c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const ulonglong2 e = D4[c / 4];
        u[c / 2] = ds2<T>(f2(s[c], s[c + 1]), f2(d[c], d[c + 1]), e.x, fp);
        u[c / 2 + 1] = ds2<T>(f2(s[c + 2], s[c + 3]), f2(d[c + 2], d[c + 3]), e.y, fp);
      }
      tmem_st16(tm + lanes + C::kDp + quarter * 32, u);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(ds_full + gr);
      mbar_arrive_warp(st_empty + i % C::kStats);
    }
    if (ok && n > 0) {
      ok = warp_wait(fin, 0, err, 114);  // all products
      tc_fence_after();
    }
    // quarters 0 and 1 take dK's channels, 2 and 3 dV's; key row each
    const bool is_k = quarter < 2;
    const float g = !ok ? NAN : is_k ? pr.scale / f : kHalf ? 1.f / kPScale : 1.f;
    const uint32_t acc = tm + lanes + (is_k ? C::kDk : C::kDv);
    const int ch = xh * 128;  // the first channel accumulated
#pragma unroll 1
    for (int c = (quarter & 1) * (C::kAcc / 2); c < ((quarter & 1) + 1) * (C::kAcc / 2); c += 16) {
      float v[16];
      if (n > 0) {
        tmem_ld16(acc + c, v);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = 0.f;
      }
      if (parts == 1) {
        stage16<T>(is_k ? s_k : s_v, row, c, v, g);  // K's and V's places
      } else if (key < sq.Tk) {
        float* out = sp.part + (((((long long)sq.b * pr.HK + hk) * sp.heavy + tile) * parts + part) * 2 + (is_k ? 0 : 1)) *
                                   kTile * pr.D + (long long)row * pr.D;
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          if (ch + c + k < pr.D)
            *reinterpret_cast<float4*>(out + ch + c + k) = make_float4(v[k] * g, v[k + 1] * g, v[k + 2] * g, v[k + 3] * g);
      }
    }
    staged();
    if (parts == 1 && warp < 8) {
      const bool kw = warp < 4;
      store_rows<T, C::kAcc / 64>(kw ? &mdk : &mdv, kw ? dk : dv, kw ? s_k : s_v, (warp & 3) * 32, sq.b, sq.k0 + c0,
                                  sq.Tk - c0, pr.Tk, hk, pr.HK, pr.D, ch);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpsEw + 1) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// dK and dV of the heavy tiles: their parts in order; a thread 4 channels of a row
template <typename T>
__global__ void __launch_bounds__(256) sum_parts(const float* __restrict__ part, T* __restrict__ dk, T* __restrict__ dv,
                                                 int Tk, int HK, int D, int heavy, int parts) {
  const int per = kTile * D / 4, i = blockIdx.x * 256 + threadIdx.x;
  const int tile = blockIdx.y >> 1, which = blockIdx.y & 1;
  const int b = blockIdx.z / HK, hk = blockIdx.z % HK;
  if (i >= per) return;
  const int row = i / (D / 4), c = i % (D / 4) * 4, key = tile * kTile + row;
  if (key >= Tk) return;
  const float* p = part + ((((long long)b * HK + hk) * heavy + tile) * parts * 2 + which) * kTile * D + (long long)row * D + c;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = 0; x < parts; ++x) {
    const float4 v = *reinterpret_cast<const float4*>(p + (long long)x * 2 * kTile * D);
    t.x += v.x;
    t.y += v.y;
    t.z += v.z;
    t.w += v.w;
  }
  T* out = (which ? dv : dk) + (((long long)b * Tk + key) * HK + hk) * D + c;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(t.x, t.y), pack16<T>(t.z, t.w));
}

template <typename T, int NS>
int launch(const void* q, const void* k, const void* v, const void* o, const void* low, const void* g, const long long* st,
           const Problem& pr, const float* lse, float* delta, void* dq, void* dk, void* dv, Split sp, ErrorWord* err,
           cudaStream_t stream) {
  CUtensorMap mq, mk, mv, mo, mdq, mdk, mdv;
  const CUtensorMapDataType dt = map_dtype<T>();
  if (!tile_map(&mq, q, dt, pr.B, pr.Tq, pr.H, pr.D, st[0], st[1], st[2], kTile) ||
      !tile_map(&mk, k, dt, pr.B, pr.Tk, pr.HK, pr.D, st[3], st[4], st[5], kTile) ||
      !tile_map(&mv, v, dt, pr.B, pr.Tk, pr.HK, pr.D, st[6], st[7], st[8], kTile) ||
      !tile_map(&mo, g, dt, pr.B, pr.Tq, pr.H, pr.D, st[9], st[10], st[11], kTile) ||
      !out_map(&mdq, dq, dt, pr.B, pr.Tq, pr.H, pr.D) || !out_map(&mdk, dk, dt, pr.B, pr.Tk, pr.HK, pr.D) ||
      !out_map(&mdv, dv, dt, pr.B, pr.Tk, pr.HK, pr.D))
    return GD_ERR_LAUNCH;
  auto ctas = [](long long rows) { return (unsigned)((rows + 16 * kRowsEach - 1) / (16 * kRowsEach)); };
  const ValueRows vr = {v, st[6], st[7], st[8], (long long)pr.Tk * pr.HK, pr.HK, ctas((long long)pr.Tq * pr.H)};
  const unsigned blocks = vr.first + (std::is_same<T, __half>::value ? ctas(vr.rows) : 0);
  delta_kernel<T><<<dim3(blocks, (unsigned)pr.B), 256, 0, stream>>>(
      static_cast<const T*>(o), static_cast<const T*>(low), static_cast<const T*>(g), st[9], st[10], st[11], delta, pr.Tq,
      pr.H, pr.D, vr, err);
  static bool done_q[kMaxDevices], done_kv[kMaxDevices];
  auto kq = dq_kernel<T, NS>;
  auto kkv = dkv_kernel<T, NS>;
  if (set_smem_once(kq, DqCfg<NS>::kSmem, done_q) != cudaSuccess ||
      set_smem_once(kkv, DkvCfg<NS>::kSmem, done_kv) != cudaSuccess)
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  const long long qt = pr.cu ? packed_items(pr.Tq, pr.N) : (pr.Tq + kTile - 1) / kTile;
  const long long kt = (pr.cu ? packed_items(pr.Tk, pr.N) : (pr.Tk + kTile - 1) / kTile) + (long long)sp.heavy * (sp.parts - 1);
  kq<<<dim3((unsigned)qt, (unsigned)pr.H, (unsigned)pr.B), kThreads, DqCfg<NS>::kSmem, stream>>>(
      mq, mk, mv, mo, mdq, pr, lse, delta, static_cast<T*>(dq), err);
  kkv<<<dim3((unsigned)kt, (unsigned)(pr.HK * (NS == 4 ? 2 : 1)), (unsigned)pr.B), kThreads + 32, DkvCfg<NS>::kSmem, stream>>>(
      mq, mk, mv, mo, mdk, mdv, pr, sp, lse, delta, static_cast<T*>(dk), static_cast<T*>(dv), err);
  if (sp.parts > 1)
    sum_parts<T><<<dim3((unsigned)((kTile * pr.D / 4 + 255) / 256), (unsigned)(2 * sp.heavy), (unsigned)(pr.B * pr.HK)), 256,
                   0, stream>>>(sp.part, static_cast<T*>(dk), static_cast<T*>(dv), pr.Tk, pr.HK, pr.D, sp.heavy, sp.parts);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

}  // namespace

int backward(const void* q, const void* k, const void* v, const void* o, const void* low, const void* g,
             const long long* strides, const Problem& pr, int dtype, const float* lse, float* delta, void* dq, void* dk, void* dv, int heavy,
             int parts, float* part, ErrorWord* err, cudaStream_t stream) {
  const Split sp = {heavy, parts, part};
  auto run = [&](auto t, auto ns) {
    return launch<decltype(t), decltype(ns)::value>(q, k, v, o, low, g, strides, pr, lse, delta, dq, dk, dv, sp, err, stream);
  };
  auto by_width = [&](auto t) {
    return pr.D <= 64    ? run(t, std::integral_constant<int, 1>{})
           : pr.D <= 128 ? run(t, std::integral_constant<int, 2>{})
                         : run(t, std::integral_constant<int, 4>{});
  };
  return dtype == GD_FLOAT16 ? by_width(__half{}) : by_width(__nv_bfloat16{});
}

}  // namespace wattn
}  // namespace gd
