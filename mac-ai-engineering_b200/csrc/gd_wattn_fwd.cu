// Causal softmax attention with a sliding window and first tokens that stay visible, forward:
//   S = scale Q K^T over the visible keys,  P = exp(S - max),  O = P V / sum P,  L = log2 of the sum of exp2(S log2 e)
// in one pass over the keys with a running maximum and sum (fp32); O stays in TMEM between key tiles. A query without a
// visible key gets zeros and L = +inf.
//
// One CTA takes 128 queries of a head. Roles: warps 0-3 softmax (a thread owns a query row, TMEM lane = row), warp 4 loads
// (TMA), warp 5 issues the products. Key tiles (128 keys) outside the window and past the first tokens are never loaded.
//   S comes from tcgen05 into TMEM in halves of 64 keys; the softmax writes a half's P over it as 16-bit pairs, where it is
//   the A operand of P V (no trip through shared memory). P is rounded to the inputs' 16-bit type (the operand type of the
//   matrix instruction); its sum is taken before the rounding, in fp32.
//   The maximum that P refers to moves only when a row outgrows it by 2^8: O is rescaled in TMEM then (rarely), and P
//   stays below 2^8. float16's P carries 2^7 more, up to the end of its range: it keeps its 11 bits down to 2^-21 of the
//   maximum's weight and is off by 2^-32 of it at most (many keys of 2^-25 beside one that outweighs them were lost together).
// D <= 128: two CTAs share an SM (<= 100 KB of shared memory, 256 TMEM columns each). While the softmax works on one half,
// the other half's P V and its next S run, so the softmax warps hardly wait: the exponentials (16 a clock and SM) and the
// products share the SM's time. S of 64 keys at a time costs the product 1.5 times its shared-memory reads of Q; S of 128
// keys in one buffer left every step's latency (4,200 clocks a tile and CTA) on the critical path.
// D <= 256: one CTA an SM, S of 128 keys double-buffered, K and V pass in halves of 128 channels through a ring of five.
// Measured (bf16, operations of visible pairs): 1 x 8192 x 16 heads (4 key heads), D 128, window 2048 139 us (870 TFLOP/s);
// 1 x 16384 x 16 causal D 128 1,150, D 256 1,010 TFLOP/s; D 64 with window 4096 395 us (615 TFLOP/s), where an exponential
// comes with half the operations of D 128 (special-function pipe 62 % busy, tensor pipe 31 %). cuBLAS: 1,641 TFLOP/s.
#include "gd_wattn.cuh"

namespace gd {
namespace wattn {
namespace {

constexpr int kWarpsSm = 4;
constexpr int kThreads = 32 * (kWarpsSm + 2);   // + loads, + products
constexpr float kMaxGrowth = 8.f;               // log2
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;  // log2 of what P carries

template <int NS>
struct Cfg {
  static constexpr bool kWide = NS == 4;
  static constexpr int kSets = kWide ? 2 : 1;              // buffers of S of 128 keys (two halves each)
  static constexpr int kUnit = (kWide ? 2 : NS) * kSlabBytes;
  static constexpr int kSlots = kWide ? 5 : NS == 1 ? 4 : 2;  // K / V units in shared memory
  static constexpr int kQBytes = NS * kSlabBytes;
  static constexpr int kCols = kWide ? 512 : 256;          // TMEM columns
  static constexpr int kO = kSets * 128;                   // O's first column
  static constexpr int kBarriers = 1 + 2 * kSlots + 4 * kSets + 3;
  static constexpr size_t kSmem = 1024 + kQBytes + (size_t)kUnit * kSlots + 8 * kBarriers + 64;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

template <typename T, int NS>
__global__ void __launch_bounds__(kThreads, NS == 4 ? 1 : 2)
    fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
               const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mo,
               const __grid_constant__ CUtensorMap ml, const Problem pr, T* __restrict__ o, T* __restrict__ o_low,
               float* __restrict__ lse, ErrorWord* err) {
  using C = Cfg<NS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::kQBytes + C::kUnit * C::kSlots);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;
  uint64_t* empty = full + C::kSlots;
  uint64_t* s_full = empty + C::kSlots;       // of each half
  uint64_t* p_full = s_full + 2 * C::kSets;
  // P V of half x: a phase a tile. Whoever waits on a phase is also needed for the next one of that barrier (a wait by
  // parity tells neighbouring phases apart, no more), hence a barrier for each half and one of its own for the end.
  uint64_t* o_done = p_full + 2 * C::kSets;
  uint64_t* fin = o_done + 2;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + C::kBarriers);
  int* info = reinterpret_cast<int*>(tslot + 1);  // the packed sequence and tile of this CTA
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2 * C::kSets; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, kWarpsSm);
    }
    mbar_init(o_done, 1);
    mbar_init(o_done + 1, 1);
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == kWarpsSm + 1) {
    tmem_alloc(tslot, C::kCols);
    tmem_relinquish();
  }
  // the queries: later tiles see more keys, so they start first
  const int item = gridDim.x - 1 - blockIdx.x, h = blockIdx.y;
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
  const uint32_t s_q = smem_u32(base), s_kv = s_q + C::kQBytes;

  if (warp == kWarpsSm) {
    if (lane == 0 && kr.n > 0) {
      const int hk = h / (pr.H / pr.HK);
      constexpr int kPer = C::kWide ? 2 : 1;  // units of a tile
      mbar_arrive_expect_tx(q_full, C::kQBytes);
      load_tile<NS>(s_q, &mq, h, sq.q0 + i0, sq.b, q_full);
      int c = 0;
      for (; c < 2 * kPer * kr.n; ++c) {  // K's units, V's units, of tile after tile
        const int slot = c % C::kSlots, use = c / C::kSlots, j = c / (2 * kPer), x = c % (2 * kPer);
        if (use > 0 && !mbar_wait(empty + slot, (use - 1) & 1, err, 60)) break;
        mbar_arrive_expect_tx(full + slot, C::kUnit);
        const CUtensorMap* m = x < kPer ? &mk : &mv;
        if constexpr (C::kWide) load_half(s_kv + slot * C::kUnit, m, x & 1, hk, sq.k0 + kr.key(j), sq.b, full + slot);
        else load_tile<NS>(s_kv + slot * C::kUnit, m, hk, sq.k0 + kr.key(j), sq.b, full + slot);
      }
      // the copies in flight land before the CTA ends, whatever became of their readers
      mbar_wait(q_full, 0, err, 61);
      for (int l = c > C::kSlots ? c - C::kSlots : 0; l < c; ++l) mbar_wait(full + l % C::kSlots, (l / C::kSlots) & 1, err, 61);
    }
  } else if (warp == kWarpsSm + 1) {
    if (kr.n > 0) {
      const uint32_t lead = elect();
      bool ok = warp_wait(q_full, 0, err, 62);
      if (pr.negate) negate_tile<NS>(s_q);  // from here on the scale is positive
      auto landed = [&](int c) { return warp_wait(full + c % C::kSlots, (c / C::kSlots) & 1, err, 63); };
      auto values = [&](int c, int j) {  // the same for a unit of tile j's values
        if (!landed(c)) return false;
        if (pr.cu != nullptr) zero_rows<C::kUnit / kSlabBytes>(s_kv + c % C::kSlots * C::kUnit, sq.Tk - kr.key(j));
        return true;
      };
      if constexpr (!C::kWide) {
        // units: K(j) = 2 j, V(j) = 2 j + 1; half x of tile j is half-tile 2 j + x
        auto scores = [&](int j, int x) {
          const int c = 2 * j;
          if (x == 0 && !landed(c)) return false;
          if (j > 0 && !warp_wait(o_done + x, (j - 1) & 1, err, 64)) return false;  // P over these columns is read
          tc_fence_after();
          mma_xyt<T, NS, 64>(lead, tm + 64 * x, s_q, s_kv + c % C::kSlots * C::kUnit + x * 64 * 128);
          mma_commit(lead, s_full + x);
          if (x == 1) mma_commit(lead, empty + c % C::kSlots);
          return true;
        };
        ok = ok && scores(0, 0) && scores(0, 1);
        for (int j = 0; ok && j < kr.n; ++j) {
          const int c = 2 * j + 1;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (x == 0) ok = values(c, j);
            if (!(ok = ok && warp_wait(p_full + x, j & 1, err, 66))) break;
            tc_fence_after();
            mma_py<T, NS, 4>(lead, tm + C::kO, tm + 64 * x, s_kv + c % C::kSlots * C::kUnit + x * 64 * 128, j > 0 || x > 0, 16);
            if (x == 1) mma_commit(lead, empty + c % C::kSlots);
            mma_commit(lead, o_done + x);
            if (j + 1 < kr.n && !(ok = scores(j + 1, x))) break;
          }
        }
      } else {
        // units: K(j) = 4 j, 4 j + 1 and V(j) = 4 j + 2, 4 j + 3, by halves of the channels
        auto scores = [&](int j) {
          if (j >= 2 && !warp_wait(o_done + 1, j & 1, err, 64)) return false;  // of tile j - 2: P over these columns is read
          const uint32_t d = tm + (j & 1) * 128;
          for (int y = 0; y < 2; ++y) {
            const int c = 4 * j + y;
            if (!landed(c)) return false;
            tc_fence_after();
            mma_xyt<T, 2>(lead, d, s_q + y * 2 * kSlabBytes, s_kv + c % C::kSlots * C::kUnit, y > 0);
            mma_commit(lead, empty + c % C::kSlots);
          }
          mma_commit(lead, s_full + 2 * (j & 1));
          mma_commit(lead, s_full + 2 * (j & 1) + 1);
          return true;
        };
        ok = ok && scores(0);
        for (int j = 0; ok && j < kr.n; ++j) {
          if (j + 1 < kr.n && !(ok = scores(j + 1))) break;
          const int c = 4 * j + 2, set = j & 1;
          ok = values(c, j) && values(c + 1, j);
          for (int x = 0; ok && x < 2; ++x) {
            if (!(ok = warp_wait(p_full + 2 * set + x, (j >> 1) & 1, err, 66))) break;
            tc_fence_after();
            for (int y = 0; y < 2; ++y) {
              const int v = (c + y) % C::kSlots;
              mma_py<T, 2, 4>(lead, tm + C::kO + y * 128, tm + set * 128 + 64 * x, s_kv + v * C::kUnit + x * 64 * 128,
                              j > 0 || x > 0, 16);
              if (x == 1) mma_commit(lead, empty + v);
            }
            mma_commit(lead, o_done + x);
          }
        }
      }
      mma_commit(lead, fin);
      warp_wait(fin, 0, err, 67);
    }
  } else if (tile >= 0) {
    const int row = threadIdx.x;  // TMEM lane
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int p = p0 + row;
    float m = -INFINITY;  // the maximum P refers to (log2 units, of scaled scores)
    F2 l2 = f2(0.f, 0.f);
    bool ok = true;
    const F2 sc = f2(pr.scale_log2, pr.scale_log2);
    for (int t = 0; ok && t < 2 * kr.n; ++t) {  // half-tiles
      const int j = t >> 1, x = t & 1, b = C::kWide ? t & 3 : x, phase = C::kWide ? j >> 1 : j;
      if (!(ok = warp_wait(s_full + b, phase & 1, err, 68))) break;
      // half-tile t - 2 is over (D <= 128: its S was issued after that), so that the wait below cannot take an older phase
      // for its own
      if (C::kWide && j > 0 && !(ok = warp_wait(o_done + x, (j - 1) & 1, err, 71))) break;
      tc_fence_after();
      const uint32_t ts = tm + lanes + b * 64;
      float s[64];
      tmem_ld64(ts, s);
      const int c0 = kr.key(j) + 64 * x;
      if (!all_visible(kr.key(j), p0, p1, pr.window, pr.sinks)) {
        const uint32_t v0 = visible_keys(c0, p, pr.window, pr.sinks), v1 = visible_keys(c0 + 32, p, pr.window, pr.sinks);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = (v0 >> i) & 1 ? s[i] : -INFINITY;
          s[32 + i] = (v1 >> i) & 1 ? s[32 + i] : -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};  // (a NaN score makes the maximum NaN, and with it the row)
#pragma unroll
      for (int i = 4; i < 60; i += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[i + 2 * e], s[i + 2 * e + 1]);
      }
      const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], s[60], s[61]), max3(s[62], s[63], s[62])) * pr.scale_log2;
      const bool grow = !(top <= m + kMaxGrowth);  // also a row's first visible key, and NaN
      if (__any_sync(0xffffffffu, grow)) {
        const float next = grow ? top : m;
        const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2(m - next);
        l2 = mul2(l2, f2(f, f));
        if (t > 0) {  // O of the half-tiles so far, once their products are done
          if (!(ok = warp_wait(o_done + (x ^ 1), (x == 0 ? j - 1 : j) & 1, err, 69))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < NS * 64; c += 16) {
            float v[16];
            uint32_t u[16];
            tmem_ld16(tm + lanes + C::kO + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[i] * f);
            tmem_st16(tm + lanes + C::kO + c, u);
          }
        }
        m = next;
      }
      const float ref = m == -INFINITY ? 0.f : m - kLift<T>;
      const F2 rf = f2(-ref, -ref);
      F2 acc = f2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float a, e;
          ex2_pair(fma2(f2(s[c + i], s[c + i + 1]), sc, rf), a, e);
          acc = add2(acc, f2(a, e));
          u[i / 2] = pack16<T>(a, e);
        }
        tmem_st16(ts + c / 2, u);
      }
      l2 = add2(l2, acc);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(p_full + b);
    }
    if (kr.n > 0) {
      ok = ok && warp_wait(fin, 0, err, 70);  // all products
      tc_fence_after();
    }
    float l, lb;
    unf2(l2, l, lb);
    l += lb;
    const int i = i0 + row;
    // A row without a visible key (its own is visible from position 0 on): zeros, whatever O's columns hold. A row whose
    // visible scores are all -inf has a sum of 0 and comes out as NaN.
    const bool none = ok && (kr.n == 0 || p < 0);
    const float inv = !ok ? NAN : none ? 0.f : 1.f / l;  // a wait that gave up leaves NaN
    if (i < sq.Tq && lse != nullptr)
      lse[((long long)sq.b * pr.H + h) * pr.Tq + sq.q0 + i] = none ? INFINITY : m - kLift<T> + log2f(l);
    // out through shared memory (Q's place and the first key unit's; a warp's own 32 rows), so that rows leave as whole lines
    // (16-byte stores a thread and row took 5 us a CTA); o_low: what the rounding took away, for the backward's delta
    const bool low = o_low != nullptr;
#pragma unroll 2
    for (int c = 0; c < NS * 64; c += 32) {
      float v[32];
      if (kr.n > 0) {
        tmem_ld32(tm + lanes + C::kO + c, v);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        uint32_t u[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = none ? 0.f : v[k + 2 * e] * inv, d = none ? 0.f : v[k + 2 * e + 1] * inv;
          u[e] = pack16<T>(a, d);
          const float2 r = unpack16<T>(u[e]);
          w[e] = pack16<T>(a - r.x, d - r.y);
        }
        const uint32_t at = tile_at(row, (c + k) >> 3);
        st_shared16(s_q + at, u);
        if (low) st_shared16(s_kv + at, w);
      }
    }
    store_rows<T, NS>(&mo, o, s_q, warp * 32, sq.b, sq.q0 + i0, sq.Tq - i0, pr.Tq, h, pr.H, pr.D);
    if (low) store_rows<T, NS>(&ml, o_low, s_kv, warp * 32, sq.b, sq.q0 + i0, sq.Tq - i0, pr.Tq, h, pr.H, pr.D);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpsSm + 1) {
    tc_fence_after();
    tmem_dealloc(tm, C::kCols);
  }
}

template <typename T, int NS>
int launch(const void* q, const void* k, const void* v, const long long* st, const Problem& pr, void* o, void* low, float* lse,
           ErrorWord* err, cudaStream_t stream) {
  CUtensorMap mq, mk, mv, mo, ml;
  if (!tile_map(&mq, q, map_dtype<T>(), pr.B, pr.Tq, pr.H, pr.D, st[0], st[1], st[2], kTile) ||
      !tile_map(&mk, k, map_dtype<T>(), pr.B, pr.Tk, pr.HK, pr.D, st[3], st[4], st[5], kTile) ||
      !tile_map(&mv, v, map_dtype<T>(), pr.B, pr.Tk, pr.HK, pr.D, st[6], st[7], st[8], kTile) ||
      !out_map(&mo, o, map_dtype<T>(), pr.B, pr.Tq, pr.H, pr.D) ||
      !out_map(&ml, low != nullptr ? low : o, map_dtype<T>(), pr.B, pr.Tq, pr.H, pr.D))
    return GD_ERR_LAUNCH;
  static bool done[kMaxDevices];
  auto kern = fwd_kernel<T, NS>;
  if (set_smem_once(kern, Cfg<NS>::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const long long tiles = pr.cu ? packed_items(pr.Tq, pr.N) : (pr.Tq + kTile - 1) / kTile;
  const dim3 grid((unsigned)tiles, (unsigned)pr.H, (unsigned)pr.B);
  kern<<<grid, kThreads, Cfg<NS>::kSmem, stream>>>(mq, mk, mv, mo, ml, pr, static_cast<T*>(o), static_cast<T*>(low), lse, err);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

}  // namespace

int forward(const void* q, const void* k, const void* v, const long long* strides, const Problem& pr, int dtype, void* o,
            void* low, float* lse, ErrorWord* err, cudaStream_t stream) {
  if (dtype == GD_FLOAT16)
    return pr.D <= 64    ? launch<__half, 1>(q, k, v, strides, pr, o, low, lse, err, stream)
           : pr.D <= 128 ? launch<__half, 2>(q, k, v, strides, pr, o, low, lse, err, stream)
                         : launch<__half, 4>(q, k, v, strides, pr, o, low, lse, err, stream);
  return pr.D <= 64    ? launch<__nv_bfloat16, 1>(q, k, v, strides, pr, o, low, lse, err, stream)
         : pr.D <= 128 ? launch<__nv_bfloat16, 2>(q, k, v, strides, pr, o, low, lse, err, stream)
                       : launch<__nv_bfloat16, 4>(q, k, v, strides, pr, o, low, lse, err, stream);
}

}  // namespace wattn
}  // namespace gd
