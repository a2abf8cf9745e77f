// Causal softmax attention with a sliding window and first tokens that stay visible, forward:
//   S = scale Q K^T over the visible keys,  P = exp(S - max),  O = P V / sum P,  L = log2 of the sum of exp2(S log2 e)
// in one pass over the keys with a running maximum and sum (fp32); O stays in TMEM between key tiles. A query without a
// visible key gets zeros and L = +inf.
//
// One CTA takes 128 queries of a head. Roles: warps 0-7 softmax (TMEM lane = query row; two threads a row, 64 key columns
// each, which agree on the row's maximum through shared memory when it moves), warp 8 loads (TMA), warp 9 issues the
// products. Key tiles outside the window and past the first tokens are never loaded.
//   S (128 x 128 fp32) comes from tcgen05 into TMEM; the softmax writes P over it as 16-bit pairs, where it is the A
//   operand of P V (no trip through shared memory). P is rounded to the inputs' 16-bit type (the operand type of the
//   matrix instruction); its sum is taken before the rounding, in fp32.
//   The maximum that P refers to moves only when a row outgrows it by 2^8: O is rescaled in TMEM then (rarely), and P
//   stays below 2^8, far inside both 16-bit types.
// D <= 128: two CTAs share an SM (<= 113 KB of shared memory, 256 TMEM columns each), so that one's products run under
// the other's softmax. D <= 256: one CTA an SM, S double-buffered: the products of the next tile run under the softmax.
#include "gd_wattn.cuh"

namespace gd {
namespace wattn {
namespace {

constexpr int kWarpsSm = 8;                     // softmax: two threads a query row, 64 columns each
constexpr int kThreads = 32 * (kWarpsSm + 2);   // + loads, + products
constexpr float kMaxGrowth = 8.f;  // log2

template <int NS>
struct Cfg {
  static constexpr int kBufs = NS == 4 ? 2 : 1;            // S buffers
  static constexpr int kSlots = NS == 1 ? 4 : 2;           // K / V tiles in shared memory
  static constexpr int kTileBytes = NS * kSlabBytes;
  static constexpr int kCols = NS == 4 ? 512 : 256;        // TMEM columns
  static constexpr int kO = kBufs * 128;                   // O's first column
  static constexpr int kBarriers = 1 + 2 * kSlots + 2 * kBufs + 2;
  static constexpr size_t kSmem = 1024 + (size_t)kTileBytes * (1 + kSlots) + 8 * kBarriers + 64 + 8 * kTile;
};

template <typename T, int NS>
__global__ void __launch_bounds__(kThreads, NS == 4 ? 1 : 2)
    fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
               const __grid_constant__ CUtensorMap mv, const Problem pr, T* __restrict__ o, T* __restrict__ o_low,
               float* __restrict__ lse,
               ErrorWord* err) {
  using C = Cfg<NS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + C::kTileBytes * (1 + C::kSlots));
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;
  uint64_t* empty = full + C::kSlots;
  uint64_t* s_full = empty + C::kSlots;
  uint64_t* p_full = s_full + C::kBufs;
  uint64_t* o_done = p_full + C::kBufs;
  uint64_t* fin = o_done + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + C::kBarriers);
  int* info = reinterpret_cast<int*>(tslot + 1);  // the packed sequence and tile of this CTA
  float* xchg = reinterpret_cast<float*>(bars + C::kBarriers) + 16;  // [2][128]: a row's two threads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < C::kBufs; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, kWarpsSm);
    }
    mbar_init(o_done, 1);
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
  if (pr.cu != nullptr) {
    if (warp == 0) {
      tile = find_item(pr.cu, pr.N, pr.Tq, item, [](int n) { return (n + kTile - 1) / kTile; }, sq);
      if (lane == 0) {
        info[0] = tile;
        info[1] = sq.q0;
        info[2] = sq.Tq;
      }
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
  } else {
    sq = {(int)blockIdx.z, 0, pr.Tq, 0, pr.Tk};
  }
  const uint32_t tm = *tslot;
  const int i0 = tile * kTile;
  const int i1 = i0 + kTile - 1 < sq.Tq - 1 ? i0 + kTile - 1 : sq.Tq - 1;
  const int p0 = i0 + sq.offset(), p1 = i1 + sq.offset();
  const KeyRange kr(tile < 0 ? -1 : p0, tile < 0 ? -1 : p1, pr.window, pr.sinks);
  const uint32_t s_q = smem_u32(base), s_kv = s_q + C::kTileBytes;

  if (warp == kWarpsSm) {
    if (lane == 0 && kr.n > 0) {
      const int hk = h / (pr.H / pr.HK);
      mbar_arrive_expect_tx(q_full, C::kTileBytes);
      load_tile<NS>(s_q, &mq, h, sq.q0 + i0, sq.b, q_full);
      int c = 0;
      bool ok = true;
      for (; c < 2 * kr.n; ++c) {
        const int slot = c % C::kSlots, use = c / C::kSlots;
        if (use > 0 && !(ok = mbar_wait(empty + slot, (use - 1) & 1, err, 60))) break;
        mbar_arrive_expect_tx(full + slot, C::kTileBytes);
        load_tile<NS>(s_kv + slot * C::kTileBytes, (c & 1) ? &mv : &mk, hk, sq.k0 + kr.key(c >> 1), sq.b, full + slot);
      }
      // the copies in flight land before the CTA ends, whatever became of their readers
      mbar_wait(q_full, 0, err, 61);
      for (int l = c > C::kSlots ? c - C::kSlots : 0; l < c; ++l) mbar_wait(full + l % C::kSlots, (l / C::kSlots) & 1, err, 61);
    }
  } else if (warp == kWarpsSm + 1) {
    if (lane == 0 && kr.n > 0) {
      bool ok = mbar_wait(q_full, 0, err, 62);
      auto scores = [&](int j) {  // S of tile j
        const int c = 2 * j, slot = c % C::kSlots, buf = j % C::kBufs;
        if (!mbar_wait(full + slot, (c / C::kSlots) & 1, err, 63)) return false;
        if (j >= C::kBufs && !mbar_wait(o_done, (j - C::kBufs) & 1, err, 64)) return false;  // P of the buffer is read
        tc_fence_after();
        mma_xyt<T, NS>(tm + buf * 128, s_q, s_kv + slot * C::kTileBytes);
        mma_commit(empty + slot);
        mma_commit(s_full + buf);
        return true;
      };
      for (int j = 0; ok && j < C::kBufs - 1 && j < kr.n; ++j) ok = scores(j);
      for (int j = 0; ok && j < kr.n; ++j) {
        if (j + C::kBufs - 1 < kr.n) ok = scores(j + C::kBufs - 1);
        const int c = 2 * j + 1, slot = c % C::kSlots, buf = j % C::kBufs;
        ok = ok && mbar_wait(full + slot, (c / C::kSlots) & 1, err, 65) && mbar_wait(p_full + buf, (j / C::kBufs) & 1, err, 66);
        if (!ok) break;
        tc_fence_after();
        mma_py<T, NS>(tm + C::kO, tm + buf * 128, s_kv + slot * C::kTileBytes, j > 0, 32);
        mma_commit(empty + slot);
        mma_commit(o_done);
      }
      mma_commit(fin);
      mbar_wait(fin, 0, err, 67);
    }
  } else if (tile >= 0) {
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;  // TMEM lane, which 64 columns
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int pair = 1 + (warp & 3);  // named barrier of the two warps that share 32 rows
    const int p = p0 + row;
    float m = -INFINITY;             // the maximum P refers to (log2 units, of scaled scores): the same in both threads
    F2 l2 = f2(0.f, 0.f);            // this thread's part of the sum
    bool ok = true;                  // (a failed wait leaves the loop's barriers in step: both warps go on without waiting)
    for (int j = 0; j < kr.n; ++j) {
      const int buf = j % C::kBufs;
      ok = ok && warp_wait(s_full + buf, (j / C::kBufs) & 1, err, 68);
      tc_fence_after();
      const uint32_t ts = tm + lanes + buf * 128 + half * 64;
      float s[64];
      tmem_ld64(ts, s);
      const int c0 = kr.key(j);
      if (!all_visible(c0, p0, p1, pr.window, pr.sinks)) {
        const uint32_t v0 = visible_keys(c0 + half * 64, p, pr.window, pr.sinks);
        const uint32_t v1 = visible_keys(c0 + half * 64 + 32, p, pr.window, pr.sinks);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = (v0 >> i) & 1 ? s[i] : -INFINITY;
          s[32 + i] = (v1 >> i) & 1 ? s[32 + i] : -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < 60; i += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[i + 2 * e], s[i + 2 * e + 1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[60 + e]);
      float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * pr.scale_log2;
      // does a row of the two warps outgrow its reference (or meet its first visible key)?
      uint32_t any;
      asm volatile(
          "{\n\t.reg .pred a, b;\n\t"
          "setp.ne.u32 a, %1, 0;\n\t"
          "barrier.cta.red.or.pred b, %2, 64, a;\n\t"
          "selp.u32 %0, 1, 0, b;\n\t}\n"
          : "=r"(any)
          : "r"((uint32_t)(top > m + kMaxGrowth)), "r"(pair)
          : "memory");
      if (any) {
        xchg[half * 128 + row] = top;
        asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair) : "memory");
        top = fmaxf(top, xchg[(half ^ 1) * 128 + row]);
        const bool grow = top > m + kMaxGrowth;
        const float next = grow ? top : m;
        const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2(m - next);
        l2 = mul2(l2, f2(f, f));
        if (j > 0) {  // O of the tiles so far, once their products are done; half of its columns each
          ok = ok && warp_wait(o_done, (j - 1) & 1, err, 69);
          tc_fence_after();
#pragma unroll 1
          for (int c = half * NS * 32; c < (half + 1) * NS * 32; c += 16) {
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
      const float ref = m == -INFINITY ? 0.f : m;
      const F2 sc = f2(pr.scale_log2, pr.scale_log2), rf = f2(-ref, -ref);
      F2 acc = f2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float a, b;
          unf2(fma2(f2(s[c + i], s[c + i + 1]), sc, rf), a, b);
          a = ex2(a);
          b = ex2(b);
          acc = add2(acc, f2(a, b));
          u[i / 2] = pack16<T>(a, b);
        }
        tmem_st16(ts + c, u);  // over this thread's own columns, a piece of 32 keys every 32 words
      }
      l2 = add2(l2, acc);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(p_full + buf);
    }
    if (kr.n > 0) {
      ok = ok && warp_wait(o_done, (kr.n - 1) & 1, err, 70);
      tc_fence_after();
    }
    float l, lb;
    unf2(l2, l, lb);
    l += lb;
    xchg[half * 128 + row] = l;  // (every row had its exchanges of the loop before the last barrier there)
    asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair) : "memory");
    l = xchg[row] + xchg[128 + row];
    const int i = i0 + row;
    const bool live = i < sq.Tq;
    const float inv = !ok ? NAN : l == 0.f ? 0.f : 1.f / l;  // a wait that gave up leaves NaN
    if (live && half == 0) lse[((long long)sq.b * pr.H + h) * pr.Tq + sq.q0 + i] = l == 0.f ? INFINITY : m + log2f(l);
    const long long at = (((long long)sq.b * pr.Tq + sq.q0 + i) * pr.H + h) * pr.D;
    const bool none = l == 0.f && ok;  // a row without a visible key: zeros, whatever O's columns hold
#pragma unroll 1
    for (int c = half * NS * 32; c < (half + 1) * NS * 32; c += 32) {
      float v[32];
      if (kr.n > 0) tmem_ld32(tm + lanes + C::kO + c, v);
      if (!live) continue;
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        if (c + k >= pr.D) break;
        uint32_t u[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = none ? 0.f : v[k + 2 * e] * inv, b = none ? 0.f : v[k + 2 * e + 1] * inv;
          u[e] = pack16<T>(a, b);
          const float2 r = unpack16<T>(u[e]);
          w[e] = pack16<T>(a - r.x, b - r.y);
        }
        *reinterpret_cast<uint4*>(o + at + c + k) = make_uint4(u[0], u[1], u[2], u[3]);
        // what the rounding took away, for the backward's delta
        if (o_low != nullptr) *reinterpret_cast<uint4*>(o_low + at + c + k) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
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
  CUtensorMap mq, mk, mv;
  if (!tile_map(&mq, q, map_dtype<T>(), pr.B, pr.Tq, pr.H, pr.D, st[0], st[1], st[2], kTile) ||
      !tile_map(&mk, k, map_dtype<T>(), pr.B, pr.Tk, pr.HK, pr.D, st[3], st[4], st[5], kTile) ||
      !tile_map(&mv, v, map_dtype<T>(), pr.B, pr.Tk, pr.HK, pr.D, st[6], st[7], st[8], kTile))
    return GD_ERR_LAUNCH;
  static bool done[kMaxDevices];
  auto kern = fwd_kernel<T, NS>;
  if (set_smem_once(kern, Cfg<NS>::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const long long tiles = pr.cu ? (long long)pr.Tq / kTile + pr.N : (pr.Tq + kTile - 1) / kTile;
  const dim3 grid((unsigned)tiles, (unsigned)pr.H, (unsigned)pr.B);
  kern<<<grid, kThreads, Cfg<NS>::kSmem, stream>>>(mq, mk, mv, pr, static_cast<T*>(o), static_cast<T*>(low), lse, err);
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
