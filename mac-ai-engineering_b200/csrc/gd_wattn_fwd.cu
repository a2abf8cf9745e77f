// Causal softmax attention with a sliding window and first tokens that stay visible, forward:
//   S = scale Q K^T over the visible keys,  P = exp(S - max),  O = P V / sum P,  L = log2 of the sum of exp2(S log2 e)
// in one pass over the keys with a running maximum and sum (fp32); O stays in TMEM between key tiles. A query without a
// visible key gets zeros and L = +inf.
//
// One CTA takes 128 queries of a head. Roles: warps 0-3 softmax (a thread owns a query row, TMEM lane = row), warp 4
// loads (TMA), warp 5 issues the products. Key tiles outside the window and past the first tokens are never loaded.
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

constexpr int kThreads = 192;
constexpr float kMaxGrowth = 8.f;  // log2

template <int NS>
struct Cfg {
  static constexpr int kBufs = NS == 4 ? 2 : 1;            // S buffers
  static constexpr int kSlots = NS == 1 ? 4 : 2;           // K / V tiles in shared memory
  static constexpr int kTileBytes = NS * kSlabBytes;
  static constexpr int kCols = NS == 4 ? 512 : 256;        // TMEM columns
  static constexpr int kO = kBufs * 128;                   // O's first column
  static constexpr int kBarriers = 1 + 2 * kSlots + 2 * kBufs + 2;
  static constexpr size_t kSmem = 1024 + (size_t)kTileBytes * (1 + kSlots) + 8 * kBarriers + 64;
};

template <typename T, int NS>
__global__ void __launch_bounds__(kThreads, NS == 4 ? 1 : 2)
    fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
               const __grid_constant__ CUtensorMap mv, const Problem pr, T* __restrict__ o, float* __restrict__ lse,
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < C::kBufs; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4);
    }
    mbar_init(o_done, 1);
    mbar_init(fin, 1);
    fence_mbar_init();
  }
  if (warp == 5) {
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

  if (warp == 4) {
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
  } else if (warp == 5) {
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
        mma_py<T, NS>(tm + C::kO, tm + buf * 128, s_kv + slot * C::kTileBytes, j > 0);
        mma_commit(empty + slot);
        mma_commit(o_done);
      }
      mma_commit(fin);
      mbar_wait(fin, 0, err, 67);
    }
  } else if (tile >= 0) {
    const int row = threadIdx.x;  // TMEM lane
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int p = p0 + row;
    float m = -INFINITY, l = 0.f;  // running maximum (log2 units, of scaled scores) and sum
    bool ok = true;
    for (int j = 0; j < kr.n; ++j) {
      const int buf = j % C::kBufs;
      if (!(ok = warp_wait(s_full + buf, (j / C::kBufs) & 1, err, 68))) break;
      tc_fence_after();
      const uint32_t ts = tm + lanes + buf * 128;
      float s[128];
      tmem_ld128(ts, s);
      const int c0 = kr.key(j);
      if (!all_visible(c0, p0, p1, pr.window, pr.sinks)) {
        // visible: key <= p, and key > p - window or key < sinks
        const int last = p - c0, from = p - pr.window + 1 - c0, sink = pr.sinks - c0;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > last || (i < from && i >= sink)) s[i] = -INFINITY;
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * pr.scale_log2;
      const bool grow = top > m + kMaxGrowth;  // also the first finite maximum
      if (__any_sync(0xffffffffu, grow)) {
        const float next = grow ? top : m;
        const float f = m == -INFINITY ? 0.f : ex2(m - next);
        l *= f;
        if (j > 0) {  // O of the tiles so far, once their products are done
          if (!(ok = warp_wait(o_done, (j - 1) & 1, err, 69))) break;
          tc_fence_after();
          const float g = grow ? f : 1.f;
#pragma unroll 1
          for (int c = 0; c < NS * 64; c += 32) {
            float v[32];
            uint32_t u[32];
            tmem_ld32(tm + lanes + C::kO + c, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(v[i] * g);
            tmem_st32(tm + lanes + C::kO + c, u);
          }
        }
        m = next;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t u[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float a = ex2(fmaf(s[c + i], pr.scale_log2, -ref)), b = ex2(fmaf(s[c + i + 1], pr.scale_log2, -ref));
          sum[i & 2] += a;
          sum[(i & 2) + 1] += b;
          u[i / 2] = pack16<T>(a, b);
        }
        tmem_st16(ts + c / 2, u);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive_warp(p_full + buf);
    }
    if (ok && kr.n > 0) {
      ok = warp_wait(o_done, (kr.n - 1) & 1, err, 70);
      tc_fence_after();
    }
    const int i = i0 + row;
    const bool live = i < sq.Tq;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN scores stay NaN
    if (live) lse[((long long)sq.b * pr.H + h) * pr.Tq + sq.q0 + i] = l == 0.f ? INFINITY : m + log2f(l);
    T* out = o + (((long long)sq.b * pr.Tq + sq.q0 + i) * pr.H + h) * pr.D;
#pragma unroll 1
    for (int c = 0; c < NS * 64 && c < pr.D; c += 32) {
      float v[32];
      if (kr.n > 0) {
        tmem_ld32(tm + lanes + C::kO + c, v);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = 0.f;
      }
      if (!live) continue;
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        if (c + k >= pr.D) break;
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a wait that gave up leaves NaN; a row without a visible key zeros
          const float a = !ok ? NAN : l == 0.f ? 0.f : v[k + 2 * e] * inv, b = !ok ? NAN : l == 0.f ? 0.f : v[k + 2 * e + 1] * inv;
          u[e] = pack16<T>(a, b);
        }
        *reinterpret_cast<uint4*>(out + c + k) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tm, C::kCols);
  }
}

template <typename T, int NS>
int launch(const void* q, const void* k, const void* v, const long long* st, const Problem& pr, void* o, float* lse,
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
  kern<<<grid, kThreads, Cfg<NS>::kSmem, stream>>>(mq, mk, mv, pr, static_cast<T*>(o), lse, err);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

}  // namespace

int forward(const void* q, const void* k, const void* v, const long long* strides, const Problem& pr, int dtype, void* o,
            float* lse, ErrorWord* err, cudaStream_t stream) {
  if (dtype == GD_FLOAT16)
    return pr.D <= 64    ? launch<__half, 1>(q, k, v, strides, pr, o, lse, err, stream)
           : pr.D <= 128 ? launch<__half, 2>(q, k, v, strides, pr, o, lse, err, stream)
                         : launch<__half, 4>(q, k, v, strides, pr, o, lse, err, stream);
  return pr.D <= 64    ? launch<__nv_bfloat16, 1>(q, k, v, strides, pr, o, lse, err, stream)
         : pr.D <= 128 ? launch<__nv_bfloat16, 2>(q, k, v, strides, pr, o, lse, err, stream)
                       : launch<__nv_bfloat16, 4>(q, k, v, strides, pr, o, lse, err, stream);
}

}  // namespace wattn
}  // namespace gd
