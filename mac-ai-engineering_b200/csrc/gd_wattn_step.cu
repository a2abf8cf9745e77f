// The single-token form of the sliding-window attention, over a cache: each request's new key and value are stored in
// their slot and the query attends to the visible positions, the new one included,
//   o = sum_j softmax_j(scale q k_j) v_j     over j <= p and (j > p - window or j < sinks),  p = lengths[b].
// Position j lives in slot j while j < S, then in slot sinks + (j - sinks) mod (S - sinks): a linear cache, or a rolling
// one that keeps its first `sinks` tokens. A request with a negative length is idle: zeros, nothing stored.
//
// Bound by the cache's bytes: a key and a value row are read once for all the query heads of their head (16 at most per
// CTA, the rows of one matrix instruction; the products use mma.sync, since 16 x 16 tiles fed by 16-byte asynchronous
// copies are far from any arithmetic limit). The visible positions of a (request, key head) are split over a cluster of
// up to 8 CTAs of four warps; every warp streams its own 16-key steps through its own stages (no barrier in the loop)
// with a running maximum and sum in fp32, and the parts are joined through distributed shared memory: one launch. When
// requests are too few to fill the GPU that way, several clusters share a (request, key head) and a second kernel joins
// their sums. Measured (bf16): 64 requests on rolling caches of 4,160 slots, 32 heads on 4 key heads of 128: 82 us (6.2
// TB/s, 95 % of a plain copy); one request at 777 positions, 16 heads on 2 of 256: 10.5 us, all latency.
#include <cooperative_groups.h>

#include <cmath>

#include "gd_common.cuh"

namespace gd {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;   // keys a warp takes at a time
constexpr int kRows = 16;   // query heads of a CTA
constexpr int kMaxClusters = 32;
constexpr int kSms = 148;   // of a B200
// log2 of what P carries before its rounding: float16's, at most 1 otherwise, would lose the keys that weigh less than 2^-14
// of the maximum (all 11 bits now down to 2^-29); the sums carry it too, and o is their quotient
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.f : 0.f;
static_assert(kThreads == 8 * kRows, "the join's factors: eight threads a row");

template <int DP>
struct Cfg {
  static constexpr int kStages = 3;
  static constexpr int kHalf = kStep * DP * 2;  // a step's keys (or values)
  static constexpr int kWarpBytes = kStages * 2 * kHalf;
  static constexpr int kQBytes = kRows * DP * 2 > 2304 ? kRows * DP * 2 : 2304;
  static constexpr size_t kSmem = kQBytes + kWarps * (size_t)kWarpBytes + 2 * kWarps * kRows * sizeof(float);
  static_assert(kWarpBytes >= kRows * DP * 4, "a warp's sums fit in its stages");
  static_assert(kQBytes >= (8 * kWarps + 2) * kRows * 4, "the join's factors fit in Q's place");
};

struct StepArgs {
  const void *q, *k, *v;  // [B, H, D], [B, HK, D]
  void *kc, *vc, *o;
  const int* lengths;
  long long kb, ks, kh, vb, vs, vh;  // cache strides in elements
  int B, S, H, HK, D, window, sinks, groups;  // groups: CTA rows of 16 query heads per key head
  float scale_log2;
  float* part;  // [B][HK groups][clusters][16][2 + D]
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ T to16(float x) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The positions a request's query sees, in order: `head` first tokens, then from .. p; and their slots.
struct Seen {
  int p, head, from, n, slot0, S, ring;
  __device__ __forceinline__ Seen(int len, int S_, int window, int sinks) : p(len), S(S_) {
    head = from = n = slot0 = 0;
    ring = S - sinks;
    if (len < 0) return;
    const int w = len < S ? window : (window < ring ? window : ring);  // a rolling cache holds no more
    from = len - w + 1 > 0 ? len - w + 1 : 0;
    head = sinks < from ? sinks : from;
    n = head + len - from + 1;
    slot0 = from < S ? from : sinks + (int)((unsigned)(from - sinks) % (unsigned)ring);
  }
  __device__ __forceinline__ int slot(int i) const {  // of visible position i
    if (i < head) return i;
    const long long s = (long long)slot0 + i - head;
    return (int)(s < S ? s : s - ring);
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) step_kernel(const StepArgs a) {
  using C = Cfg<DP>;
  constexpr int kChunks = DP / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y / a.groups, g0 = blockIdx.y % a.groups * kRows, b = blockIdx.z;
  const int G = a.H / a.HK, rows = G - g0 < kRows ? G - g0 : kRows;
  cg::cluster_group cluster = cg::this_cluster();
  const int cs = (int)cluster.num_blocks();
  const Seen seen(__ldg(a.lengths + b), a.S, a.window, a.sinks);
  // this CTA's share, in whole steps
  const int steps = (seen.n + kStep - 1) / kStep;
  const int s0 = (int)((long long)steps * blockIdx.x / gridDim.x), s1 = (int)((long long)steps * (blockIdx.x + 1) / gridDim.x);

  // Q, rows past the group and channels past D zero
  const uint32_t sq = smem_u32(smem);
  const T* q = static_cast<const T*>(a.q) + ((long long)b * a.H + hk * G + g0) * a.D;
  for (int i = threadIdx.x; i < kRows * kChunks; i += kThreads) {
    const int r = i / kChunks, c = i % kChunks;
    const bool live = r < rows && c * 8 < a.D;
    cp16(sq + r * DP * 2 + ((c ^ (r & 7)) << 4), live ? q + (long long)r * a.D + c * 8 : q, live);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");

  const T* kn = static_cast<const T*>(a.k) + ((long long)b * a.HK + hk) * a.D;
  const T* vn = static_cast<const T*>(a.v) + ((long long)b * a.HK + hk) * a.D;
  T* kc = static_cast<T*>(a.kc) + b * a.kb + hk * a.kh;
  T* vc = static_cast<T*>(a.vc) + b * a.vb + hk * a.vh;
  // the share that holds the new token stores it (no CTA reads that slot from the cache)
  if (seen.n > 0 && s1 == steps && s0 < s1 && g0 == 0) {
    const long long at = seen.slot(seen.n - 1);
    for (int c = threadIdx.x; c * 8 < a.D; c += kThreads) {
      *reinterpret_cast<uint4*>(kc + at * a.ks + c * 8) = *reinterpret_cast<const uint4*>(kn + c * 8);
      *reinterpret_cast<uint4*>(vc + at * a.vs + c * 8) = *reinterpret_cast<const uint4*>(vn + c * 8);
    }
  }

  const uint32_t stages = sq + C::kQBytes + warp * C::kWarpBytes;
  auto load = [&](int s, int stage) {  // step s of the visible positions; rows past the last are zeros
    const uint32_t dst = stages + stage * 2 * C::kHalf;
    const int first = s * kStep, at0 = seen.slot(first);
    if (s >= s1) {
    } else if (first + kStep < seen.n && (first >= seen.head || first + kStep <= seen.head) &&
               seen.slot(first + kStep - 1) == at0 + kStep - 1) {
      // adjacent slots, none of them the new token's: a lane keeps its channels and walks the rows (the general way below
      // takes twice the instructions of everything else in the step)
      constexpr int kRowsAtOnce = 32 / kChunks > 0 ? 32 / kChunks : 1;
      const int r0 = lane / kChunks, c = lane % kChunks;
      const bool live = c * 8 < a.D;
      const T* pk = kc + (long long)(at0 + r0) * a.ks + (live ? c * 8 : 0);
      const T* pv = vc + (long long)(at0 + r0) * a.vs + (live ? c * 8 : 0);
#pragma unroll
      for (int r = 0; r < kStep; r += kRowsAtOnce) {
        const int row = r + r0;
        const uint32_t d = dst + row * DP * 2 + ((c ^ (row & 7)) << 4);
        cp16(d, pk, live);
        cp16(d + C::kHalf, pv, live);
        pk += kRowsAtOnce * a.ks;
        pv += kRowsAtOnce * a.vs;
      }
    } else {
#pragma unroll 1
      for (int i = lane; i < kStep * kChunks; i += 32) {
        const int r = i / kChunks, c = i % kChunks, at = s * kStep + r;
        const bool live = at < seen.n && c * 8 < a.D;
        const bool newest = at == seen.n - 1;
        const long long slot = live ? seen.slot(at) : 0;
        const uint32_t d = dst + r * DP * 2 + ((c ^ (r & 7)) << 4);
        const int off = live ? c * 8 : 0;
        cp16(d, (newest ? kn : kc + slot * a.ks) + off, live);
        cp16(d + C::kHalf, (newest ? vn : vc + slot * a.vs) + off, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // of rows lane / 4 and lane / 4 + 8
  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) load(s0 + warp + i * kWarps, i);
  asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");  // Q, of all threads
  __syncthreads();
  // Q's fragments: in registers up to 128 channels
  constexpr bool kQRegs = DP <= 128;
  uint32_t qf[kQRegs ? DP / 16 : 1][4];
  const int r8 = lane & 7, mat = lane >> 3;
  auto q_at = [&](int k) {
    const int qr = r8 + (mat & 1) * 8, qc = 2 * k + (mat >> 1);
    return sq + qr * DP * 2 + ((qc ^ (qr & 7)) << 4);
  };
  if constexpr (kQRegs) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) ldsm4(qf[k], q_at(k));
  }
  int stage = 0;
  for (int s = s0 + warp; s < s1; s += kWarps) {
    __syncwarp();  // every lane is done with the stage that is loaded next
    load(s + (C::kStages - 1) * kWarps, stage == 0 ? C::kStages - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
    __syncwarp();
    const uint32_t sk = stages + stage * 2 * C::kHalf, sv = sk + C::kHalf;
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
    // S [16 heads x 16 keys]
    float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      uint32_t qa[4], kb[4];
      if constexpr (kQRegs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) qa[e] = qf[k][e];
      } else {
        ldsm4(qa, q_at(k));
      }
      const int kr = r8 + (mat >> 1) * 8, kcn = 2 * k + (mat & 1);
      ldsm4(kb, sk + kr * DP * 2 + ((kcn ^ (kr & 7)) << 4));
      mma16816<T>(c[0], qa, kb[0], kb[1]);
      mma16816<T>(c[1], qa, kb[2], kb[3]);
    }
    // keys 8 t + 2 (lane % 4) + e
    const int left = seen.n - s * kStep;  // keys of the step
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 8 * t + 2 * (lane & 3) + (e & 1);
        c[t][e] = key < left ? c[t][e] * a.scale_log2 : -INFINITY;
      }
    float t0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
    float t1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
    }
    if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1)) {
      const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
      const float f0 = m0 == -INFINITY ? 0.f : ex2f(m0 - n0), f1 = m1 == -INFINITY ? 0.f : ex2f(m1 - n1);
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        o[i][0] *= f0;
        o[i][1] *= f0;
        o[i][2] *= f1;
        o[i][3] *= f1;
      }
      m0 = n0;
      m1 = n1;
    }
    const float r0 = m0 == -INFINITY ? 0.f : m0 - kLift<T>, r1 = m1 == -INFINITY ? 0.f : m1 - kLift<T>;
    uint32_t pa[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float x0 = ex2f(c[t][0] - r0), x1 = ex2f(c[t][1] - r0), y0 = ex2f(c[t][2] - r1), y1 = ex2f(c[t][3] - r1);
      l0 += x0 + x1;
      l1 += y0 + y1;
      pa[2 * t] = pack<T>(x0, x1);
      pa[2 * t + 1] = pack<T>(y0, y1);
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      uint32_t vb[4];
      const int vr = r8 + (mat & 1) * 8, vcn = 2 * i + (mat >> 1);
      ldsm4t(vb, sv + vr * DP * 2 + ((vcn ^ (vr & 7)) << 4));
      mma16816<T>(o[2 * i], pa, vb[0], vb[1]);
      mma16816<T>(o[2 * i + 1], pa, vb[2], vb[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  // the warp's sums over its stages: [16][DP] fp32; maxima and sums beside them
#pragma unroll
  for (int w = 1; w <= 2; w <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, w);
    l1 += __shfl_xor_sync(0xffffffffu, l1, w);
  }
  float* acc = reinterpret_cast<float*>(smem + C::kQBytes + warp * C::kWarpBytes);
  float* ms = reinterpret_cast<float*>(smem + C::kQBytes + kWarps * C::kWarpBytes);  // [warp][16]
  float* ls = ms + kWarps * kRows;
  const int r = lane >> 2;
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
    const int c = 8 * i + 2 * (lane & 3);
    *reinterpret_cast<float2*>(acc + r * DP + c) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(acc + (r + 8) * DP + c) = make_float2(o[i][2], o[i][3]);
  }
  if ((lane & 3) == 0) {
    ms[warp * kRows + r] = m0;
    ms[warp * kRows + r + 8] = m1;
    ls[warp * kRows + r] = l0;
    ls[warp * kRows + r + 8] = l1;
  }
  cluster.sync();
  // each CTA of the cluster joins its share of the (head, channel) pairs over all its CTAs' warps (the parts), in order.
  // First the parts' factors exp2(maximum - overall maximum), and the overall sums: Q's place, free by now
  const int clusters = gridDim.x / cs, rank = (int)cluster.block_rank(), parts = cs * kWarps;
  float* fac = reinterpret_cast<float*>(smem);  // [part][16]
  float* tops = fac + 8 * kWarps * kRows;       // [16], then the sums [16]
  {
    const int row = threadIdx.x >> 3, x = threadIdx.x & 7;  // eight threads a row, a CTA of the cluster each
    const float* rm = cluster.map_shared_rank(ms, x < cs ? x : 0);
    const float* rl = cluster.map_shared_rank(ls, x < cs ? x : 0);
    float mw[kWarps], lw[kWarps], top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      mw[w] = x < cs ? rm[w * kRows + row] : -INFINITY;
      lw[w] = x < cs ? rl[w * kRows + row] : 0.f;
      top = fmaxf(top, mw[w]);
    }
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = mw[w] == -INFINITY ? 0.f : ex2f(mw[w] - top);
      if (x < cs) fac[(x * kWarps + w) * kRows + row] = f;
      l = fmaf(lw[w], f, l);
    }
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (x == 0) {
      tops[row] = top;
      tops[kRows + row] = l;
    }
  }
  __syncthreads();
  for (int i = rank * kThreads + threadIdx.x; i < rows * (a.D / 2); i += cs * kThreads) {
    const int row = i / (a.D / 2), c = i % (a.D / 2) * 2;
    const float top = tops[row], l = tops[kRows + row];
    float y0 = 0.f, y1 = 0.f;
#pragma unroll 8
    for (int x = 0; x < parts; ++x) {
      const float* ra = cluster.map_shared_rank(reinterpret_cast<float*>(smem + C::kQBytes), x / kWarps);
      const float2 z = *reinterpret_cast<const float2*>(ra + x % kWarps * (C::kWarpBytes / 4) + row * DP + c);
      const float f = fac[x * kRows + row];
      y0 = fmaf(z.x, f, y0);
      y1 = fmaf(z.y, f, y1);
    }
    // NaN scores appear in no maximum but in the sums, and stay NaN
    if (clusters > 1) {
      float* out = a.part + ((((long long)b * gridDim.y + blockIdx.y) * clusters + blockIdx.x / cs) * kRows + row) * (2 + a.D);
      if (c == 0) {
        out[0] = top;
        out[1] = l;
      }
      out[2 + c] = y0;
      out[3 + c] = y1;
    } else {
      const float inv = 1.f / l;  // a sum of 0 over visible keys (scores of -inf) gives NaN; an idle request zeros
      uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + ((long long)b * a.H + hk * G + g0 + row) * a.D + c);
      *out = seen.n == 0 ? 0u : pack<T>(y0 * inv, y1 * inv);
    }
  }
  cluster.sync();  // no CTA ends while another reads its shared memory
}

// Joins the clusters' sums, in order; one CTA per (CTA row of heads, request).
template <typename T>
__global__ void __launch_bounds__(256) step_join(const StepArgs a, int clusters) {
  const int hk = blockIdx.x / a.groups, g0 = blockIdx.x % a.groups * kRows, b = blockIdx.y;
  const int G = a.H / a.HK, rows = G - g0 < kRows ? G - g0 : kRows;
  const float* part = a.part + ((long long)b * gridDim.x + blockIdx.x) * clusters * kRows * (2 + a.D);
  const bool idle = __ldg(a.lengths + b) < 0;
  for (int i = threadIdx.x; i < rows * a.D; i += 256) {
    const int row = i / a.D, c = i % a.D;
    float top = -INFINITY, l = 0.f, y = 0.f;
    for (int x = 0; x < clusters; ++x) top = fmaxf(top, part[((long long)x * kRows + row) * (2 + a.D)]);
    for (int x = 0; x < clusters; ++x) {
      const float* p = part + ((long long)x * kRows + row) * (2 + a.D);
      const float f = p[0] == -INFINITY ? 0.f : ex2f(p[0] - top);
      l = fmaf(p[1], f, l);
      y = fmaf(p[2 + c], f, y);
    }
    static_cast<T*>(a.o)[((long long)b * a.H + hk * G + g0 + row) * a.D + c] = to16<T>(idle ? 0.f : y / l);
  }
}

// CTAs of a cluster and clusters per (request, key head): enough to give every SM a CTA, at least 64 keys (a step for
// each warp) a CTA at the most that can be visible; a second kernel's launch pays from 512 keys a CTA.
struct Split {
  int cs, clusters;
};
Split split_of(int B, int S, int HK, int groups, int window, int sinks) {
  long long most = window == 0 ? S : (long long)window + sinks;
  if (most > S) most = S;
  long long want = (kSms + (long long)B * HK * groups - 1) / ((long long)B * HK * groups);
  const long long fit = (most + kWarps * kStep - 1) / (kWarps * kStep);
  if (want > fit) want = fit;
  Split s = {1, 1};
  while (s.cs < 8 && s.cs * 2 <= want) s.cs *= 2;
  if (want > 8 && most > 8 * 512) s.clusters = (int)((want + 7) / 8 < kMaxClusters ? (want + 7) / 8 : kMaxClusters);
  return s;
}
size_t part_bytes(int B, int HK, int groups, int D, const Split& s) {
  return s.clusters > 1 ? (size_t)B * HK * groups * s.clusters * kRows * (2 + D) * sizeof(float) : 0;
}

template <typename T, int DP>
int launch(const StepArgs& a, const Split& s, cudaStream_t stream) {
  static bool done[kMaxDevices];
  auto kern = step_kernel<T, DP>;
  if (set_smem_once(kern, Cfg<DP>::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(s.cs * s.clusters), (unsigned)(a.HK * a.groups), (unsigned)a.B);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<DP>::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)s.cs;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  if (s.clusters > 1) {
    step_join<T><<<dim3((unsigned)(a.HK * a.groups), (unsigned)a.B), 256, 0, stream>>>(a, s.clusters);
    if (cudaPeekAtLastError() != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  }
  return GD_OK;
}
template <typename T>
int by_width(const StepArgs& a, const Split& s, cudaStream_t stream) {
  return a.D <= 64 ? launch<T, 64>(a, s, stream) : a.D <= 128 ? launch<T, 128>(a, s, stream) : launch<T, 256>(a, s, stream);
}

bool sizes_ok(int B, int S, int H, int HK, int D, int window, int sinks) {
  return B >= 0 && B <= 65535 && S > 0 && H > 0 && HK > 0 && H % HK == 0 && H <= 65535 && D > 0 && D % 8 == 0 && D <= 256 &&
         window >= 0 && sinks >= 0;
}
// Whether no two rows of D elements of a cache [B, S, HK] share memory: each stride passes what the smaller ones span (the
// kernel's CTAs write rows of their own at the same time).
bool rows_apart(const long long* st, int B, int S, int HK, int D) {
  long long x[3] = {st[0], st[1], st[2]}, n[3] = {B, S, HK};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (x[j] > x[j + 1]) {
        const long long a = x[j], b = n[j];
        x[j] = x[j + 1], n[j] = n[j + 1];
        x[j + 1] = a, n[j + 1] = b;
      }
  long long span = D;
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (x[i] < span || x[i] >= (1ll << 40)) return false;
    span += (n[i] - 1) * x[i];
  }
  return true;
}
int groups_of(int H, int HK) { return (H / HK + kRows - 1) / kRows; }

}  // namespace
}  // namespace gd

extern "C" size_t gd_wattn_step_workspace_bytes(int B, int S, int H, int HK, int D, int window, int sinks) {
  if (!gd::sizes_ok(B, S, H, HK, D, window, sinks) || B == 0) return 0;
  const int groups = gd::groups_of(H, HK);
  return gd::part_bytes(B, HK, groups, D, gd::split_of(B, S, HK, groups, window, sinks));
}

extern "C" int gd_wattn_step(const void* q, const void* k, const void* v, void* k_cache, void* v_cache, const int* lengths,
                             void* o, int dtype, int B, int S, int H, int HK, int D, const long long* strides, int window,
                             int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gd;
  if (dtype != GD_FLOAT16 && dtype != GD_BFLOAT16) return GD_ERR_ARG;
  if (!sizes_ok(B, S, H, HK, D, window, sinks) || !std::isfinite(scale)) return GD_ERR_SHAPE;
  if (B == 0) return GD_OK;
  if (q == nullptr || k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr || lengths == nullptr ||
      o == nullptr || strides == nullptr)
    return GD_ERR_ARG;
  uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                  reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
                  reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(workspace);
  for (int i = 0; i < 6; ++i) {
    const int n = i % 3 == 0 ? B : i % 3 == 1 ? S : HK;
    if (n > 1) all |= (uintptr_t)strides[i] * 2;
  }
  if (!rows_apart(strides, B, S, HK, D) || !rows_apart(strides + 3, B, S, HK, D)) return GD_ERR_ALIGN;
  if ((all & 15) != 0 || (reinterpret_cast<uintptr_t>(lengths) & 3) != 0) return GD_ERR_ALIGN;
  const int groups = groups_of(H, HK);
  const Split s = split_of(B, S, HK, groups, window, sinks);
  if (part_bytes(B, HK, groups, D, s) > 0 && (workspace == nullptr || workspace_bytes < part_bytes(B, HK, groups, D, s)))
    return GD_ERR_WORKSPACE;
  StepArgs a;
  a.q = q, a.k = k, a.v = v, a.kc = k_cache, a.vc = v_cache, a.o = o, a.lengths = lengths;
  a.kb = strides[0], a.ks = strides[1], a.kh = strides[2], a.vb = strides[3], a.vs = strides[4], a.vh = strides[5];
  a.B = B, a.S = S, a.H = H, a.HK = HK, a.D = D, a.groups = groups;
  a.window = window == 0 ? 0x7fffffff : window;
  a.sinks = sinks < S ? sinks : S - 1;  // a cache of first tokens only: all of them are visible anyway
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  return dtype == GD_FLOAT16 ? by_width<__half>(a, s, cs) : by_width<__nv_bfloat16>(a, s, cs);
}
