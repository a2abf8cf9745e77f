// The gated delta rule's recurrent form, for single tokens and short runs over kept states. For each request and value head,
// with the state S [DK, DV] in fp32, token after token:
//   S <- exp(g) S,   d = beta (v - S^T k),   S <- S + k d^T,   o = S^T q
// (q and k l2-normalised where asked, q scaled by DK^-1/2). Both products with the state are taken before d is known:
//   o = exp(g) (S^T q) + (q . k) d,
// so a token costs one pass over S in registers and one join over the rows.
//
// Bound by memory: 8 DK DV bytes of a head's state for about 7 DK DV operations a token. The state is read once into
// registers, run through all tokens of the call, and written once. A CTA takes a slice of a head's value columns (the
// recurrence never mixes them): a thread holds four adjacent columns of ROWS rows, a row group of lanes reads a row's slice
// as whole 128-byte lines.
#include <cstdint>

#include "gd_common.cuh"

namespace gd {
namespace rule_step {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRun = 8;         // tokens whose rows are staged at a time
constexpr int kMaxWidth = 256;  // DK, DV

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

// Whether request b's written slot is read or written by another request of the call (the whole CTA; one answer).
__device__ __forceinline__ bool contested(const Args& a, int b, int to) {
  bool hit = false;
  for (int j = threadIdx.x; j < a.B; j += kThreads)
    if (j != b) {
      const int x = __ldg(a.in + j), y = __ldg(a.out + j);
      hit |= x >= 0 && y >= 0 && (x == to || y == to);  // (an idle request reads and writes nothing)
    }
  return __syncthreads_or(hit) != 0;
}

// W: columns a CTA takes; ROWS: rows a thread holds (ROWS * 256 * 4 / W >= DK).
template <typename T, typename TV, int W, int ROWS>
__global__ void __launch_bounds__(kThreads) step_kernel(const Args a) {
  constexpr int LC = W / 4;             // lanes across a row's slice
  constexpr int RG = kThreads / LC;     // rows a pass of all threads covers
  __shared__ __align__(16) float sk[kRun][kMaxWidth], sq[kRun][kMaxWidth];
  __shared__ __align__(16) float sv[kRun][W];
  __shared__ float s_qk[kRun], s_decay[kRun], s_beta[kRun];
  __shared__ __align__(16) float red[2][2][kWarps][W];  // [token parity][k, q][warp][column]

  const int b = blockIdx.y, slices = (a.DV + W - 1) / W, h = blockIdx.x / slices, c0 = (blockIdx.x - h * slices) * W;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cl = threadIdx.x % LC, rg = threadIdx.x / LC, col = c0 + cl * 4;
  const int hk = h / (a.H / a.HK);
  const bool mine = col < a.DV;  // (DV is a multiple of 4)
  const int from = a.in == nullptr ? b : __ldg(a.in + b), to = a.out == nullptr ? b : __ldg(a.out + b);
  const long long rows0 = (long long)b * a.T;
  T* const o = static_cast<T*>(a.o);

  // an idle request gives zeros; one whose slot does not exist, or that another request writes or reads, gives NaN; neither
  // touches the states
  const bool idle = from < 0 || to < 0;
  const bool bad = !idle && (from >= a.slots || to >= a.slots || (a.out != nullptr && contested(a, b, to)));
  if (idle || bad) {
    const float x = idle ? 0.f : NAN;
    for (int t = rg; t < a.T; t += RG)
      if (mine)
        for (int i = 0; i < 4; ++i) o[((rows0 + t) * a.H + h) * a.DV + col + i] = cvt_out<T>(x);
    return;
  }

  float4 s[ROWS];
  const long long head = ((long long)a.H * from + h) * a.DK;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = rg + i * RG;
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.s_in != nullptr && mine && r < a.DK)
      s[i] = __ldcs(reinterpret_cast<const float4*>(a.s_in + (head + r) * a.DV + col));
  }

  for (int t0 = 0; t0 < a.T; t0 += kRun) {
    const int n = a.T - t0 < kRun ? a.T - t0 : kRun;
    if (t0 > 0) __syncthreads();  // the rows of the tokens before are read
    // q and k of token t0 + j by warp j: normalised, scaled, and their product
    for (int j = warp; j < n; j += kWarps) {
      const T* q = static_cast<const T*>(a.q) + ((rows0 + t0 + j) * a.HK + hk) * a.DK;
      const T* k = static_cast<const T*>(a.k) + ((rows0 + t0 + j) * a.HK + hk) * a.DK;
      float x[kMaxWidth / 32], y[kMaxWidth / 32], qq = 0.f, kk = 0.f, qk = 0.f;
#pragma unroll
      for (int i = 0; i < kMaxWidth / 32; ++i) {
        const int d = lane + 32 * i;
        x[i] = d < a.DK ? to_f32<T>(q[d]) : 0.f;
        y[i] = d < a.DK ? to_f32<T>(k[d]) : 0.f;
        qq = fmaf(x[i], x[i], qq);
        kk = fmaf(y[i], y[i], kk);
      }
      float fq = rsqrtf((float)a.DK), fk = 1.f;
      if (a.l2norm) {
        fq *= rsqrtf(warp_sum(qq) + 1e-6f);
        fk = rsqrtf(warp_sum(kk) + 1e-6f);
      }
#pragma unroll
      for (int i = 0; i < kMaxWidth / 32; ++i) {
        const int d = lane + 32 * i;
        x[i] *= fq;
        y[i] *= fk;
        qk = fmaf(x[i], y[i], qk);
        sq[j][d] = x[i];
        sk[j][d] = y[i];
      }
      qk = warp_sum(qk);
      const long long row = (rows0 + t0 + j) * a.H + h;
      if (lane == 0) {
        s_qk[j] = qk;
        s_decay[j] = expf(a.g[row]);
        s_beta[j] = a.beta[row];
      }
      for (int c = lane; c < W; c += 32)
        sv[j][c] = c0 + c < a.DV ? to_f32<TV>(static_cast<const TV*>(a.v)[row * a.DV + c0 + c]) : 0.f;
    }
    __syncthreads();
    for (int j = 0; j < n; ++j) {
      const float decay = s_decay[j];
      float4 pk = make_float4(0.f, 0.f, 0.f, 0.f), pq = pk;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float k = sk[j][rg + i * RG], q = sq[j][rg + i * RG];  // (zeros past DK)
        pk.x = fmaf(k, s[i].x, pk.x);
        pk.y = fmaf(k, s[i].y, pk.y);
        pk.z = fmaf(k, s[i].z, pk.z);
        pk.w = fmaf(k, s[i].w, pk.w);
        pq.x = fmaf(q, s[i].x, pq.x);
        pq.y = fmaf(q, s[i].y, pq.y);
        pq.z = fmaf(q, s[i].z, pq.z);
        pq.w = fmaf(q, s[i].w, pq.w);
      }
#pragma unroll
      for (int m = LC; m < 32; m *= 2) {  // the warp's row groups
        pk.x += __shfl_xor_sync(0xffffffffu, pk.x, m);
        pk.y += __shfl_xor_sync(0xffffffffu, pk.y, m);
        pk.z += __shfl_xor_sync(0xffffffffu, pk.z, m);
        pk.w += __shfl_xor_sync(0xffffffffu, pk.w, m);
        pq.x += __shfl_xor_sync(0xffffffffu, pq.x, m);
        pq.y += __shfl_xor_sync(0xffffffffu, pq.y, m);
        pq.z += __shfl_xor_sync(0xffffffffu, pq.z, m);
        pq.w += __shfl_xor_sync(0xffffffffu, pq.w, m);
      }
      float(*rk)[W] = red[j & 1][0], (*rq)[W] = red[j & 1][1];
      if (lane < LC) {
        *reinterpret_cast<float4*>(&rk[warp][cl * 4]) = pk;
        *reinterpret_cast<float4*>(&rq[warp][cl * 4]) = pq;
      }
      __syncthreads();  // (the other parity's sums are read before the next token's barrier)
      float4 d = make_float4(0.f, 0.f, 0.f, 0.f), y = d;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 u = *reinterpret_cast<const float4*>(&rk[w][cl * 4]);
        d.x += u.x;
        d.y += u.y;
        d.z += u.z;
        d.w += u.w;
      }
      const float4 v = *reinterpret_cast<const float4*>(&sv[j][cl * 4]);
      const float bt = s_beta[j];
      d.x = bt * (v.x - decay * d.x);
      d.y = bt * (v.y - decay * d.y);
      d.z = bt * (v.z - decay * d.z);
      d.w = bt * (v.w - decay * d.w);
      if (rg == 0 && mine) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 u = *reinterpret_cast<const float4*>(&rq[w][cl * 4]);
          y.x += u.x;
          y.y += u.y;
          y.z += u.z;
          y.w += u.w;
        }
        const float qk = s_qk[j];
        T* p = o + ((rows0 + t0 + j) * a.H + h) * a.DV + col;
        p[0] = cvt_out<T>(fmaf(qk, d.x, decay * y.x));
        p[1] = cvt_out<T>(fmaf(qk, d.y, decay * y.y));
        p[2] = cvt_out<T>(fmaf(qk, d.z, decay * y.z));
        p[3] = cvt_out<T>(fmaf(qk, d.w, decay * y.w));
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float k = sk[j][rg + i * RG];
        s[i].x = fmaf(k, d.x, decay * s[i].x);
        s[i].y = fmaf(k, d.y, decay * s[i].y);
        s[i].z = fmaf(k, d.z, decay * s[i].z);
        s[i].w = fmaf(k, d.w, decay * s[i].w);
      }
    }
  }
  if (a.s_out == nullptr || !mine) return;
  const long long dst = ((long long)a.H * to + h) * a.DK;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = rg + i * RG;
    if (r < a.DK) __stcs(reinterpret_cast<float4*>(a.s_out + (dst + r) * a.DV + col), s[i]);
  }
}

template <typename T, typename TV, int W, int ROWS>
int launch_as(const Args& a, cudaStream_t stream) {
  const dim3 grid((unsigned)(a.H * ((a.DV + W - 1) / W)), (unsigned)a.B);
  step_kernel<T, TV, W, ROWS><<<grid, kThreads, 0, stream>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, typename TV>
int launch(const Args& a, cudaStream_t stream) {
  return a.DK <= 128 ? launch_as<T, TV, 32, 4>(a, stream) : launch_as<T, TV, 32, 8>(a, stream);
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
  if (B < 0 || B > 65535 || T < 0 || H <= 0 || HK <= 0 || H % HK != 0 || H > (1 << 24) || DK <= 0 || DK % 32 != 0 ||
      DK > kMaxWidth || DV <= 0 || DV % 32 != 0 || DV > kMaxWidth || n_slots < 0 ||
      (slots == nullptr && n_slots < B))
    return GD_ERR_SHAPE;
  if (B == 0) return GD_OK;
  if ((slots == nullptr) != (out_slots == nullptr)) return GD_ERR_ARG;
  if (T > 0 && (q == nullptr || k == nullptr || v == nullptr || g == nullptr || beta == nullptr || o == nullptr))
    return GD_ERR_ARG;
  if (!aligned16(s_in) || !aligned16(s_out)) return GD_ERR_ALIGN;
  Args a;
  a.q = q, a.k = k, a.v = v, a.g = g, a.beta = beta, a.s_in = s_in, a.s_out = s_out, a.in = slots, a.out = out_slots;
  a.o = o, a.B = B, a.T = T, a.H = H, a.HK = HK, a.DK = DK, a.DV = DV, a.slots = n_slots;
  a.l2norm = (flags & GD_L2NORM) != 0;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (dtype == GD_FLOAT32) return launch<float, float>(a, cs);
  if (dtype == GD_FLOAT16) return vdtype == dtype ? launch<__half, __half>(a, cs) : launch<__half, float>(a, cs);
  return vdtype == dtype ? launch<__nv_bfloat16, __nv_bfloat16>(a, cs) : launch<__nv_bfloat16, float>(a, cs);
}
