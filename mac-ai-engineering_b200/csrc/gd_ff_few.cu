// The gated feed-forward block for few tokens (a decoding step's): both products are as long as the weights are to read.
//   first kernel:  h = silu(x Wg^T) * (x Wu^T)        second:  y = h Wd^T
// Bound by the weights' bytes, 6 D F for a call. The weights are the M side of the products (a tile of 128 of their rows; in the
// first kernel 64 of w_gate's and the same 64 of w_up's), the tokens the N side (16 to 128, zeros past the last), so a tile's
// weights pass through a CTA once, by TMA through a ring of stages, three CTAs an SM. The contraction is
// split over a cluster of CTAs: few tiles still put bytes in flight on every SM, and all CTAs run at once, where memory, not their
// share of the SMs, decides when they end. Their partial products are added in shared memory of the cluster, in a fixed order.
// The second kernel starts while the first one ends (programmatic launch): its ring fills with weights before h is waited for.
#include "gd_ff.cuh"
#include "gd_gemm.cuh"

namespace gd {
namespace ff {
namespace {

using gemm::kBlockK;
constexpr int kRowsM = 128;      // rows of weights a tile has
constexpr int kThreads = 32 * 6; // warps 0 - 3: epilogue, 4: loads, 5: products

struct FewParams {
  CUtensorMap w[2], t;  // weights (the second kernel: w[0] alone), tokens
  int n, cols, blocks;  // tokens; the output's columns; stages of the whole contraction
  long long ld;         // elements from row to row of the output
  void* out;            // [n, cols]
};

template <int N>
struct FewCfg {
  static constexpr int kW = kRowsM * 128, kT = N * 128;  // bytes of a stage: weights, tokens
  // three CTAs an SM: at 16 tokens, 4,096 x 12,288 four stages take 53 us, five (two CTAs an SM) 58 us, three 55 us
  static constexpr int kStages = N == 16 ? 4 : N <= 64 ? 3 : 2;
  static constexpr int kRing = kStages * (kW + kT);
  static constexpr int kPart = N * kRowsM * 4;           // a CTA's partial products (in the ring's place)
  static_assert(kPart <= kRing, "partial products");
  static_assert(3 * (kRing + 2304) <= 227 * 1024, "three CTAs an SM");
  static constexpr size_t kSmem = 1024 + kRing + 8 * (2 * kStages + 1) + 16;
  static constexpr int kCols = N < 32 ? 32 : N;          // TMEM columns
};

__device__ __forceinline__ void load_box(uint32_t lead, uint32_t dst, const CUtensorMap* m, int x, int y, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}\n" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(smem_u32(bar)), "r"(lead)
      : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// GATED: the first kernel. gridDim.x = tiles * (cluster size).
template <typename T, int N, bool GATED>
__global__ void __launch_bounds__(kThreads) few_kernel(const __grid_constant__ FewParams p) {
  using C = FewCfg<N>;
  constexpr int kFeatures = GATED ? kRowsM / 2 : kRowsM;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(base + C::kRing);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  uint32_t size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const uint32_t rank = gemm::cluster_rank();
  const int tile = blockIdx.x / size, f0 = tile * kFeatures;
  const int from = (int)((long long)p.blocks * rank / size), to = (int)((long long)p.blocks * (rank + 1) / size);

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(tslot, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, *tslot, 0), s_base = smem_u32(base);
  // (the first kernel's inputs may come from the kernel before it in the stream, which need not know of this)
  if (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  bool fed = true;  // (the products' warp) no wait for a stage gave up
  if (warp == 4) {
    const uint32_t lead = wattn::elect();
    const int total = to - from;
    auto weights = [&](int i) {
      const int slot = i % C::kStages, k = (from + i) * kBlockK;
      const uint32_t a = s_base + slot * (C::kW + C::kT);
      if (lead) mbar_arrive_expect_tx(full + slot, C::kW + C::kT);
      load_box(lead, a, &p.w[0], k, f0, full + slot);
      load_box(lead, a + C::kW / 2, GATED ? &p.w[1] : &p.w[0], k, GATED ? f0 : f0 + 64, full + slot);
    };
    auto tokens = [&](int i) {
      const int slot = i % C::kStages;
      load_box(lead, s_base + slot * (C::kW + C::kT) + C::kW, &p.t, (from + i) * kBlockK, 0, full + slot);
    };
    const int first = total < C::kStages ? total : C::kStages;
    for (int i = 0; i < first; ++i) weights(i);
    if (!GATED) asm volatile("griddepcontrol.wait;\n\tfence.proxy.async;" ::: "memory");  // h
    for (int i = 0; i < first; ++i) tokens(i);
    int i = first;
    for (; i < total; ++i) {
      if (!gemm::warp_wait(empty + i % C::kStages, (i / C::kStages - 1) & 1, nullptr, 0)) break;
      weights(i);
      tokens(i);
    }
    for (int j = i > C::kStages ? i - C::kStages : 0; j < i; ++j)  // the copies in flight land before the CTA ends
      gemm::warp_wait(full + j % C::kStages, (j / C::kStages) & 1, nullptr, 0);
  } else if (warp == 5) {
    const uint32_t lead = wattn::elect();
    const int total = to - from;
    constexpr uint32_t id = wattn::idesc<T>(kRowsM, N, false);
    for (int i = 0; i < total; ++i) {
      const int slot = i % C::kStages;
      if (!(fed = gemm::warp_wait(full + slot, (i / C::kStages) & 1, nullptr, 0))) break;
      tc_fence_after();
      const uint32_t a = wattn::desc_k(s_base + slot * (C::kW + C::kT)), b = wattn::desc_k(s_base + slot * (C::kW + C::kT) + C::kW);
#pragma unroll
      for (int k = 0; k < kBlockK / 16; ++k) wattn::mma_ss(lead, tm, a + 2 * k, b + 2 * k, id, i > 0 || k > 0);
      wattn::mma_commit(lead, empty + slot);
    }
    wattn::mma_commit(lead, done);
    gemm::warp_wait(done, 0, nullptr, 0);
  }
  const bool ok = __syncthreads_and(warp >= 4 ? fed : gemm::warp_wait(done, 0, nullptr, 0)) != 0;
  float* const part = reinterpret_cast<float*>(base);  // [token][row of the tile]; the ring is read and its copies have landed
  if (warp < 4) {
    tc_fence_after();
    const float bad = ok ? 0.f : NAN;
#pragma unroll 1
    for (int c = 0; c < N; c += 16) {
      float v[16];
      if (to > from) {
        tmem_ld16(tm + ((uint32_t)(warp * 32) << 16) + c, v);
      } else {  // (a contraction of fewer stages than CTAs)
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * kRowsM + threadIdx.x] = v[i] + bad;
    }
  }
  tc_fence_before();
  __syncthreads();
  gemm::cluster_sync();  // all partial products are there
  // a CTA adds its share of the tile's outputs, the CTAs' parts in their order
  T* const out = static_cast<T*>(p.out);
  const int cells = p.n * kFeatures;
  for (int i = rank * kThreads + threadIdx.x; i < cells; i += size * kThreads) {
    const int t = i / kFeatures, f = i - t * kFeatures;
    const uint32_t at = s_base + (t * kRowsM + f) * 4;
    float a = 0.f, b = 0.f;
    for (uint32_t r = 0; r < size; ++r) {
      uint32_t there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(r));
      a += ld_cluster(there);
      if (GATED) b += ld_cluster(there + kRowsM / 2 * 4);
    }
    if (f0 + f < p.cols) out[t * p.ld + f0 + f] = cvt_out<T>(GATED ? a * gemm::sigmoid(a) * b : a);
  }
  if (warp == 5) tmem_dealloc(tm, C::kCols);
  gemm::cluster_sync();  // the parts are read
}

// CTAs of a cluster: as many as still run all at once, three on each of 148 SMs (memory then works at its rate whatever the
// SMs' shares are), but eight at most (the second product of a block 2,048 wide has 16 tiles, and so 128 CTAs of the 444 that
// fit; 4,096 wide 256), and none with less than four stages. At 4 tokens, 2,048 x 6,144 that is four (20 us; a fifth, and with it a
// second turn of CTAs: 23 us; one CTA an SM: 23 us), at 64 tokens, 4,096 x 12,288 two (60 us; one: 66, four: 69 us); at
// 1 token, 1,024 x 2,816 the least length holds (9.6 us; two stages: 11 us).
int split_of(int tiles, int blocks) {
  int s = 3 * 148 / tiles;
  if (s > 8) s = 8;
  if (s > blocks / 4) s = blocks / 4;
  return s < 1 ? 1 : s;
}

template <typename T, int N, bool GATED>
int launch(const FewParams& p, int tiles, bool early, cudaStream_t stream) {
  static bool done[kMaxDevices];
  auto kern = few_kernel<T, N, GATED>;
  if (set_smem_once(kern, FewCfg<N>::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  const int split = split_of(tiles, p.blocks);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split)), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = FewCfg<N>::kSmem;
  cfg.stream = stream, cfg.attrs = at, cfg.numAttrs = early ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

template <typename T, int N>
int run(const Problem& q, void* h, void* y, cudaStream_t stream) {
  constexpr CUtensorMapDataType dt = map_dtype<T>();
  FewParams p = {};
  p.n = q.rows, p.cols = q.F, p.blocks = gemm::blocks_of(q.D, kBlockK), p.out = h, p.ld = pitch(q.F);
  if (!gemm::matrix_map(&p.w[0], q.wg, dt, q.F, q.D, q.ldg, 64) || !gemm::matrix_map(&p.w[1], q.wu, dt, q.F, q.D, q.ldu, 64) ||
      !gemm::matrix_map(&p.t, q.x, dt, q.rows, q.D, q.ldx, N))
    return GD_ERR_LAUNCH;
  if (const int st = launch<T, N, true>(p, gemm::blocks_of(q.F, kRowsM / 2), false, stream)) return st;
  p.cols = q.O, p.blocks = gemm::blocks_of(q.F, kBlockK), p.out = y, p.ld = q.O;
  if (!gemm::matrix_map(&p.w[0], q.wd, dt, q.O, q.F, q.ldd, 64) || !gemm::matrix_map(&p.t, h, dt, q.rows, q.F, pitch(q.F), N))
    return GD_ERR_LAUNCH;
  return launch<T, N, false>(p, gemm::blocks_of(q.O, kRowsM), true, stream);
}

template <typename T>
int run_as(const Problem& q, void* h, void* y, cudaStream_t stream) {
  return q.rows <= 16   ? run<T, 16>(q, h, y, stream)
         : q.rows <= 32 ? run<T, 32>(q, h, y, stream)
         : q.rows <= 64 ? run<T, 64>(q, h, y, stream)
                        : run<T, 128>(q, h, y, stream);
}

}  // namespace

int forward_few(const Problem& q, int dtype, void* h, void* y, cudaStream_t stream) {
  return dtype == GD_FLOAT16 ? run_as<__half>(q, h, y, stream) : run_as<__nv_bfloat16>(q, h, y, stream);
}

}  // namespace ff
}  // namespace gd
