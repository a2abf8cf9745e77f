// Matrix products on tcgen05 with an epilogue each, the core of the gated feed-forward block (gd_ff.cu) and of the vocabulary
// projection's cross entropy (gd_xent.cu):  C[M, N] = sum over k of A[m, k] B[n, k],  16-bit operands, fp32 accumulators.
//
// Each operand is read where the caller has it: rows of k (K-major: a matrix whose rows are m or n) or rows of m or n
// (MN-major: a matrix whose rows are k); the tensor core takes both from the same 128-byte swizzled tiles, only descriptor and
// tensor map differ. TMA fills what lies past a matrix with zeros, so no size has to fill a tile.
//
// A pair of CTAs (cluster of two, tcgen05 cta_group::2) computes 256 x 256: each CTA holds its 128 rows of A and 128 of the 256
// rows of B, so that a product of 64 k reads 32 KB of shared memory an SM where a lone CTA's 128 x 256 would read 48 KB. Roles:
// warp 0 loads (TMA, a ring of stages), warp 1 of the first CTA issues the products, warps 4 - 11 are the epilogue (a thread
// owns a row and half of the tile's columns; TMEM lane = row). The accumulator is double-buffered (2 x 256 TMEM columns), so a
// tile's epilogue runs under the next one's products. The CTAs are persistent and walk the tiles of up to kMaxOps problems.
//
// Bound by the tensor pipe (97 % busy under four gradients at once) at the clock that the power limit leaves (1.45 to 1.6 GHz).
// bf16, 16,384 rows, 2,048 x 6,144: the second product 268 us (1,540 TFLOP/s; cuBLAS 264), gate and up 524 us (1,575), the four
// gradients 1,385 us (1,490). With g and u kept gate and up take 578 us, and dh 413 us (1,000): their epilogues' 0.8 and 1.2 GB
// cross between the SMs and L2 beside the operands' (dh without its loads 350 us, without its stores 333, without both 281;
// neither TMA nor the warps' own accesses, 8 or 16 epilogue warps, 4 or 5 stages changed that by more than 3 %). Cross entropy,
// 7,370 rows, 2,048 x 128,000: logits 2.87 to 3.15 ms (1,230 to 1,350), with their gradients stored 2.96 to 3.28 ms, its two
// gradients 5.9 to 6.65 ms, all at the clocks of a long run (1.3 to 1.45 GHz). 777 rows, 50,257 words: the logits 128 us at 1.54
// GHz, 93 % of the tensor pipe.
#pragma once

#include <utility>

#include "gd_wattn.cuh"

namespace gd {
namespace gemm {

using wattn::elect;
using wattn::ex2;
using wattn::pack16;
using wattn::st_shared16;
using wattn::warp_wait;

constexpr int kBlockK = 64;            // k of a stage: one 128-byte row of the swizzle
constexpr int kHalf = 128;             // rows of A, and of B, that a CTA holds
constexpr int kTileM = 256, kTileN = 256;
constexpr int kOperand = kHalf * 128;  // bytes of a CTA's part of an operand's stage
constexpr int kStage = 2 * kOperand;
constexpr int kSlab = 32 * 128;        // a warp's 32 rows of 64 16-bit columns, on their way out
constexpr int kStrip = 32 * 64;        // the same of 32 columns, in or out (64-byte swizzle)
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (4 + kEpiWarps);
constexpr int kMaxOps = 4;
constexpr int kGroupM = 8;             // row tiles that are walked together, column tile after column tile (L2)
constexpr float kLog2e = 1.4426950408889634f;
// Stages whose time a tile's way out takes, where its contraction is shorter (64 rows, 2,048 wide, 128,000 words, both gradients'
// products, one stage a tile of dW: 222 us; counted as 4 stages 251, 12 227, as it is 390)
constexpr int kLeast = 8;
constexpr int kRun = 12;  // stages of a logit's run, at most (see sums_in_runs)

enum Epilogue {
  kStore,    // C, times a factor, in 16 bits; or summed over calls in fp32 (see Op::sum)
  kSwiglu,   // B's two halves are the gate's and the up projection's rows: h = silu(g) u (and g, u where kept)
  kDSwiglu,  // C = dh: dg, du (and h again) from the kept g, u
  kLse,      // each row's maximum and sum of exponentials over the tile's columns, and its label's logit
  kDLogit    // (softmax - onehot) times the row's factor, in 16 bits
};

// The tensor core's adder cuts off what lies below its accumulator, always towards zero: a sum of D products in one go loses about
// a quarter of D / 16 x 2^-24 of itself (2e-6 at 2,048 terms; twice that and more where all terms have one sign). Logits
// are therefore summed in runs of at most 768 terms (two runs at least, from two stages on), a run an accumulator, and the runs
// added in float32 registers by the epilogue's threads, which hold their 128 columns: what is lost does not grow with D. Losses of
// 777 rows, 5,000 words, bf16, are off by 3.4e-7 of their norm at D = 2,048 (a float32 product's: 3.4e-7), 3.5e-7 at 8,192
// (7.5e-7); with one sign 3.5e-7 (3.2e-6) and 7.3e-7 (1.4e-5). Reading an accumulator takes about 2,000 clocks beside the
// products, which two accumulators hide where a run is long enough: 777 rows, 2,048 wide, 50,257 words take 149.6 us, in one go
// 147.9, in runs of 512 terms 156 (2.5e-7), of 256 terms 185 (1.2e-7). 750 rows of 768 terms (two runs of six stages), 32,003
// words, float16: the logits 38 us instead of 32.5, with their gradients stored 40 instead of 35. 128 sums a thread want more
// registers than twelve warps share evenly: the first four warps give some away.
constexpr bool sums_in_runs(int E) { return E == kLse || E == kDLogit; }
constexpr int kFewRegs = 80, kManyRegs = 208;
__host__ __device__ inline int run_stages(int stages) {  // of every run but the last
  int runs = (stages + kRun - 1) / kRun;
  if (runs < 2) runs = 2;
  return (stages + runs - 1) / runs;
}

// One product. a[s], b[s]: the operands of contraction segment s (kSwiglu: b[0] gate, b[1] up, one segment).
struct Op {
  CUtensorMap a[2], b[2], c;
  int tiles_m, tiles_n;
  int kb[2];            // stages of each segment
  int slices, per;      // (kStore) the contraction in `slices` parts of `per` stages, each a tile of its own
  bool a_mn, b_mn;
  bool m_live, k_live;  // only the first *Params::live rows of C, or of the contraction, count
  int M, N;
  // kStore: 0 = C in 16 bits; 1 = C into `sum`; 2 = added to `sum`; 3 = `sum` + C in 16 bits. The sums lie as the threads
  // hold them: [slice][tile][CTA][column][row].
  int sum_mode;
  float* sum;
  const float* factor;  // NULL: 1
  bool unscale;         // C is divided by what dg and du carry (Params::bounds)
};

struct Params {
  Op op[kMaxOps];
  int ops;
  const int* live;          // NULL: all
  CUtensorMap x[3];         // g and u as they are kept: the upper halves of their float32 bits, and the bytes below them
  CUtensorMap y[2];         // kDSwiglu: du (Op::c is dg), h
  bool keep;                // kSwiglu: store g, u; kDSwiglu: store h
  // float16's feed-forward block: the bits of max |g|, max |u| (kSwiglu collects them); max ||dy row||_1, max |w_down|
  uint32_t *bounds, *more;
  // kLse, kDLogit
  const int* labels;        // of the live rows (-1: none in the vocabulary)
  int v0;                   // the first column's place in the vocabulary
  float2* part;             // [2 tiles_n][M]: maximum, sum of the exponentials of what is below it
  float* target;            // [M]: the label's logit
  const float2* lse;        // [M]: the row's maximum, log2 of its sum
  const float* row_scale;   // [M]
  ErrorWord* err;
  int expire;               // (tests) the epilogue's wait that counts as given up
};

template <int E>
struct Cfg {
  static constexpr int kOut = E == kDSwiglu ? 6 * kStrip : E == kSwiglu ? 4 * kStrip : kSlab;  // a warp's
  static constexpr int kStages = E == kDSwiglu ? 4 : E == kSwiglu ? 5 : 6;
  static constexpr int kBarriers = 2 * kStages + 4 + 1 + 2 * kEpiWarps;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kEpiWarps * kOut + 8 * kBarriers + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// ---- host: a [rows, cols] matrix of 16-bit values, `ld` elements from row to row, as boxes of box_cols (64 or 32) x box_rows
inline bool matrix_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, long long rows, long long cols, long long ld,
                       int box_rows, int box_cols = 64) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld : (cols + 7) / 8 * 8) * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(m, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// an operand: K-major [m or n, k], or MN-major [k, m or n]
inline bool operand_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, long long rows, long long cols, long long ld,
                        bool mn) {
  return matrix_map(m, base, dt, rows, cols, ld, mn ? kBlockK : kHalf);
}
// what a warp stores or loads: 32 rows of 64 columns, or of 32 (kSwiglu, kDSwiglu)
inline bool strip_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, long long rows, long long cols, long long ld) {
  return matrix_map(m, base, dt, rows, cols, ld, 32, 32);
}
inline bool slab_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, long long rows, long long cols, long long ld) {
  return matrix_map(m, base, dt, rows, cols, ld, 32);
}
inline int blocks_of(long long n, int b) { return (int)((n + b - 1) / b); }

// ---- device: clusters, pairs of CTAs
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {  // the same place in the cluster's first CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(0));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Waits (the whole warp, one answer) for a phase that threads of the other CTA arrive at, too.
__device__ __forceinline__ bool cluster_wait(uint64_t* bar, uint32_t parity, ErrorWord* err, int where) {
  long long t0 = 0;
  bool ok = false;
  for (int turn = 0;; ++turn) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    ok = done != 0;
    if (ok) break;
    if (turn == 0) t0 = clock64();
    if (clock64() - t0 > kWaitCycles) {
      report(err, GD_ERR_TIMEOUT, where);
      break;
    }
  }
  return __all_sync(0xffffffffu, ok);
}
// (tests) Whether the wait `where`, though it ended well, counts as given up.
__device__ __forceinline__ bool expires(const Params& p, int where) {
  if (p.expire != where) return false;
  report(p.err, GD_ERR_TIMEOUT, where);
  return true;
}
// A box into this CTA's shared memory, counted on a barrier of the pair's first CTA.
__device__ __forceinline__ void load_pair(uint32_t lead, uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];\n\t}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(bar), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void load_slab(uint32_t dst, const CUtensorMap* m, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void store_slab(const CUtensorMap* m, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(m)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 x, {%1, %6};\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(lead), "r"(wattn::kDescHigh)
      : "memory");
}
// both CTAs' barriers at this place complete when the products so far have
__device__ __forceinline__ void commit_pair(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}\n" ::"r"(
          smem_u32(bar)),
      "r"(lead), "h"((uint16_t)3)
      : "memory");
}

// The rows that count are known on the device only: sizes that depend on them are computed where they are used.
__device__ __forceinline__ int row_tiles(const Op& o, int live) { return o.m_live ? (live + kTileM - 1) / kTileM : o.tiles_m; }
__device__ __forceinline__ int tiles_of(const Op& o, int live) { return row_tiles(o, live) * o.tiles_n * o.slices; }
template <int E>
__device__ __forceinline__ int all_tiles(const Params& p, int live) {
  int n = 0;
  for (int i = 0; i < (E == kStore ? p.ops : 1); ++i) n += tiles_of(p.op[i], live);
  return n;
}
// The tiles that a pair takes: the first problem's in turn; then, where some pairs have one tile of it more, the others make up for
// that with later problems' (shorter) tiles before all take turns again. (1,500 rows, half of them
// live, 768 wide, 32,003 words: dx's slices and dW 83 us instead of 96 at one clock)
struct Walk {
  int pair, pairs, tiles, first, mine, behind, extra;  // first: the first problem's tiles; behind: pairs with one less of them
  template <int E>
  __device__ __forceinline__ static Walk of(const Params& p, int live, int pair, int pairs);
  __device__ __forceinline__ int operator()(int i) const {  // the pair's i-th tile, or -1
    if (i < mine) return pair + i * pairs;
    i -= mine;
    const bool late = pair >= pairs - behind;
    if (late && i < extra) return first + pair - (pairs - behind) + i * behind;
    const int t = first + extra * behind + pair + (late ? i - extra : i) * pairs;
    return t < tiles ? t : -1;
  }
};
struct Where {
  int op, at, slice, m, n;  // the problem, the tile in it, its slice, the tile's first row and column
};
template <int E>
__device__ __forceinline__ Where locate(const Params& p, int tile, int live) {
  Where w;
  w.op = w.slice = 0;
  w.at = tile;
  if (E == kStore)
    for (; w.op + 1 < p.ops; ++w.op) {
      const int c = tiles_of(p.op[w.op], live);
      if (w.at < c) break;
      w.at -= c;
    }
  const Op& o = p.op[w.op];
  const int rows = row_tiles(o, live);
  int t = w.at;
  if (E == kStore && o.slices > 1) {
    w.slice = t / (rows * o.tiles_n);
    t -= w.slice * rows * o.tiles_n;
  }
  const int band = kGroupM * o.tiles_n, g = t / band, r = t - g * band;
  const int high = rows - g * kGroupM < kGroupM ? rows - g * kGroupM : kGroupM;
  w.m = (g * kGroupM + r % high) * kTileM;
  w.n = (r / high) * (E == kSwiglu ? kHalf : kTileN);
  return w;
}
// the tile's stages, of both segments one after the other, and the first of them
__device__ __forceinline__ int first_segment(const Op& o, int live) {
  return o.k_live ? (live + kBlockK - 1) / kBlockK : o.kb[0];
}
__device__ __forceinline__ int stages_of(const Op& o, const Where& w, int live, int& from) {
  const int n = first_segment(o, live) + o.kb[1];
  from = w.slice * o.per;
  return o.slices == 1 ? n : n - from < o.per ? (n > from ? n - from : 0) : o.per;
}

template <int E>
__device__ __forceinline__ Walk Walk::of(const Params& p, int live, int pair, int pairs) {
  Walk w;
  w.pair = pair, w.pairs = pairs, w.tiles = all_tiles<E>(p, live), w.first = tiles_of(p.op[0], live);
  w.mine = w.first > pair ? (w.first - pair + pairs - 1) / pairs : 0;
  w.behind = pairs - w.first % pairs, w.extra = 0;
  if (E == kStore && p.ops > 1 && w.behind < pairs) {
    auto length = [&](const Op& o) {  // (a tile's way out takes as long as kLeast stages)
      const int n = o.slices > 1 ? o.per : first_segment(o, live) + o.kb[1];
      return n < kLeast ? kLeast : n;
    };
    w.extra = length(p.op[0]) / length(p.op[1]);
    if (w.extra > (w.tiles - w.first) / w.behind) w.extra = (w.tiles - w.first) / w.behind;
  }
  return w;
}

__device__ __forceinline__ uint32_t slab_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t strip_at(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ void put_strip(uint32_t strip, int lane, const uint32_t (&u)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t v[4] = {u[4 * c], u[4 * c + 1], u[4 * c + 2], u[4 * c + 3]};
    st_shared16(strip + strip_at(lane, c), v);
  }
}
// 64 packed columns of the thread's row into its warp's slab
__device__ __forceinline__ void put_row(uint32_t slab, int lane, const uint32_t (&u)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t v[4] = {u[4 * c], u[4 * c + 1], u[4 * c + 2], u[4 * c + 3]};
    st_shared16(slab + slab_at(lane, c), v);
  }
}
__device__ __forceinline__ void ld_shared16(uint32_t a, uint32_t (&u)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
               : "r"(a)
               : "memory");
}
// The warp's slab of 32 x 64 values leaves for rows m0 .. of matrix m, columns n0 ..; what lies past the matrix is cut off.
// `u`: the thread's row. Waits until the slab's previous content is read.
__device__ __forceinline__ void send_row(const CUtensorMap* m, uint32_t slab, int lane, int n0, int m0, const uint32_t (&u)[32]) {
  if (lane == 0) bulk_wait_read0();
  __syncwarp();
  put_row(slab, lane, u);
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    store_slab(m, n0, m0, slab);
    bulk_commit();
  }
}

// g and u are kept as the upper 24 of their 32 bits, in three matrices of 16-bit words: the upper halves of g's, of u's, and the
// next byte of both (g's first). Rounded to 16 bits they would add two roundings to the weights' gradients, which have one of
// their own and one of dg or du: 1.8 times the error of a float32 form rounded at its end, with 24 bits 1.4 times.
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ uint32_t next_bytes(float g0, float u0, float g1, float u1) {
  return __byte_perm(__byte_perm(__float_as_uint(g0), __float_as_uint(u0), 0x0051),
                     __byte_perm(__float_as_uint(g1), __float_as_uint(u1), 0x0051), 0x5410);
}
// and back (the byte once more below itself: half of what the cut took away, and an infinity stays one)
__device__ __forceinline__ void kept_values(uint32_t g, uint32_t u, uint32_t low, float& g0, float& g1, float& u0, float& u1) {
  g0 = __uint_as_float(__byte_perm(g, low, 0x1044));
  g1 = __uint_as_float(__byte_perm(g, low, 0x3266));
  u0 = __uint_as_float(__byte_perm(u, low, 0x1055));
  u1 = __uint_as_float(__byte_perm(u, low, 0x3277));
}
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + ex2(-kLog2e * x)); }

// The power of two that dg and du carry in float16, the same for a whole call: |dh| <= ||dy row||_1 max |w_down|, |silu'| < 1.1
// and |silu(g)| <= |g| bound both by B, and 2^15 is the largest power of two in range. Without a bound above 0: 1.
__device__ __forceinline__ float carried(const uint32_t* b, const uint32_t* more) {
  if (b == nullptr) return 1.f;
  const float g = __uint_as_float(b[0]), u = __uint_as_float(b[1]);
  const float most = __uint_as_float(more[0]) * __uint_as_float(more[1]) * fmaxf(g, 1.1f * u);
  if (!(most > 0.f && most < INFINITY)) return 1.f;
  const int e = 14 - ilogbf(most);
  return ldexpf(1.f, e < -100 ? -100 : e > 100 ? 100 : e);
}

template <typename T, int E>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Params p) {
  using C = Cfg<E>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slabs = base + C::kStages * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(slabs + kEpiWarps * C::kOut);
  uint64_t* full = bars;                 // of the pair: the first CTA's are used
  uint64_t* empty = full + C::kStages;   // each CTA's own
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;    // of the pair: the first CTA's are used
  uint64_t* fin = acc_empty + 2;
  uint64_t* aux = fin + 1;               // each epilogue warp's own loads, two in turn
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + C::kBarriers);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int live = p.live == nullptr ? 0 : __ldg(p.live);
  const Walk walk = Walk::of<E>(p, live, pair, pairs);

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 2 * kEpiWarps);
    }
    mbar_init(fin, 1);
    for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(aux + i, 1);
    fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tm = __shfl_sync(0xffffffffu, *tslot, 0);
  const uint32_t s_base = smem_u32(base);
  if (warp < 4) {
    if constexpr (sums_in_runs(E)) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
    if (warp == 0) {
      // The whole warp runs this, one elected lane's instructions take effect: addresses and coordinates stay in uniform registers.
      // (Issued from a branch of one lane, a stage's loads took longer than its products where a launch holds several problems:
      // 1,215 instead of 1,540 TFLOP/s.)
      const uint32_t lead = elect();
      int slot = 0, laps = 0, issued = 0;
      bool ok = true;
      for (int i = 0, tile; ok && (tile = walk(i)) >= 0; ++i) {
        Where w = locate<E>(p, tile, live);
        w.op = __shfl_sync(0xffffffffu, w.op, 0);
        const Op& op = p.op[w.op];
        const int am = __shfl_sync(0xffffffffu, w.m + (int)rank * kHalf, 0);
        const int bn = __shfl_sync(0xffffffffu, E == kSwiglu ? w.n : w.n + (int)rank * kHalf, 0);
        auto segment = [&](auto a_mn, auto b_mn, const CUtensorMap* ma, const CUtensorMap* mb, int from, int n) {
          for (int kb = from; kb < from + n; ++kb) {
            if (laps > 0 && !(ok = warp_wait(empty + slot, (laps - 1) & 1, p.err, 80))) return;
            if (rank == 0 && lead) mbar_arrive_expect_tx(full + slot, 2 * kStage);
            const uint32_t bar = in_first_cta(full + slot), a = s_base + slot * kStage, b = a + kOperand;
            if (a_mn) {
              load_pair(lead, a, ma, am, kb * kBlockK, bar);
              load_pair(lead, a + kOperand / 2, ma, am + 64, kb * kBlockK, bar);
            } else {
              load_pair(lead, a, ma, kb * kBlockK, am, bar);
            }
            if (b_mn) {
              load_pair(lead, b, mb, bn, kb * kBlockK, bar);
              load_pair(lead, b + kOperand / 2, mb, bn + 64, kb * kBlockK, bar);
            } else {
              load_pair(lead, b, mb, kb * kBlockK, bn, bar);
            }
            ++issued;
            if (++slot == C::kStages) {
              slot = 0;
              ++laps;
            }
          }
        };
        using Yes = std::true_type;
        using No = std::false_type;
        for (int s = 0; ok && s < 2; ++s) {
          const CUtensorMap *ma = &op.a[s], *mb = E == kSwiglu ? &op.b[rank] : &op.b[s];
          // the tile's stages in this segment
          int first;
          const int all = stages_of(op, w, live, first), one = first_segment(op, live);
          const int here = s == 0 ? 0 : one, size = s == 0 ? one : op.kb[1];
          int from = first > here ? first - here : 0, n = (first + all - here < size ? first + all - here : size) - from;
          n = __shfl_sync(0xffffffffu, n, 0);
          from = __shfl_sync(0xffffffffu, from, 0);
          if constexpr (E == kStore) {
            const int layout = __shfl_sync(0xffffffffu, (op.a_mn ? 2 : 0) + (op.b_mn ? 1 : 0), 0);
            if (layout == 0) segment(No{}, No{}, ma, mb, from, n);
            else if (layout == 1) segment(No{}, Yes{}, ma, mb, from, n);
            else segment(Yes{}, Yes{}, ma, mb, from, n);
          } else {
            segment(No{}, std::integral_constant<bool, E == kDSwiglu>{}, ma, mb, from, n);
          }
        }
      }
      // The copies in flight land before the CTAs end, whatever became of their readers (they are counted on the first CTA's
      // barriers; the pair ends together).
      const int left = issued > C::kStages ? issued - C::kStages : 0;
      if (rank == 0)
        for (int i = left; i < issued; ++i) warp_wait(full + i % C::kStages, (i / C::kStages) & 1, p.err, 81);
      // So do the arrivals of the last products, which the first CTA's tensor core sends to both: a CTA that ended before them
      // would be written to when its shared memory is another's.
      for (int i = left; ok && i < issued; ++i) ok = warp_wait(empty + i % C::kStages, (i / C::kStages) & 1, p.err, 87);
    } else if (warp == 1) {
      if (rank == 0) {
        const uint32_t lead = elect();
        int slot = 0, laps = 0, turn = 0;  // turn: of the accumulators
        bool ok = true;
        for (int it = 0, tile; ok && (tile = walk(it)) >= 0; ++it) {
          const Where w = locate<E>(p, tile, live);
          const Op& op = p.op[w.op];
          int from;
          const int n = __shfl_sync(0xffffffffu, stages_of(op, w, live, from), 0);
          const int run = sums_in_runs(E) ? run_stages(n) : 0;
          // (the layouts are constants of each loop: descriptors and steps stay in uniform registers, which the instruction reads)
          auto products = [&](auto a_mn, auto b_mn) {
            constexpr uint32_t id = wattn::idesc<T>(256, 256, false) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
            constexpr uint32_t a_hi = a_mn ? (kOperand / 2 >> 4) << 16 : 1u << 16;
            constexpr uint32_t b_hi = b_mn ? (kOperand / 2 >> 4) << 16 : 1u << 16;
            constexpr uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;  // 16 k further, in 16 bytes
            uint32_t d = 0;
            auto begin = [&] {  // an accumulator whose last content is read
              const int buf = turn & 1;
              if (turn >= 2 && !(ok = cluster_wait(acc_empty + buf, ((turn >> 1) - 1) & 1, p.err, 82))) return;
              tc_fence_after();
              d = tm + buf * kTileN;
            };
            auto end = [&] { commit_pair(lead, acc_full + (turn++ & 1)); };
            begin();
            int at = 0;  // the stage in its run
            for (int kb = 0; ok && kb < n; ++kb) {
              if constexpr (sums_in_runs(E)) {
                if (at == run) {
                  end();
                  begin();
                  if (!ok) break;
                  at = 0;
                }
              }
              if (!(ok = cluster_wait(full + slot, laps & 1, p.err, 83))) break;
              tc_fence_after();
              const uint32_t a = ((s_base + slot * kStage) >> 4) | a_hi, b = ((s_base + slot * kStage + kOperand) >> 4) | b_hi;
  #pragma unroll
              for (int k = 0; k < kBlockK / 16; ++k) mma_pair(lead, d, a + k * a_step, b + k * b_step, id, at > 0 || k > 0);
              commit_pair(lead, empty + slot);
              ++at;
              if (++slot == C::kStages) {
                slot = 0;
                ++laps;
              }
            }
            if (ok) end();
          };
          using Yes = std::true_type;
          using No = std::false_type;
          if constexpr (E == kStore) {
            const int layout = __shfl_sync(0xffffffffu, (op.a_mn ? 2 : 0) + (op.b_mn ? 1 : 0), 0);
            if (layout == 0) products(No{}, No{});
            else if (layout == 1) products(No{}, Yes{});
            else products(Yes{}, Yes{});
          } else {
            products(No{}, std::integral_constant<bool, E == kDSwiglu>{});
          }
        }
        commit_pair(lead, fin);  // (a pair whose waits gave up ends with no product in flight)
      }
      warp_wait(fin, 0, p.err, 84);  // (both: it arrives in both, also where the pair has no tile and nothing else to wait for)
    }
  } else {
    if constexpr (sums_in_runs(E)) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
    const int ew = warp - 4, quad = warp & 3, half = ew >> 2;  // a warp reads the TMEM lanes of its quarter
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t slab = smem_u32(slabs) + ew * C::kOut;
    bool ok = true;
    int it = 0, turn = 0;  // (of the accumulators)
    // kDSwiglu: the kept g and u of 32 columns, a step of four to a tile, into one of two sets of strips, a step ahead of its use
    int step = 0;
    auto fetch = [&](int at, const Where& w) {  // step `at` is step at & 3 of w's tile
      const int n0 = w.n + half * 128 + (at & 3) * 32, m0 = w.m + (int)rank * kHalf + quad * 32;
      if (m0 >= p.op[0].M || n0 >= p.op[0].N) return;
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        const uint32_t to = slab + (at & 1) * 3 * kStrip;
        bulk_wait_read0();  // the step before the one that calls this stored from these strips
        mbar_arrive_expect_tx(aux + 2 * ew + (at & 1), 3 * kStrip);
#pragma unroll
        for (int i = 0; i < 3; ++i) load_slab(to + i * kStrip, &p.x[i], n0, m0, aux + 2 * ew + (at & 1));
      }
    };
    auto send_strips = [&](const Op& op, uint32_t strips, int n0, int m0) {  // dg, du and h
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        store_slab(&op.c, n0, m0, strips);
        store_slab(&p.y[0], n0, m0, strips + kStrip);
        if (p.keep) store_slab(&p.y[1], n0, m0, strips + 2 * kStrip);
        bulk_commit();
      }
    };
    if (E == kDSwiglu && walk(0) >= 0) fetch(0, locate<E>(p, walk(0), live));
    uint32_t landed = 0;  // kDSwiglu: the phase of each set's barrier (a step past the matrix loads nothing)
    int late = -1;        // kDSwiglu: the set whose wait gave up: what it waited for may still come, so the other set sends NaN
    for (int tile; (tile = walk(it)) >= 0; ++it) {
      const Where w = locate<E>(p, tile, live);
      const Op& op = p.op[w.op];
      const int m0 = w.m + (int)rank * kHalf + quad * 32, row = m0 + lane;
      const int rows = op.m_live ? live : op.M;  // (kDLogit: zeros in the rows past them)
      auto has = [&](int n0) { return m0 < (E == kDLogit ? op.M : rows) && n0 < op.N; };
      auto acquire = [&] {  // an accumulator is formed: its columns
        ok = ok && warp_wait(acc_full + (turn & 1), (turn >> 1) & 1, p.err, 85) && !expires(p, 85);
        tc_fence_after();
        return tm + lanes + (turn & 1) * kTileN;
      };
      auto release = [&] {  // it is read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(in_first_cta(acc_empty + (turn & 1)));
        ++turn;
      };
      uint32_t t0 = 0;
      float logit[2][sums_in_runs(E) ? 64 : 1];  // the row's 128 sums
      if constexpr (sums_in_runs(E)) {
#pragma unroll
        for (int i = 0; i < 64; ++i) logit[0][i] = logit[1][i] = 0.f;
        int from;
        const int n = stages_of(op, w, live, from), run = run_stages(n);
#pragma unroll 1
        for (int k = 0; k < n; k += run) {
          const uint32_t t = acquire() + half * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32(t + c * 32, v);
            if (c == 3) release();
#pragma unroll
            for (int i = 0; i < 32; ++i) logit[c >> 1][(c & 1) * 32 + i] += v[i];
          }
        }
      } else {
        t0 = acquire();
      }
      const float bad = ok ? 0.f : NAN;  // a wait that gave up leaves NaN

      if constexpr (E == kStore) {
        const float f = (op.factor != nullptr ? __ldg(op.factor) : op.unscale ? 1.f / carried(p.bounds, p.more) : 1.f) + bad;
        float* sum = op.sum_mode == 0 ? nullptr
                                      : op.sum + (((long long)w.at * 2 + rank) * kTileN + half * 128) * kHalf +
                                            quad * 32 + lane;
        int from;
        const bool none = stages_of(op, w, live, from) == 0;  // a sum over nothing
#pragma unroll 1
        for (int s = 0; s < 2; ++s) {
          const int c = half * 128 + s * 64, n0 = w.n + c;
          float v[64];
          wattn::tmem_ld64(t0 + c, v);
          if (s == 1) release();
          if (!has(n0)) continue;
          if (none) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = 0.f;
          }
          if (op.sum_mode != 0) {
            float* at = sum + (long long)s * 64 * kHalf;
            if (op.sum_mode != 1) {
#pragma unroll
              for (int i = 0; i < 64; ++i) v[i] += at[(long long)i * kHalf];
            }
            if (op.sum_mode != 3) {
#pragma unroll
              for (int i = 0; i < 64; ++i) at[(long long)i * kHalf] = v[i] + bad;
              continue;
            }
          }
          uint32_t u[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) u[i] = pack16<T>(v[2 * i] * f, v[2 * i + 1] * f);
          send_row(&op.c, slab, lane, n0, m0, u);
        }
      } else if constexpr (E == kSwiglu) {
        float top_g = 0.f, top_u = 0.f;
#pragma unroll 1
        for (int s = 0; s < 2; ++s) {
          const int c = half * 64 + s * 32, n0 = w.n + c;
          float g[32], u[32];
          tmem_ld32(t0 + c, g);
          tmem_ld32(t0 + kHalf + c, u);
          if (s == 1) release();
          if (!has(n0)) continue;
          if (!ok) {  // (NaN in what is kept, too)
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = u[i] = NAN;
          }
          uint32_t h[16], gh[16], uh[16], low[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            h[i / 2] = pack16<T>(g[i] * sigmoid(g[i]) * u[i], g[i + 1] * sigmoid(g[i + 1]) * u[i + 1]);
            gh[i / 2] = upper_halves(g[i], g[i + 1]);
            uh[i / 2] = upper_halves(u[i], u[i + 1]);
            low[i / 2] = next_bytes(g[i], u[i], g[i + 1], u[i + 1]);
            if constexpr (std::is_same<T, __half>::value) {  // (zeros past the matrix)
              top_g = wattn::max3(top_g, fabsf(g[i]), fabsf(g[i + 1]));
              top_u = wattn::max3(top_u, fabsf(u[i]), fabsf(u[i + 1]));
            }
          }
          if (lane == 0) bulk_wait_read0();
          __syncwarp();
          put_strip(slab, lane, h);
          if (p.keep) {
            put_strip(slab + kStrip, lane, gh);
            put_strip(slab + 2 * kStrip, lane, uh);
            put_strip(slab + 3 * kStrip, lane, low);
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            store_slab(&op.c, n0, m0, slab);
            if (p.keep) {
#pragma unroll
              for (int i = 0; i < 3; ++i) store_slab(&p.x[i], n0, m0, slab + (i + 1) * kStrip);
            }
            bulk_commit();
          }
        }
        if constexpr (std::is_same<T, __half>::value) {
          if (p.keep) {
            top_g = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_g)));
            top_u = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_u)));
            if (lane == 0) {
              atomicMax(p.bounds, __float_as_uint(top_g));
              atomicMax(p.bounds + 1, __float_as_uint(top_u));
            }
          }
        }
      } else if constexpr (E == kDSwiglu) {
        const float f = carried(p.bounds, p.more) + bad;
#pragma unroll 1
        for (int s = 0; s < 4; ++s, ++step) {
          const int c = half * 128 + s * 32, n0 = w.n + c, set = step & 1;
          float d[32];
          tmem_ld32(t0 + c, d);
          if (s == 3) release();
          const bool here = has(n0);
          if (here && late < 0) {
            if (warp_wait(aux + 2 * ew + set, (landed >> set) & 1, p.err, 86) && !expires(p, 86)) landed ^= 1u << set;
            else late = set;
          }
          if (late < 0) {
            if (s < 3) fetch(step + 1, w);
            else if (walk(it + 1) >= 0) fetch(step + 1, locate<E>(p, walk(it + 1), live));
          }
          if (!here) continue;
          if (late >= 0) {  // NaN from here on (0x7fff in both types), nothing more is loaded
            const uint32_t nan[4] = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
            const uint32_t strips = slab + (late ^ 1) * 3 * kStrip;
            if (lane == 0) bulk_wait_read0();
            __syncwarp();
#pragma unroll 1
            for (int i = 0; i < 12; ++i) st_shared16(strips + (i / 4) * kStrip + strip_at(lane, i & 3), nan);
            send_strips(op, strips, n0, m0);
            continue;
          }
          const uint32_t strips = slab + set * 3 * kStrip;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {  // a chunk of 8 columns of the thread's row, in place
            const uint32_t at = strips + strip_at(lane, i / 8);
            uint32_t g[4], u[4], h[4];
            ld_shared16(at, g);
            ld_shared16(at + kStrip, u);
            ld_shared16(at + 2 * kStrip, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float g0, g1, u0, u1;
              kept_values(g[j], u[j], h[j], g0, g1, u0, u1);
              const float s0 = sigmoid(g0), s1 = sigmoid(g1), a0 = g0 * s0, a1 = g1 * s1;
              const float d0 = d[i + 2 * j] * f, d1 = d[i + 2 * j + 1] * f;
              h[j] = pack16<T>(a0 * u0, a1 * u1);
              g[j] = pack16<T>(d0 * u0 * (s0 + a0 * (1.f - s0)), d1 * u1 * (s1 + a1 * (1.f - s1)));
              u[j] = pack16<T>(d0 * a0, d1 * a1);
            }
            st_shared16(at, g);
            st_shared16(at + kStrip, u);
            st_shared16(at + 2 * kStrip, h);
          }
          send_strips(op, strips, n0, m0);
        }
      } else if constexpr (E == kLse) {
        const int lab = row < rows ? __ldg(p.labels + row) : -1;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int n0 = w.n + half * 128 + s * 64;
          float(&v)[64] = logit[s];
          if (n0 >= op.N) continue;
          const bool here = lab >= n0 && lab < n0 + 64;
          if (__any_sync(0xffffffffu, here)) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) x = lab == n0 + i ? v[i] : x;
            if (here) p.target[row] = x + bad;
          }
          if (n0 + 64 > op.N) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = n0 + i < op.N ? v[i] : -INFINITY;
          }
          float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int i = 4; i < 60; i += 8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = wattn::max3(mx[e], v[i + 2 * e], v[i + 2 * e + 1]);
          }
          const float high = wattn::max3(wattn::max3(mx[0], mx[1], mx[2]), wattn::max3(mx[3], v[60], v[61]),
                                         wattn::max3(v[62], v[63], v[62]));
          const float next = wattn::max3(top, high, high), ref = next == -INFINITY ? 0.f : next;
          float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 64; ++i) a[i & 3] += ex2((v[i] - ref) * kLog2e);  // (1 at the maximum)
          sum = sum * ex2((top - ref) * kLog2e) + ((a[0] + a[1]) + (a[2] + a[3]));
          top = next;
        }
        if (row < rows && w.n + half * 128 < op.N)
          p.part[(long long)(w.n / kTileN * 2 + half) * op.M + row] = make_float2(top, sum + bad);
      } else {  // kDLogit
        const bool kept = row < rows;
        const int at = kept ? __ldg(p.labels + row) - p.v0 : -1;
        const float2 lse = kept ? __ldg(p.lse + row) : make_float2(0.f, 0.f);
        const float f = kept ? __ldg(p.row_scale + row) + bad : 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int n0 = w.n + half * 128 + s * 64;
          float(&v)[64] = logit[s];
          if (!has(n0)) continue;
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = ex2(fmaf(v[i] - lse.x, kLog2e, -lse.y));
          if (__any_sync(0xffffffffu, at >= n0 && at < n0 + 64)) {
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] -= at == n0 + i ? 1.f : 0.f;
          }
          uint32_t u[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const uint32_t x = pack16<T>(v[2 * i] * f, v[2 * i + 1] * f);
            u[i] = kept ? x : 0u;
          }
          send_row(&op.c, slab, lane, n0, m0, u);
        }
      }
    }
    if (late >= 0) warp_wait(aux + 2 * ew + late, (landed >> late) & 1, p.err, 86);  // its copies land before the CTA ends
    if (lane == 0) bulk_wait_read0();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
}

// The sums of slices, in their order, in 16 bits: row i of out [n, D] is row place[i] of C (NULL: i; -1: zeros). A thread has 8
// columns of a row, a warp 32 rows.
template <typename T>
__global__ void __launch_bounds__(256) sum_slices_kernel(const float* __restrict__ sum, int slices, int tiles_n, int n, int D,
                                                         const int* __restrict__ live, const int* __restrict__ place,
                                                         const float* __restrict__ factor, const uint32_t* bounds,
                                                         const uint32_t* more, T* __restrict__ out) {
  const int i = blockIdx.x * 32 + (threadIdx.x & 31), c = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 8;
  if (i >= n || c >= D) return;
  const int r = place == nullptr ? i : __ldg(place + i), rows = ((live == nullptr ? n : __ldg(live)) + kTileM - 1) / kTileM;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (r >= 0) {
    // the tile's index as the products' kernel counts them
    const int tm = r / kTileM, tn = c / kTileN, g = tm / kGroupM, high = min(rows - g * kGroupM, kGroupM);
    const int tile = g * kGroupM * tiles_n + tn * high + tm % kGroupM;
    const float f = factor != nullptr ? __ldg(factor) : 1.f / carried(bounds, more);
    for (int s = 0; s < slices; ++s) {
      const long long t = (long long)s * rows * tiles_n + tile;
      const float* at = sum + ((t * 2 + r % kTileM / kHalf) * kTileN + c % kTileN) * kHalf + r % kHalf;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += at[j * kHalf];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
  }
  store8<T>(out + (long long)i * D + c, v);
}
template <typename T>
int sum_slices(const float* sum, const Op& o, int n, int D, const int* live, const int* place, const uint32_t* bounds,
               const uint32_t* more, void* out, cudaStream_t stream) {
  const dim3 grid((unsigned)blocks_of(n, 32), (unsigned)blocks_of(D, 64));
  sum_slices_kernel<T><<<grid, 256, 0, stream>>>(sum, o.slices, o.tiles_n, n, D, live, place, o.factor, bounds, more,
                                                 static_cast<T*>(out));
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}
// How a contraction of `stages` for `tiles` tiles is cut, with 64 MiB of sums at most. {slices, stages of one} Where others
// of `rest` stages in all run beside it: a tile's length into about half of a pair's share of the whole, 16 stages or more. Alone:
// into what takes the fewest stages' times, the turns that 74 pairs take, each as long as a slice and its way out, and the joining.
// (256 rows, 4,096 x 12,288, the block's second product: four slices, 64 tiles in one turn; five would be 80 in two.)
struct Cut {
  int slices, per;
};
inline long long length_of(long long stages) { return stages < kLeast ? kLeast : stages; }  // as Walk counts them
inline Cut cut_of(long long tiles, long long stages, long long rest, int D) {
  Cut c = {1, (int)stages};
  if (blocks_of(D, 64) > 65535) return c;
  const long long room = (64ll << 20) / (tiles * kTileM * kTileN * 4);
  if (rest == 0) {
    long long least = (tiles + 73) / 74 * (stages + kLeast);
    for (int s = 2; s <= room && s <= stages / 12; ++s) {
      const int per = blocks_of(stages, s), slices = blocks_of(stages, per);
      const long long time = (tiles * slices + 73) / 74 * (per + kLeast) + 10 + tiles * slices / 8;
      if (time < least) least = time, c = {slices, per};
    }
    return c;
  }
  long long share = (tiles * stages + rest) / 74 / 2;
  if (share < 16) share = 16;
  if (stages <= share + share / 2) return c;
  c.slices = blocks_of(stages, (int)share);
  if (c.slices > room) c.slices = room < 1 ? 1 : (int)room;
  c.per = blocks_of(stages, c.slices);
  c.slices = blocks_of(stages, c.per);
  return c;
}
inline size_t cut_bytes(const Cut& c, long long tiles) {
  return c.slices > 1 ? (size_t)c.slices * tiles * kTileM * kTileN * 4 : 0;
}

// Whether C's tiles can be counted (they are ints, several problems' together).
inline bool countable(long long M, long long N) { return (M + 127) / 128 * ((N + 127) / 128) < (1ll << 28); }

// Persistent pairs: as many as SMs allow. They take the tiles in turn, the problems' with the longest contractions first (4,093
// rows, 1,000 x 2,728, float16, the block's four gradients and its second product: 111 us, with the longest last 120).
template <typename T, int E>
int launch(Params& p, cudaStream_t stream) {
  auto length = [](const Op& o) { return o.slices > 1 ? o.per : o.kb[0] + o.kb[1]; };
  for (int i = 1; i < p.ops; ++i)
    for (int j = i; j > 0 && length(p.op[j]) > length(p.op[j - 1]); --j) std::swap(p.op[j], p.op[j - 1]);
  int tiles = 0;
  for (int i = 0; i < p.ops; ++i) {
    if (p.op[i].slices < 1) p.op[i].slices = 1;
    tiles += p.op[i].tiles_m * p.op[i].tiles_n * p.op[i].slices;
  }
  if (tiles == 0) return GD_OK;
  static bool done[kMaxDevices];
  auto kern = gemm_kernel<T, E>;
  if (set_smem_once(kern, Cfg<E>::kSmem, done) != cudaSuccess) return (cudaGetLastError(), GD_ERR_LAUNCH);
  if constexpr (sums_in_runs(E)) {  // the launch has the warps' shares (else the epilogue would wait for registers for good)
    static bool fits = false;
    cudaFuncAttributes at;
    if (!fits && (cudaFuncGetAttributes(&at, kern) != cudaSuccess ||
                  !(fits = at.numRegs * kThreads >= 128 * kFewRegs + 32 * kEpiWarps * kManyRegs)))
      return (cudaGetLastError(), GD_ERR_LAUNCH);
  }
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return (cudaGetLastError(), GD_ERR_LAUNCH);
  const int pairs = tiles < sms / 2 ? tiles : sms / 2;
  kern<<<2 * pairs, kThreads, Cfg<E>::kSmem, stream>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? GD_OK : (cudaGetLastError(), GD_ERR_LAUNCH);
}

}  // namespace gemm
}  // namespace gd
