// Shared parts of the softmax-attention kernels (causal, sliding window, first tokens that stay visible): the tile ranges,
// packed rows, the swizzled tiles that TMA writes and tcgen05 reads, TMEM operands.
//
// A tile is 128 rows (tokens of one head) by NS slabs of 64 channels; a slab is 128 rows of 128 bytes in the 128-byte
// swizzle (TMA box 64 x 1 x 128 x 1), 16 KB. The same bytes are a K-major operand (rows = M or N, channels = K) and an
// MN-major one (rows = K, channels = M or N): only the descriptor differs. Channels past D and tokens past T read as
// zeros (TMA's fill), so head widths up to NS * 64 and ragged lengths need no copies.
#pragma once

#include "gd_common.cuh"

namespace gd {
namespace wattn {

constexpr int kTile = 128;
constexpr int kSlabBytes = kTile * 128;
constexpr int kNoWindow = 0x3fffffff;
constexpr float kLog2e = 1.4426950408889634f;

struct Problem {
  int B, Tq, Tk, H, HK;    // packed rows: B = 1, Tq = Tk = all rows
  int D;
  int window, sinks;       // key j is visible to position p: j <= p and (j > p - window or j < sinks)
  // scale, and scale * log2(e). The forward, whose mask and maximum come before its scale, takes a positive scale_log2 and
  // the scale's sign apart (Q takes it).
  float scale, scale_log2;
  bool negate;
  const int* cu;           // packed rows' boundaries [N + 1], or NULL
  int N;
};

// One row of the batch or one packed sequence: the rows it covers, and its queries' first position.
struct Seq {
  int b, q0, Tq, k0, Tk;
  __device__ __forceinline__ int offset() const { return Tk - Tq; }  // query i stands at position i + offset
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// The packed sequence that owns work item `item`, when a run of n rows has count(n) items; returns its index within the
// sequence, or -1 past the last. After the sequences' items come those of the rows before the first and behind the last, which
// belong to none: `gap` is set (their results are zeros). One whole warp. Boundaries are clamped into [0, rows], and one below
// an earlier one counts as that one: whatever cu holds, every row has exactly one owner.
template <typename Count>
__device__ __forceinline__ int find_item(const int* cu, int N, int rows, int item, Count count, Seq& s, bool& gap) {
  constexpr int kPer = 8;
  const int lane = threadIdx.x & 31;
  int before = 0, top = 0;  // items and the highest boundary so far
  gap = false;
  for (int base = 0; base < N; base += 32 * kPer) {
    int first[kPer], len[kPer], high = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int n = base + lane * kPer + i;
      first[i] = high = max(high, n < N ? clampi(__ldg(cu + n), 0, rows) : 0);  // the lane's highest so far
    }
    int upto = high;  // of the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto = max(upto, y);
    }
    int below = __shfl_up_sync(0xffffffffu, upto, 1);
    below = lane > 0 ? max(below, top) : top;
    int end = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int n = base + lane * kPer + i;
      first[i] = max(first[i], below);
      len[i] = n < N ? max(clampi(__ldg(cu + n + 1), 0, rows) - first[i], 0) : 0;
      end = max(end, first[i] + len[i]);
      sum += count(len[i]);
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (item < before + total) {
      int at = before + incl - sum, found = -1, f0 = 0, fl = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int c = count(len[i]);
        if (found < 0 && item >= at && item < at + c) {
          found = item - at;
          f0 = first[i];
          fl = len[i];
        }
        at += c;
      }
      const unsigned who = __ballot_sync(0xffffffffu, found >= 0);
      const int src = __ffs(who) - 1;
      s.b = 0;
      s.q0 = s.k0 = __shfl_sync(0xffffffffu, f0, src);
      s.Tq = s.Tk = __shfl_sync(0xffffffffu, fl, src);
      return __shfl_sync(0xffffffffu, found, src);
    }
    before += total;
    top = __reduce_max_sync(0xffffffffu, end);
  }
  gap = true;
  const int head = clampi(__ldg(cu), 0, rows);
  int i = item - before;
  s.b = 0;
  s.q0 = s.k0 = 0;
  s.Tq = s.Tk = head;
  if (i < count(head)) return i;
  i -= count(head);
  s.q0 = s.k0 = top;
  s.Tq = s.Tk = rows - top;
  return i < count(rows - top) ? i : -1;
}
// The items of N packed sequences of `rows` rows in all, in tiles of kTile, with the two runs of rows that belong to none
inline long long packed_items(int rows, int N) { return (long long)rows / kTile + N + 2; }

// The key tiles that queries [i0, i1] (positions p0 .. p1) of a sequence see: the first `head` tiles, then tiles
// lo .. lo + n - head - 1.
struct KeyRange {
  int n, head, lo;
  __device__ __forceinline__ KeyRange(int p0, int p1, int window, int sinks) {
    n = head = lo = 0;
    if (p1 < 0) return;  // no position reached: no key visible
    const int hi = p1 / kTile;
    const int from = p0 - window + 1;
    lo = from > 0 ? from / kTile : 0;
    head = (sinks + kTile - 1) / kTile;
    if (head > lo) head = lo;
    n = head + hi - lo + 1;
  }
  __device__ __forceinline__ int key(int j) const { return (j < head ? j : lo + j - head) * kTile; }  // tile j's first key
};

// mbar_wait by a whole warp, with one answer for all its lanes (the aligned tcgen05 instructions that follow need that).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, ErrorWord* err, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, where));
}

// Does every query at positions p0 .. p1 see all keys c .. c + 127?
__device__ __forceinline__ bool all_visible(int c, int p0, int p1, int window, int sinks) {
  return c + kTile - 1 <= p0 && (c > p1 - window || c + kTile <= sinks);
}

// ---- host: [B, T, heads, D] rows read through strides (in elements) as boxes of 64 channels x `box_t` tokens of a head
inline bool tile_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int B, int T, int heads, int D,
                     long long sb, long long st, long long sh, int box_t) {
  EncodeTiled enc = encode_tiled();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T, (cuuint64_t)B};
  // a dimension of one entry has no stride of its own: any multiple of 16 bytes
  const cuuint64_t strides[3] = {(cuuint64_t)(heads > 1 ? sh : D) * 2, (cuuint64_t)(T > 1 ? st : D) * 2,
                                 (cuuint64_t)(B > 1 ? sb : D) * 2};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)box_t, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(m, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// a contiguous output [B, T, heads, D], stored 32 rows at a time
inline bool out_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int B, int T, int heads, int D) {
  return tile_map(m, base, dt, B, T, heads, D, (long long)T * heads * D, (long long)heads * D, D, 32);
}

// all NS slabs of the tile at token t of head h, row b
template <int NS>
__device__ __forceinline__ void load_tile(uint32_t smem, const CUtensorMap* m, int h, int t, int b, uint64_t* bar) {
#pragma unroll
  for (int s = 0; s < NS; ++s)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem + s * kSlabBytes),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(64 * s), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
        : "memory");
}

// half x (128 channels, two slabs) of a 256-channel tile
__device__ __forceinline__ void load_half(uint32_t smem, const CUtensorMap* m, int x, int h, int t, int b, uint64_t* bar) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem + s * kSlabBytes),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(64 * (2 * x + s)), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
        : "memory");
}

// ---- tcgen05 products. The whole warp that issues them runs the same code, one elected lane's instructions take effect
// (`lead`): warp-uniform addresses and descriptors stay in uniform registers, which the instruction reads. (Issued from a
// branch of one lane, every product first moved its operands there: 80 to 100 clocks an instruction of 64.)
__device__ __forceinline__ uint32_t elect() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, e;\n\t}\n"
      : "=r"(lead));
  return lead;
}
// Shared-memory descriptors in the 128-byte swizzle (layout type 2): the high word is the same for all, 8-row groups 1024
// bytes apart. Low word, K-major: 16 channels further = 32 bytes; MN-major: 64-channel groups one slab apart, 16 rows
// further = 2048 bytes.
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return (addr >> 4) | ((uint32_t)(kSlabBytes >> 4) << 16); }
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool b_mn) {
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 x, {%1, %6};\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(lead), "r"(kDescHigh)
      : "memory");
}
// A in TMEM (128 lanes, 16-bit pairs in 32-bit columns)
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(id), "r"(acc), "r"(lead), "r"(kDescHigh)
      : "memory");
}
// `bar` completes when the lead lane's products so far have
__device__ __forceinline__ void mma_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// D[128 x N] = X Y^T: X 128 rows, Y N rows, of NS slabs, contracted over their channels
template <typename T, int NS, int N = 128>
__device__ __forceinline__ void mma_xyt(uint32_t lead, uint32_t d, uint32_t x, uint32_t y, bool acc = false) {
  const uint32_t a = desc_k(x), b = desc_k(y);
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      mma_ss(lead, d, a + s * (kSlabBytes >> 4) + 2 * k, b + s * (kSlabBytes >> 4) + 2 * k, idesc<T>(128, N, false),
             acc || s > 0 || k > 0);
}
// D[128 x NS 64] (+)= P Y: P in TMEM (128 rows, 16 K contracted columns as 8 K words), Y's rows contracted. P stands in
// pieces of 32 contracted columns (16 words), `gap` words apart.
template <typename T, int NS, int K = 8>
__device__ __forceinline__ void mma_py(uint32_t lead, uint32_t d, uint32_t p, uint32_t y, bool acc, int gap) {
  const uint32_t b = desc_mn(y);
#pragma unroll
  for (int k = 0; k < K; ++k)
    mma_ts(lead, d, p + (k & 1) * 8 + (k >> 1) * gap, b + 128 * k, idesc<T>(128, NS * 64, true), acc || k > 0);
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two fp32 values at once (the packed instructions take an issue slot for two operations)
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unf2(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// bits [from, end) of 32 (any ints)
__device__ __forceinline__ uint32_t bits(int from, int end) {
  const uint32_t lo = from <= 0 ? 0xffffffffu : from >= 32 ? 0u : 0xffffffffu << from;
  const uint32_t hi = end >= 32 ? 0xffffffffu : end <= 0 ? 0u : 0xffffffffu >> (32 - end);
  return lo & hi;
}
// the visible ones of keys c .. c + 31 to position p: key <= p, and key > p - window or key < sinks
__device__ __forceinline__ uint32_t visible_keys(int c, int p, int window, int sinks) {
  return (bits(p - window + 1 - c, p + 1 - c) | bits(0, sinks - c)) & bits(0, p + 1 - c);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ex2_pair(F2 x, float& a, float& b) {
  unf2(x, a, b);
  a = ex2(a);
  b = ex2(b);
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// 64 consecutive fp32 columns of the thread's own lane, one wait.
__device__ __forceinline__ void tmem_ld64(uint32_t a, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(a), "r"(a + 32)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

// registers -> 16 consecutive words of the thread's own lane (asynchronous: tmem_st_wait).
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 32 of them.
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&u));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}

// byte of 16-byte chunk c (8 channels) of a row in a swizzled tile
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  return (c >> 3) * kSlabBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void st_shared16(uint32_t a, const uint32_t (&u)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
}
// A tile that has landed, NS slabs: rows from .. to - 1 set to 0, thread `id` of `n`. For rows past the end of a packed
// sequence: they are the next one's, whose infinities and NaN would meet weights of 0 in the product that sums over them.
// That product is issued after a barrier that every one of these threads arrives at.
template <int NS>
__device__ __forceinline__ void zero_rows(uint32_t smem, int from, int to, int id, int n) {
  const uint32_t zero[4] = {0, 0, 0, 0};
#pragma unroll 1
  for (int s = 0; s < NS; ++s)
#pragma unroll 1
    for (int a = from * 128 + id * 16; a < to * 128; a += n * 16) st_shared16(smem + s * kSlabBytes + a, zero);
  fence_async_smem();
}
// the same by the warp that issues the product
template <int NS>
__device__ __forceinline__ void zero_rows(uint32_t smem, int from) {
  if (from >= kTile) return;
  zero_rows<NS>(smem, from, kTile, threadIdx.x & 31, 32);
  __syncwarp();
}
// A tile of 16-bit values that has landed, NS slabs, times -1; by the warp that issues the products that read it.
template <int NS>
__device__ __forceinline__ void negate_tile(uint32_t smem) {
#pragma unroll 1
  for (int a = (threadIdx.x & 31) * 16; a < NS * kSlabBytes; a += 32 * 16) {
    uint32_t u[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                 : "r"(smem + a)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] ^= 0x80008000u;
    st_shared16(smem + a, u);
  }
  fence_async_smem();
  __syncwarp();
}
// Rows row0 .. row0 + 31 of a swizzled tile in shared memory -> tokens t0 + row of head h, row b of a [B, T, heads, D] array,
// rows below `live` only, NS slabs from channel ch on; one whole warp, whose own rows these are (or after a barrier). By
// TMA (one lane issues it and waits until shared memory is read; the array's end cuts it off) unless rows past `live` belong
// to someone else.
template <typename T, int NS>
__device__ __forceinline__ void store_rows(const CUtensorMap* m, T* out, uint32_t smem, int row0, int b, int t0, int live,
                                           int T_, int h, int heads, int D, int ch = 0) {
  if (row0 >= live) return;
  if (live - row0 >= 32 || t0 + live == T_) {
    fence_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int s = 0; s < NS; ++s)
        if (ch + s * 64 < D)
          asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                           reinterpret_cast<uint64_t>(m)),
                       "r"(ch + 64 * s), "r"(h), "r"(t0 + row0), "r"(b), "r"(smem + s * kSlabBytes + row0 * 128)
                       : "memory");
      bulk_commit();
      bulk_wait_read0();
    }
    return;
  }
  __syncwarp();
  const int chunks = (D - ch < NS * 64 ? D - ch : NS * 64) >> 3, lane = threadIdx.x & 31, n = (live - row0) * chunks;
  out += (((long long)b * T_ + t0 + row0) * heads + h) * D + ch;
  for (int i = lane; i < n; i += 32) {
    const int r = i / chunks, c = i - r * chunks;
    uint4 u;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "r"(smem + tile_at(row0 + r, c))
                 : "memory");
    *reinterpret_cast<uint4*>(out + (long long)r * heads * D + c * 8) = u;
  }
}

// The entry points' parts (host): strides of q, k, v in elements, (batch, token, head) each; low: what o's rounding took
// away (may be NULL in the forward)
int forward(const void* q, const void* k, const void* v, const long long* strides, const Problem& pr, int dtype, void* o,
            void* low, float* lse, ErrorWord* err, cudaStream_t stream);
// (and of dO: strides[9 .. 11]); the first `heavy` key tiles are cut into `parts` CTAs with fp32 partial tiles at `part`
int backward(const void* q, const void* k, const void* v, const void* o, const void* low, const void* g,
             const long long* strides, const Problem& pr, int dtype, const float* lse, float* delta, void* dq, void* dk, void* dv, int heavy,
             int parts, float* part, ErrorWord* err, cudaStream_t stream);

}  // namespace wattn
}  // namespace gd
