// The gated feed-forward block's sizes and parts (host).
#pragma once

#include <cuda_runtime.h>

namespace gd {
namespace ff {

struct Problem {
  const void *x, *wg, *wu, *wd;
  long long ldx, ldg, ldu, ldd;  // elements from row to row
  int rows, D, F, O;
};

// Elements from row to row of h, dg, du and what is kept of g and u: whole 128-byte lines. (4,093 rows of 2,728 columns, 1,000
// wide, float16: the products of a training pass take 223 us; with rows of 5,456 bytes they took 322 us)
inline long long pitch(int F) { return (F + 63) / 64 * 64; }

// y for at most kFew rows, h [rows, F] on the way (gd_ff_few.cu)
constexpr int kFew = 128;
int forward_few(const Problem& q, int dtype, void* h, void* y, cudaStream_t stream);

}  // namespace ff
}  // namespace gd
