// Reads of a GEMM result left as K-split partial sums (PartSum), shared by its consumers.
#pragma once

#include "prefill.h"

namespace chonk {
namespace {

// part_gather in two halves, so that the first round's loads can be issued
// early and summed where the values are needed: part_issue loads splits 0..3
// (clamped to the last split) of elements j[e]; part_finish adds them in split
// order and reads any further splits four at a time.
template <int N>
__device__ __forceinline__ void part_issue(const PartSum& P, int t, const int (&j)[N], float (&w)[N][4]) {
  const float* q = P.p + (int64_t)t * P.ld;
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int z = 0; z < 4; ++z) w[e][z] = q[(int64_t)min(z, P.ks - 1) * P.zs + j[e]];
}
template <int N>
__device__ __forceinline__ void part_finish(const PartSum& P, int t, const int (&j)[N], float (&w)[N][4],
                                            float (&v)[N]) {
  const float* q = P.p + (int64_t)t * P.ld;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    v[e] = w[e][0];
#pragma unroll
    for (int z = 1; z < 4; ++z) v[e] = z < P.ks ? v[e] + w[e][z] : v[e];
  }
  for (int z0 = 4; z0 < P.ks; z0 += 4) {
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int z = 0; z < 4; ++z) w[e][z] = q[(int64_t)min(z0 + z, P.ks - 1) * P.zs + j[e]];
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int z = 0; z < 4; ++z) v[e] = z0 + z < P.ks ? v[e] + w[e][z] : v[e];
  }
}

// Elements j[e] (valid columns) of row t of a deferred result: the partials
// are read four splits at a time, every load of a round issued before any is
// added (split indices past ks are clamped to the last split and their sums
// not taken, so no load sits behind a branch: a conditional load makes the
// compiler wait for every outstanding load where the paths join); the sums
// add the partials in split order. With ks <= 4 a call costs one memory round
// trip for all N elements.
template <int N>
__device__ __forceinline__ void part_gather(const PartSum& P, int t, const int (&j)[N], float (&v)[N]) {
  if (P.ks == 1) {
    const float* q = P.p + (int64_t)t * P.ld;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = q[j[e]];
    return;
  }
  float w[N][4];
  part_issue<N>(P, t, j, w);
  part_finish<N>(P, t, j, w, v);
}

}  // namespace
}  // namespace chonk
