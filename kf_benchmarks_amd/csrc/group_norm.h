// Shared by group_norm.hip (images) and group_norm_rows.hip (one row an image).
#pragma once
#include "act.h"
#include "raw.h"

namespace kfb {
namespace gn {

struct Args {
  const void* x;
  const void* dy;
  void* y;  // forward: y, backward: dx
  const float *gamma, *beta;
  float *mean, *rstd;  // [N][G]
  float* part;         // backward: [slabs][2][C], sum e xh | sum e
  long N, HW;
  int C, G, cpg;
  float eps;
  Act act;
};

// e = dy act'(u) and xh of a thread's V channels, whose groups' mean and 1 / std
// are mu and rs (VG = 1: one group, else one for each channel)
template <typename T, int V, int VG, int KIND>
__device__ __forceinline__ void grad_terms(const Args& a, const Raw<T, V>& x, const Raw<T, V>& dy,
                                           const float (&mu)[VG], const float (&rs)[VG],
                                           const float (&ga)[V], const float (&be)[V],
                                           float (&e)[V], float (&xh)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    xh[i] = (x[i] - mu[i % VG]) * rs[i % VG];
    e[i] = dy[i] * act_grad<KIND>(fmaf(xh[i], ga[i], be[i]), a.act);
  }
}

template <int V>
__device__ __forceinline__ void load_params(const float* p, int c, bool on, float other,
                                            float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = on && p ? p[c + i] : other;
}

// Rows (group_norm_rows.hip): whether they take a shape, the slabs of channel
// sums of their backward, and the launches.
bool rows_take(int dtype, long N, long HW, int C, int G, int V);
long rows_slabs(int dtype, long N, int C, int G, int V);
hipError_t rows_fwd(int dtype, const Args& a, int V, hipStream_t s);
hipError_t rows_bwd(int dtype, const Args& a, int V, hipStream_t s);

}  // namespace gn
}  // namespace kfb
