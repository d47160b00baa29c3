// Group norm of single rows (one token an image): a group is cpg neighbouring
// values, held by L = 2^i <= 64 lanes, K vectors each, so a wave holds 64 / L
// groups and every sum is a few lane exchanges: no LDS and no barriers.  The
// formulas are group_norm.hip's.
//
// Bound by HBM.  A set of L lanes keeps one group index g (gamma, beta and, in the
// backward, the channel sums stay in registers) and walks over the rows, the next
// row loaded while one is worked on.  8192 waves, one row at a time: 22.2 us for
// 13984 rows of 1600 bf16 values in 8 groups (4.0 TB/s; a copy reaches 5.2);
// 4096 waves took 25.3 us, two rows at a time 25.1, 16384 waves (each reads gamma
// and beta, as many bytes as its rows) 33.6.  With SiLU 28 us forward and 53 us backward
// (134 MB of x, dy and dx: 2.6 TB/s), and 7 us for the channel sums.
#include "group_norm.h"

namespace kfb {
namespace gn {

constexpr int RNT = 256, RK = 8;

struct Rows {
  int L, nv;   // lanes of a group, its vectors
  int sets;    // lane sets of the launch: slabs * G
  int slabs;   // rows n, n + slabs, ... belong to slab n
};

// sum over the L lanes of a set (L uniform: scalar branches)
__device__ __forceinline__ float set_sum(float v, int L) {
  if (L > 1) v += __shfl_xor(v, 1, 64);
  if (L > 2) v += __shfl_xor(v, 2, 64);
  if (L > 4) v += __shfl_xor(v, 4, 64);
  if (L > 8) v += __shfl_xor(v, 8, 64);
  if (L > 16) v += __shfl_xor(v, 16, 64);
  if (L > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

template <typename T, int V, int KIND, int K>
__global__ void __launch_bounds__(RNT) gn_rows_fwd_k(Args a, Rows w) {
  const int set = (int)((blockIdx.x * RNT + threadIdx.x) / w.L), j = threadIdx.x % w.L;
  if (set >= w.sets) return;
  const int g = set % a.G, c0 = g * a.cpg;
  float ga[K][V], be[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int jv = j + k * w.L;
    load_params<V>(a.gamma, c0 + jv * V, jv < w.nv, 1.f, ga[k]);
    load_params<V>(a.beta, c0 + jv * V, jv < w.nv, 0.f, be[k]);
  }
  const float inv = 1.f / (float)a.cpg;
  const T* __restrict__ x = (const T*)a.x + c0 + j * V;
  T* __restrict__ y = (T*)a.y + c0 + j * V;
  Raw<T, V> next[K];
  auto fetch = [&](long n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      next[k].zero();
      if (j + k * w.L < w.nv) next[k].load(x + n * a.C + (long)k * w.L * V);
    }
  };
  long n = set / a.G;
  if (n < a.N) fetch(n);
  for (; n < a.N; n += w.slabs) {
    Raw<T, V> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k] = next[k];
    if (n + w.slabs < a.N) fetch(n + w.slabs);  // while this row is worked on
    float s = 0.f, m2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s += raw[k][i];
    const float mu = set_sum(s, w.L) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + k * w.L < w.nv)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = raw[k][i] - mu;
          m2 = fmaf(d, d, m2);
        }
    const float rs = 1.f / sqrtf(set_sum(m2, w.L) * inv + a.eps);
    if (j == 0) {
      a.mean[n * a.G + g] = mu;
      a.rstd[n * a.G + g] = rs;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + k * w.L < w.nv) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
          o[i] = act_fwd<KIND>(fmaf((raw[k][i] - mu) * rs, ga[k][i], be[k][i]), a.act);
        store_vec<T, V>(y + n * a.C + (long)k * w.L * V, o);
      }
  }
}

template <typename T, int V, int KIND, int K>
__global__ void __launch_bounds__(RNT) gn_rows_bwd_k(Args a, Rows w) {
  const int set = (int)((blockIdx.x * RNT + threadIdx.x) / w.L), j = threadIdx.x % w.L;
  if (set >= w.sets) return;
  const int g = set % a.G, c0 = g * a.cpg, slab = set / a.G;
  float ga[K][V], be[K][V], cp[K][V], cq[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int jv = j + k * w.L;
    load_params<V>(a.gamma, c0 + jv * V, jv < w.nv, 1.f, ga[k]);
    load_params<V>(a.beta, c0 + jv * V, jv < w.nv, 0.f, be[k]);
#pragma unroll
    for (int i = 0; i < V; ++i) cp[k][i] = cq[k][i] = 0.f;
  }
  const float inv = 1.f / (float)a.cpg;
  const T* __restrict__ x = (const T*)a.x + c0 + j * V;
  const T* __restrict__ dy = (const T*)a.dy + c0 + j * V;
  T* __restrict__ dx = (T*)a.y + c0 + j * V;
  Raw<T, V> nx[K], nd[K];
  float nmu = 0.f, nrs = 0.f;
  auto fetch = [&](long n) {
    nmu = a.mean[n * a.G + g];
    nrs = a.rstd[n * a.G + g];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + k * w.L < w.nv) {
        nx[k].load(x + n * a.C + (long)k * w.L * V);
        nd[k].load(dy + n * a.C + (long)k * w.L * V);
      }
  };
  if (slab < a.N) fetch(slab);
  for (long n = slab; n < a.N; n += w.slabs) {
    Raw<T, V> rx[K], rd[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rx[k] = nx[k];
      rd[k] = nd[k];
    }
    const float mu[1] = {nmu}, rs[1] = {nrs};
    if (n + w.slabs < a.N) fetch(n + w.slabs);  // while this row is worked on
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + k * w.L < w.nv) {
        float e[V], xh[V];
        grad_terms<T, V, 1, KIND>(a, rx[k], rd[k], mu, rs, ga[k], be[k], e, xh);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          cp[k][i] += e[i];
          cq[k][i] = fmaf(e[i], xh[i], cq[k][i]);
          s1 = fmaf(ga[k][i], e[i], s1);
          s2 = fmaf(ga[k][i] * e[i], xh[i], s2);
        }
      }
    s1 = set_sum(s1, w.L) * inv;
    s2 = set_sum(s2, w.L) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (j + k * w.L < w.nv) {
        float e[V], xh[V];
        grad_terms<T, V, 1, KIND>(a, rx[k], rd[k], mu, rs, ga[k], be[k], e, xh);
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = rs[0] * (fmaf(ga[k][i], e[i], -s1) - xh[i] * s2);
        store_vec<T, V>(dx + n * a.C + (long)k * w.L * V, e);
      }
  }
  float* out = a.part + (long)slab * 2 * a.C + c0 + j * V;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (j + k * w.L < w.nv)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        out[k * w.L * V + i] = cq[k][i];
        out[a.C + k * w.L * V + i] = cp[k][i];
      }
}

// Lane sets that fill the card and no more than the rows need.  Backward: each
// slab of rows leaves 2 C sums to add up, so it has half the waves.
static Rows rows_of(long N, int C, int G, int V, bool bwd, int& K) {
  Rows w;
  w.nv = C / G / V;
  w.L = 1;
  while (w.L < 64 && w.L < w.nv) w.L *= 2;
  K = ceil_div(w.nv, w.L);
  const long waves = bwd ? 4096 : 8192;
  long slabs = ceil_div(waves * 64 / w.L, G);
  const long most = bwd ? ceil_div(N, 4) : N;
  if (slabs > most) slabs = most;
  if (bwd && slabs > 1024) slabs = 1024;
  w.slabs = (int)slabs;
  w.sets = w.slabs * G;
  return w;
}

bool rows_take(int dtype, long N, long HW, int C, int G, int V) {
  const int full = dtype == F32 ? 4 : 8, cpg = C / G;
  return HW == 1 && cpg % V == 0 && (V == full || V == 1) && cpg / V <= 64 * RK && G <= (1 << 20);
}

long rows_slabs(int dtype, long N, int C, int G, int V) {
  int K;
  return rows_of(N, C, G, V, true, K).slabs;
}

#define KFB_ROWS(T, v, k, V, K, ...)                                                     \
  if (v > 1) {                                                                           \
    constexpr int V = 16 / sizeof(T);                                                    \
    if (k == 1) { constexpr int K = 1; __VA_ARGS__; }                                     \
    else if (k == 2) { constexpr int K = 2; __VA_ARGS__; }                                \
    else if (k <= 4) { constexpr int K = 4; __VA_ARGS__; }                                \
    else { constexpr int K = 8; __VA_ARGS__; }                                            \
  } else {                                                                               \
    constexpr int V = 1;                                                                 \
    if (k <= 2) { constexpr int K = 2; __VA_ARGS__; }                                     \
    else { constexpr int K = 8; __VA_ARGS__; }                                            \
  }

hipError_t rows_fwd(int dtype, const Args& a, int V_, hipStream_t s) {
  int k;
  const Rows w = rows_of(a.N, a.C, a.G, V_, false, k);
  KFB_DISPATCH_DTYPE(dtype, T, KFB_DISPATCH_ACT(a.act.kind, KIND, KFB_ROWS(T, V_, k, V, K, {
    hipLaunchKernelGGL((gn_rows_fwd_k<T, V, KIND, K>), dim3(ceil_div((long)w.sets * w.L, RNT)),
                       dim3(RNT), 0, s, a, w);
  })));
  return hipGetLastError();
}

hipError_t rows_bwd(int dtype, const Args& a, int V_, hipStream_t s) {
  int k;
  const Rows w = rows_of(a.N, a.C, a.G, V_, true, k);
  KFB_DISPATCH_DTYPE(dtype, T, KFB_DISPATCH_ACT(a.act.kind, KIND, KFB_ROWS(T, V_, k, V, K, {
    hipLaunchKernelGGL((gn_rows_bwd_k<T, V, KIND, K>), dim3(ceil_div((long)w.sets * w.L, RNT)),
                       dim3(RNT), 0, s, a, w);
  })));
  return hipGetLastError();
}

}  // namespace gn
}  // namespace kfb
