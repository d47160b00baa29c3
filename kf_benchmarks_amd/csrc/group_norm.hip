// Group norm with an activation on channels-last activations [N][HW][C]:
// group g of image n is HW rows x cpg = C / G channels, M = HW cpg values,
//   mu = mean, r = 1 / sqrt(var + eps), xh = (x - mu) r,
//   y = act(gamma xh + beta);
//   e = dy act'(gamma xh + beta), dbeta = sum e, dgamma = sum e xh,
//   dx = r (gamma e - (s1 + xh s2) / M), s1 = sum_g gamma e, s2 = sum_g gamma e xh.
// The backward recomputes xh and the activation from x: nothing but mu and r
// is stored.  All sums are fp32; the variance is that of the centred values.
#include "act.h"

namespace kfb {
namespace gn {

constexpr int NT = 256;

struct Args {
  const void* x;
  const void* dy;
  void* y;  // forward: y, backward: dx
  const float *gamma, *beta;
  float *mean, *rstd;  // [N][G]
  float* part;         // backward: [N][2][C], sum e xh | sum e of each image
  long N, HW;
  int C, G, cpg, act;
  float eps;
};

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) s += red[w];
  return s;
}

// One workgroup per (image, group), lanes along the channels: TC columns x
// NT / TC rows, TC a power of two.
template <typename T>
__global__ void __launch_bounds__(NT) gn_fwd_any_k(Args a, int tc) {
  __shared__ float red[NT / 64];
  const int c0 = threadIdx.x % tc, r0 = threadIdx.x / tc, rp = NT / tc;
  for (long id = blockIdx.x; id < a.N * a.G; id += gridDim.x) {
  const int g = (int)(id % a.G);
  const long n = id / a.G;
  const T* __restrict__ x = (const T*)a.x + n * a.HW * a.C + (long)g * a.cpg;
  T* __restrict__ y = (T*)a.y + n * a.HW * a.C + (long)g * a.cpg;
  const float inv = 1.f / ((float)a.HW * a.cpg);
  float s = 0.f;
  for (long r = r0; r < a.HW; r += rp)
    for (int c = c0; c < a.cpg; c += tc) s += to_f32(x[r * a.C + c]);
  const float mu = block_sum(s, red) * inv;
  s = 0.f;
  for (long r = r0; r < a.HW; r += rp)
    for (int c = c0; c < a.cpg; c += tc) {
      const float d = to_f32(x[r * a.C + c]) - mu;
      s = fmaf(d, d, s);
    }
  const float rs = 1.f / sqrtf(block_sum(s, red) * inv + a.eps);
  if (threadIdx.x == 0) {
    a.mean[id] = mu;
    a.rstd[id] = rs;
  }
  for (int c = c0; c < a.cpg; c += tc) {
    const int ch = g * a.cpg + c;
    const float ga = a.gamma ? a.gamma[ch] : 1.f, be = a.beta ? a.beta[ch] : 0.f;
    for (long r = r0; r < a.HW; r += rp)
      y[r * a.C + c] = from_f32<T>(act_fwd(fmaf((to_f32(x[r * a.C + c]) - mu) * rs, ga, be), a.act));
  }
  }
}

template <typename T>
__global__ void __launch_bounds__(NT) gn_bwd_any_k(Args a, int tc) {
  __shared__ float red[NT / 64], colp[NT], colq[NT];
  const int c0 = threadIdx.x % tc, r0 = threadIdx.x / tc, rp = NT / tc;
  for (long id = blockIdx.x; id < a.N * a.G; id += gridDim.x) {
  const int g = (int)(id % a.G);
  const long n = id / a.G;
  const long base = n * a.HW * a.C + (long)g * a.cpg;
  const T* __restrict__ x = (const T*)a.x + base;
  const T* __restrict__ dy = (const T*)a.dy + base;
  T* __restrict__ dx = (T*)a.y + base;
  const float mu = a.mean[id], rs = a.rstd[id];
  float s1 = 0.f, s2 = 0.f;
  for (int cb = 0; cb < a.cpg; cb += tc) {
    const int c = cb + c0, ch = g * a.cpg + c;
    const bool on = c < a.cpg;
    const float ga = on && a.gamma ? a.gamma[ch] : 1.f, be = on && a.beta ? a.beta[ch] : 0.f;
    float p = 0.f, q = 0.f;
    if (on)
      for (long r = r0; r < a.HW; r += rp) {
        const float xh = (to_f32(x[r * a.C + c]) - mu) * rs;
        const float e = to_f32(dy[r * a.C + c]) * act_grad(fmaf(xh, ga, be), a.act);
        p += e;
        q = fmaf(e, xh, q);
      }
    __syncthreads();
    colp[threadIdx.x] = p;
    colq[threadIdx.x] = q;
    __syncthreads();
    if (r0 == 0 && on) {
      for (int r = 1; r < rp; ++r) {
        p += colp[r * tc + c0];
        q += colq[r * tc + c0];
      }
      a.part[n * 2 * a.C + ch] = q;
      a.part[n * 2 * a.C + a.C + ch] = p;
      s1 = fmaf(ga, p, s1);
      s2 = fmaf(ga, q, s2);
    }
  }
  const float inv = 1.f / ((float)a.HW * a.cpg);
  s1 = block_sum(s1, red) * inv;
  s2 = block_sum(s2, red) * inv;
  for (int c = c0; c < a.cpg; c += tc) {
    const int ch = g * a.cpg + c;
    const float ga = a.gamma ? a.gamma[ch] : 1.f, be = a.beta ? a.beta[ch] : 0.f;
    for (long r = r0; r < a.HW; r += rp) {
      const float xh = (to_f32(x[r * a.C + c]) - mu) * rs;
      const float e = to_f32(dy[r * a.C + c]) * act_grad(fmaf(xh, ga, be), a.act);
      dx[r * a.C + c] = from_f32<T>(rs * (fmaf(ga, e, -s1) - xh * s2));
    }
  }
  }
}

// dgamma / dbeta = sum over the slabs of part [S][2][C], in slab order per
// thread row and then over the rows: the same sum on every run.
__global__ void __launch_bounds__(NT)
gn_param_grad_k(const float* __restrict__ part, long S, int C, float* __restrict__ dgamma,
                float* __restrict__ dbeta, int acc_g, int acc_b) {
  __shared__ float red[NT];
  const int cl = threadIdx.x % 16, r0 = threadIdx.x / 16;
  const int c = blockIdx.x * 16 + cl;  // of 2 C
  float s = 0.f;
  if (c < 2 * C)
    for (long r = r0; r < S; r += NT / 16) s += part[r * 2 * C + c];
  red[threadIdx.x] = s;
  __syncthreads();
  if (r0 == 0 && c < 2 * C) {
    for (int r = 1; r < NT / 16; ++r) s += red[r * 16 + cl];
    float* out = c < C ? dgamma : dbeta;
    const int acc = c < C ? acc_g : acc_b, i = c < C ? c : c - C;
    if (out) out[i] = acc ? out[i] + s : s;
  }
}

// a launch holds fewer than 2^32 threads: the workgroups loop over the rest
inline dim3 groups_grid(long N, int G) { return dim3((unsigned)(N * G < (1l << 20) ? N * G : 1l << 20)); }

inline int columns(int cpg) {
  int tc = 1;
  while (tc < cpg && tc < NT) tc *= 2;
  return tc;
}

}  // namespace gn
}  // namespace kfb

using namespace kfb;

// Workspace (floats) of the forward and of the backward.
KFB_API long kfb_gn_fwd_ws(int dtype, long N, long HW, int C, int G) { return 0; }
KFB_API long kfb_gn_bwd_ws(int dtype, long N, long HW, int C, int G) { return N * 2 * C; }

KFB_API hipError_t kfb_gn_fwd(int dtype, const void* x, void* y, long N, long HW, int C, int G,
                              const float* gamma, const float* beta, float eps, int act,
                              float* mean, float* rstd, float* ws, hipStream_t stream) {
  if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G) return hipErrorInvalidValue;
  gn::Args a{x, nullptr, y, gamma, beta, mean, rstd, nullptr, N, HW, C, G, C / G, act, eps};
  KFB_DISPATCH_DTYPE(dtype, T, {
    hipLaunchKernelGGL((gn::gn_fwd_any_k<T>), gn::groups_grid(N, G), dim3(gn::NT), 0, stream, a,
                       gn::columns(C / G));
  });
  return hipGetLastError();
}

KFB_API hipError_t kfb_gn_bwd(int dtype, const void* dy, const void* x, void* dx, long N, long HW,
                              int C, int G, const float* gamma, const float* beta, int act,
                              const float* mean, const float* rstd, float* dgamma, float* dbeta,
                              int acc_gamma, int acc_beta, float* ws, hipStream_t stream) {
  if (N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || !ws)
    return hipErrorInvalidValue;
  gn::Args a{x, dy, dx, gamma, beta, (float*)mean, (float*)rstd, ws, N, HW, C, G, C / G, act, 0.f};
  KFB_DISPATCH_DTYPE(dtype, T, {
    hipLaunchKernelGGL((gn::gn_bwd_any_k<T>), gn::groups_grid(N, G), dim3(gn::NT), 0, stream, a,
                       gn::columns(C / G));
  });
  if (dgamma || dbeta)
    hipLaunchKernelGGL(gn::gn_param_grad_k, dim3(ceil_div(2 * C, 16)), dim3(gn::NT), 0, stream, ws,
                       N, C, dgamma, dbeta, acc_gamma, acc_beta);
  return hipGetLastError();
}
