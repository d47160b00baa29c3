// Short causal convolution over time, per channel, with a bias and an
// activation, on time-major sequences [T][B][D]:
//   u_s = bias + sum_k w[k] x_{s - K + 1 + k},  y_s = act(u_s),  1 <= K <= 8,
// w [K][D], bias [D] fp32; x before a sequence's start is its state [K-1][B][D]
// or zero.  Position s is time s, or len - 1 - s in reverse; rows at or past a
// sequence's length give y = 0 and take no gradient.
//
// Bound by HBM.  A thread owns V channels (16 bytes) of one sequence and a run
// of RUN positions, with the last K inputs in registers: each input is read
// once, and the K - 1 inputs before a run once more (from cache).
#include "act.h"

namespace kfb {
namespace cconv {

constexpr int RUN = 16, KMAX = 8;

struct Args {
  const void *x, *dy, *x0;  // x0: state [K-1][B][D] or null
  long ldx, ldy;
  const float *w, *bias;
  const int* len;
  void *y, *xT;             // xT: state after the last position, or null
  void *dx, *dx0;
  const void* dxT;          // gradient of xT or null
  float* part;              // [slabs][K + 1][D], dw | dbias
  int T, B, D, K, reverse;
  Act act;
};

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return a.len ? min(max(a.len[b], 0), a.T) : a.T;
}

__device__ __forceinline__ long row_of(const Args& a, int b, int s, int len) {
  const int t = a.reverse && s < len ? len - 1 - s : s;
  return (long)t * a.B + b;
}

// input at position s (< len) of sequence b: the state for s < 0
template <typename T, int V>
__device__ __forceinline__ void input(const Args& a, int b, int c, int s, int len, float (&v)[V]) {
  if (s >= 0 && s < len) {
    load_vec<T, V>((const T*)a.x + row_of(a, b, s, len) * a.ldx + c, v);
  } else if (s < 0 && s >= 1 - a.K && a.x0) {
    load_vec<T, V>((const T*)a.x0 + ((long)(s + a.K - 1) * a.B + b) * a.D + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.f;
  }
}

template <typename T, int V, int KIND>
__global__ void __launch_bounds__(256) fwd_k(Args a, int runs) {
  const int cv = a.D / V;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)cv * a.B) return;
  const int c = (int)(i % cv) * V, b = (int)(i / cv), K = a.K;
  const int len = seq_len(a, b);
  if ((int)blockIdx.y == runs) {  // the state after the last position
    for (int j = 0; j < K - 1; ++j) {
      float v[V];
      input<T, V>(a, b, c, len - (K - 1) + j, len, v);
      store_vec<T, V>((T*)a.xT + ((long)j * a.B + b) * a.D + c, v);
    }
    return;
  }
  float bias[V];
#pragma unroll
  for (int k = 0; k < V; ++k) bias[k] = a.bias ? a.bias[c + k] : 0.f;
  const int s0 = blockIdx.y * RUN, s1 = min(s0 + RUN, a.T);
  for (int s = s0; s < s1; ++s) {
    float u[V];
#pragma unroll
    for (int k = 0; k < V; ++k) u[k] = 0.f;
    if (s < len) {
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] = bias[k];
      for (int j = 0; j < K; ++j) {
        float v[V];
        input<T, V>(a, b, c, s - K + 1 + j, len, v);
#pragma unroll
        for (int k = 0; k < V; ++k) u[k] = fmaf(a.w[(long)j * a.D + c + k], v[k], u[k]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] = act_fwd<KIND>(u[k], a.act);
    }
    store_vec<T, V>((T*)a.y + row_of(a, b, s, len) * a.D + c, u);
  }
}

// gradient of u at position s
template <typename T, int V, int KIND>
__device__ __forceinline__ void pre_grad(const Args& a, int b, int c, int s, int len,
                                         const float (&bias)[V], float (&e)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) e[k] = 0.f;
  if (s < 0 || s >= len) return;
  float u[V];
#pragma unroll
  for (int k = 0; k < V; ++k) u[k] = bias[k];
  if (a.act.kind != CLAMP || a.act.lo == 0.f)
    for (int j = 0; j < a.K; ++j) {
      float v[V];
      input<T, V>(a, b, c, s - a.K + 1 + j, len, v);
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] = fmaf(a.w[(long)j * a.D + c + k], v[k], u[k]);
    }
  load_vec<T, V>((const T*)a.dy + row_of(a, b, s, len) * a.ldy + c, e);
#pragma unroll
  for (int k = 0; k < V; ++k) e[k] *= act_grad<KIND>(u[k], a.act);
}

// dx_s = sum_k w[k] e_{s + K - 1 - k}; for s < 0 that is the state's gradient.
// The last K - 1 inputs also take the gradient of the state that was returned.
template <typename T, int V, int KIND>
__global__ void __launch_bounds__(256) dgrad_k(Args a, int runs) {
  const int cv = a.D / V;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)cv * a.B) return;
  const int c = (int)(i % cv) * V, b = (int)(i / cv), K = a.K;
  const int len = seq_len(a, b);
  float bias[V];
#pragma unroll
  for (int k = 0; k < V; ++k) bias[k] = a.bias ? a.bias[c + k] : 0.f;
  const bool state = (int)blockIdx.y == runs;
  const int s0 = state ? 1 - K : blockIdx.y * RUN, s1 = state ? 0 : min(s0 + RUN, a.T);
  for (int s = s0; s < s1; ++s) {
    float g[V];
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = 0.f;
    if (s < len) {
      for (int j = 0; j < K; ++j) {
        float e[V];
        pre_grad<T, V, KIND>(a, b, c, s + K - 1 - j, len, bias, e);
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] = fmaf(a.w[(long)j * a.D + c + k], e[k], g[k]);
      }
      if (a.dxT && s >= len - (K - 1)) {
        float v[V];
        load_vec<T, V>((const T*)a.dxT + ((long)(s - len + K - 1) * a.B + b) * a.D + c, v);
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] += v[k];
      }
    }
    if (state) store_vec<T, V>((T*)a.dx0 + ((long)(s + K - 1) * a.B + b) * a.D + c, g);
    else store_vec<T, V>((T*)a.dx + row_of(a, b, s, len) * a.D + c, g);
  }
}

// dw[k] = sum e_s x_{s - K + 1 + k}, dbias = sum e_s: a slab of jobs
// (sequence, run) per workgroup row, no atomics.
template <typename T, int V, int KIND>
__global__ void __launch_bounds__(256) wgrad_k(Args a, int runs, int slabs) {
  const int cv = a.D / V;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= cv) return;
  const int c = i * V, K = a.K;
  float bias[V], acc[KMAX + 1][V];
#pragma unroll
  for (int k = 0; k < V; ++k) bias[k] = a.bias ? a.bias[c + k] : 0.f;
#pragma unroll
  for (int j = 0; j <= KMAX; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) acc[j][k] = 0.f;
  for (long job = blockIdx.y; job < (long)a.B * runs; job += slabs) {
    const int b = (int)(job % a.B), s0 = (int)(job / a.B) * RUN, len = seq_len(a, b);
    for (int s = s0; s < min(s0 + RUN, len); ++s) {
      float e[V];
      pre_grad<T, V, KIND>(a, b, c, s, len, bias, e);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[KMAX][k] += e[k];
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        if (j >= K) break;
        float v[V];
        input<T, V>(a, b, c, s - K + 1 + j, len, v);
#pragma unroll
        for (int k = 0; k < V; ++k) acc[j][k] = fmaf(e[k], v[k], acc[j][k]);
      }
    }
  }
  float* out = a.part + (long)blockIdx.y * (K + 1) * a.D + c;
#pragma unroll
  for (int k = 0; k < V; ++k) {
#pragma unroll
    for (int j = 0; j < KMAX; ++j)
      if (j < K) out[(long)j * a.D + k] = acc[j][k];
    out[(long)K * a.D + k] = acc[KMAX][k];
  }
}

__global__ void __launch_bounds__(256)
param_grad_k(const float* __restrict__ p, int S, int K, int D, float* dw, float* db, int acc_w,
             int acc_b) {
  const long total = (long)(K + 1) * D;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int k = 0; k < S; ++k) s += p[k * total + i];
  const bool isw = i < (long)K * D;
  float* out = isw ? dw : db;
  if (!out) return;
  out += isw ? i : i - (long)K * D;
  *out = (isw ? acc_w : acc_b) ? *out + s : s;
}

// One token: y from the state and x, the state [K-1][B][D] moved on by one.
template <typename T, int V, int KIND>
__global__ void __launch_bounds__(256) step_k(Args a, T* __restrict__ state) {
  const int cv = a.D / V;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)cv * a.B) return;
  const int c = (int)(i % cv) * V, b = (int)(i / cv), K = a.K;
  float u[V], v[V];
#pragma unroll
  for (int k = 0; k < V; ++k) u[k] = a.bias ? a.bias[c + k] : 0.f;
  for (int j = 0; j < K; ++j) {
    if (j < K - 1) load_vec<T, V>(state + ((long)j * a.B + b) * a.D + c, v);
    else load_vec<T, V>((const T*)a.x + b * a.ldx + c, v);
#pragma unroll
    for (int k = 0; k < V; ++k) u[k] = fmaf(a.w[(long)j * a.D + c + k], v[k], u[k]);
    if (j) store_vec<T, V>(state + ((long)(j - 1) * a.B + b) * a.D + c, v);
  }
#pragma unroll
  for (int k = 0; k < V; ++k) u[k] = act_fwd<KIND>(u[k], a.act);
  store_vec<T, V>((T*)a.y + (long)b * a.D + c, u);
}

inline bool bad(const Args& a) {
  return a.T <= 0 || a.B <= 0 || a.D <= 0 || a.K < 1 || a.K > KMAX;
}

inline int slabs(long jobs) { return (int)(jobs < 256 ? jobs : 256); }

}  // namespace cconv
}  // namespace kfb

using namespace kfb;

#define KFB_CCONV_VEC(T, vec, V, ...)                                     \
  if (vec) { constexpr int V = 16 / sizeof(T); __VA_ARGS__; }              \
  else { constexpr int V = 1; __VA_ARGS__; }

KFB_API int kfb_cconv_max_taps() { return cconv::KMAX; }

KFB_API long kfb_cconv_bwd_ws(int T, int B, int D, int K) {
  return (long)cconv::slabs((long)B * ceil_div(T, cconv::RUN)) * (K + 1) * D;
}

KFB_API hipError_t kfb_cconv_fwd(int dtype, int vec, const void* x, long ldx, const void* x0,
                                 const float* w, const float* bias, const int* len, void* y,
                                 void* xT, int T, int B, int D, int K, int act, int reverse,
                                 hipStream_t stream) {
  cconv::Args a{};
  a.x = x; a.ldx = ldx; a.x0 = x0; a.w = w; a.bias = bias; a.len = len; a.y = y; a.xT = xT;
  a.T = T; a.B = B; a.D = D; a.K = K; a.act = act_of(act); a.reverse = reverse;
  const int runs = ceil_div(T, cconv::RUN);
  if (cconv::bad(a) || runs > 65534) return hipErrorInvalidValue;
  KFB_DISPATCH_DTYPE(dtype, E, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    KFB_CCONV_VEC(E, vec, V, {
      hipLaunchKernelGGL((cconv::fwd_k<E, V, KIND>), dim3(ceil_div((long)D / V * B, 256), runs + (xT && K > 1 ? 1 : 0)),
                         dim3(256), 0, stream, a, runs);
    });
  }));
  return hipGetLastError();
}

KFB_API hipError_t kfb_cconv_bwd(int dtype, int vec, const void* dy, long ldy, const void* x,
                                 long ldx, const void* x0, const float* w, const float* bias,
                                 const int* len, const void* dxT, void* dx, void* dx0, float* dw,
                                 float* db, int acc_w, int acc_b, float* ws, int T, int B, int D,
                                 int K, int act, int reverse, hipStream_t stream) {
  cconv::Args a{};
  a.dy = dy; a.ldy = ldy; a.x = x; a.ldx = ldx; a.x0 = x0; a.w = w; a.bias = bias; a.len = len;
  a.dxT = dxT; a.dx = dx; a.dx0 = dx0; a.part = ws;
  a.T = T; a.B = B; a.D = D; a.K = K; a.act = act_of(act); a.reverse = reverse;
  const int runs = ceil_div(T, cconv::RUN);
  if (cconv::bad(a) || runs > 65534 || !ws) return hipErrorInvalidValue;
  const int S = cconv::slabs((long)B * runs);
  KFB_DISPATCH_DTYPE(dtype, E, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    KFB_CCONV_VEC(E, vec, V, {
      hipLaunchKernelGGL((cconv::dgrad_k<E, V, KIND>), dim3(ceil_div((long)D / V * B, 256), runs + (dx0 && K > 1 ? 1 : 0)),
                         dim3(256), 0, stream, a, runs);
      hipLaunchKernelGGL((cconv::wgrad_k<E, V, KIND>), dim3(ceil_div(D / V, 256), S), dim3(256), 0, stream,
                         a, runs, S);
    });
  }));
  hipLaunchKernelGGL(cconv::param_grad_k, dim3(ceil_div((long)(K + 1) * D, 256)), dim3(256), 0,
                     stream, ws, S, K, D, dw, db, acc_w, acc_b);
  return hipGetLastError();
}

KFB_API hipError_t kfb_cconv_step(int dtype, int vec, const void* x, long ldx, void* state,
                                  const float* w, const float* bias, void* y, int B, int D, int K,
                                  int act, hipStream_t stream) {
  cconv::Args a{};
  a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.y = y;
  a.T = 1; a.B = B; a.D = D; a.K = K; a.act = act_of(act);
  if (cconv::bad(a)) return hipErrorInvalidValue;
  KFB_DISPATCH_DTYPE(dtype, E, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    KFB_CCONV_VEC(E, vec, V, {
      hipLaunchKernelGGL((cconv::step_k<E, V, KIND>), dim3(ceil_div((long)D / V * B, 256)), dim3(256), 0,
                         stream, a, (E*)state);
    });
  }));
  return hipGetLastError();
}
