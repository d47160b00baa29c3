// Short causal convolution over time, per channel, with a bias and an
// activation, on time-major sequences [T][B][D]:
//   u_s = bias + sum_k w[k] x_{s - K + 1 + k},  y_s = act(u_s),  1 <= K <= 8,
// w [K][D], bias [D] fp32; x before a sequence's start is its state [K-1][B][D]
// or zero.  Position s is time s, or len - 1 - s in reverse; rows at or past a
// sequence's length give y = 0 and take no gradient.
//
// Bound by HBM.  A thread owns V channels of one sequence and a run of positions,
// with the last K inputs (backward: also the last K gradients of u) in registers
// and a batch of loads in flight: each input is read once, and the K - 1 rows next to a
// run once more (from cache).  u is computed again in the backward, nothing but x
// is kept.  874 x 16 x 1600 bf16 values, 4 taps, SiLU: 22.3 us forward (4.0 TB/s; a
// copy reaches 5.2), 44 us backward (3.1 TB/s).
#include "act.h"
#include "raw.h"

namespace kfb {
namespace cconv {

// most taps; positions whose loads are in flight together, forward and backward
// (backward with 8: 216 registers, 62 us for 874 x 16 x 1600 bf16, with 4: 158, 44 us)
constexpr int KMAX = 8, UF = 8, UB = 4;

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

// One sequence's rows of a [T][B] tensor: position s (< len) at base + s * step.
// Loads are unconditional, of the nearest position inside (row 0 of an empty
// sequence), and zeroed after: no branch stands between the loads in flight.
template <typename T> struct Line {
  T* base;
  long step;
  int len;

  template <int V> __device__ __forceinline__ void load(int s, Raw<T, V>& v) const {
    v.load(base + min(s, len > 0 ? len - 1 : 0) * step);
    v.keep(s < len);
  }
};

template <typename T>
__device__ __forceinline__ Line<T> line(const Args& a, const void* p, long ld, int b, int c, int len) {
  const long step = (long)a.B * ld;
  Line<T> l{(T*)p + (long)b * ld + c, step, len};
  if (a.reverse && len > 0) {
    l.base += (len - 1) * step;
    l.step = -step;
  }
  return l;
}

// the input at position s, which may lie before the sequence: its state
template <typename T, int V>
__device__ __forceinline__ void input(const Args& a, const Line<T>& x, int b, int c, int s, Raw<T, V>& v) {
  if (s >= 0) x.load(s, v);
  else if (s >= 1 - a.K && a.x0) v.load((const T*)a.x0 + ((long)(s + a.K - 1) * a.B + b) * a.D + c);
  else v.zero();
}

// w[j], j = 0..KP-1, are the taps of the inputs s - KP + 1 .. s; those before the
// K used ones are skipped, not multiplied by zero (0 * inf).
template <int KP, int V>
__device__ __forceinline__ void load_taps(const Args& a, int c, float (&w)[KP][V]) {
#pragma unroll
  for (int j = 0; j < KP; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) w[j][k] = j >= KP - a.K ? a.w[(long)(j - KP + a.K) * a.D + c + k] : 0.f;
}

template <typename T, int V, int KIND, int KP, bool EXACT>
__global__ void __launch_bounds__(256) fwd_k(Args a, int run, int runs) {
  const int cv = a.D / V;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)cv * a.B) return;
  const int c = (int)(i % cv) * V, b = (int)(i / cv), skip = EXACT ? 0 : KP - a.K;
  const int len = seq_len(a, b);
  const Line<T> x = line<T>(a, a.x, a.ldx, b, c, len);
  if ((int)blockIdx.y == runs) {  // the state after the last position
    for (int j = 0; j < a.K - 1; ++j) {
      Raw<T, V> v;
      float f[V];
      input<T, V>(a, x, b, c, len - (a.K - 1) + j, v);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = v[k];
      store_vec<T, V>((T*)a.xT + ((long)j * a.B + b) * a.D + c, f);
    }
    return;
  }
  const Line<T> y = line<T>(a, a.y, (long)a.D, b, c, len);
  float w[KP][V], bias[V];
  load_taps<KP, V>(a, c, w);
#pragma unroll
  for (int k = 0; k < V; ++k) bias[k] = a.bias ? a.bias[c + k] : 0.f;
  const int s0 = blockIdx.y * run, s1 = min(s0 + run, a.T);
  Raw<T, V> win[KP - 1 + UF];
#pragma unroll
  for (int j = 0; j < KP - 1; ++j) input<T, V>(a, x, b, c, s0 - KP + 1 + j, win[j]);
  for (int s = s0; s < s1; s += UF) {
#pragma unroll
    for (int r = 0; r < UF; ++r) x.load(s + r, win[KP - 1 + r]);
#pragma unroll
    for (int r = 0; r < UF; ++r) {
      float u[V];
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] = bias[k];
#pragma unroll
      for (int j = 0; j < KP; ++j)
        if (EXACT || j >= skip)
#pragma unroll
          for (int k = 0; k < V; ++k) u[k] = fmaf(w[j][k], win[r + j][k], u[k]);
#pragma unroll
      for (int k = 0; k < V; ++k) u[k] = s + r < len ? act_fwd<KIND>(u[k], a.act) : 0.f;
      T* at = s + r < len ? y.base + (s + r) * y.step : (T*)a.y + ((long)(s + r) * a.B + b) * a.D + c;
      if (s + r < s1) store_vec<T, V>(at, u);
    }
#pragma unroll
    for (int j = 0; j < KP - 1; ++j) win[j] = win[UF + j];
  }
}

// Going up through the positions p of a run and the K - 1 behind it:
//   e_p = dy_p act'(u_p);  dw[k] += e_p x_{p-K+1+k}, dbias += e_p (p in the run);
//   dx_s = sum_k w[k] e_{s+K-1-k} is complete at p = s + K - 1; s < 0 is the state,
//   and the last K - 1 inputs take the gradient of the state that was returned.
// A workgroup is CX column vectors x 256 / CX jobs (sequence, run); its parameter
// sums go to its slab of part, no atomics.
template <typename T, int V, int KIND, int KP, bool EXACT, int CX>
__global__ void __launch_bounds__(256) bwd_k(Args a, int run, int runs) {
  constexpr int JY = 256 / CX;
  __shared__ float red[JY][CX * V + 1];
  const int K = EXACT ? KP : a.K, skip = KP - K;
  const int cl = threadIdx.x % CX, ty = threadIdx.x / CX;
  const int c = (blockIdx.x * CX + cl) * V;
  const bool on = c < a.D;
  float w[KP][V], bias[V], dw[KP][V], db[V];
#pragma unroll
  for (int j = 0; j < KP; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) dw[j][k] = w[j][k] = 0.f;
#pragma unroll
  for (int k = 0; k < V; ++k) db[k] = bias[k] = 0.f;
  float wl[EXACT ? 1 : KP][V];  // tap j at j, where w has it at j + skip
  if constexpr (!EXACT)
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) wl[j][k] = on && j < K ? a.w[(long)j * a.D + c + k] : 0.f;
  if (on) {
    load_taps<KP, V>(a, c, w);
#pragma unroll
    for (int k = 0; k < V; ++k) bias[k] = a.bias ? a.bias[c + k] : 0.f;
  }
  const bool linear = KIND == CLAMP && a.act.lo != a.act.lo;
  const long jobs = on ? (long)a.B * runs : 0;
  for (long job = (long)blockIdx.y * JY + ty; job < jobs; job += (long)gridDim.y * JY) {
    const int b = (int)(job / runs), s0 = (int)(job % runs) * run, s1 = min(s0 + run, a.T);
    const int len = seq_len(a, b);
    const Line<T> x = line<T>(a, a.x, a.ldx, b, c, len), dy = line<T>(a, a.dy, a.ldy, b, c, len),
                  dx = line<T>(a, a.dx, (long)a.D, b, c, len);
    Raw<T, V> win[KP - 1 + UB];
    float ew[KP][V];  // e at p - KP + 1 .. p
#pragma unroll
    for (int j = 0; j < KP - 1; ++j) input<T, V>(a, x, b, c, s0 - KP + 1 + j, win[j]);
#pragma unroll
    for (int j = 0; j < KP; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) ew[j][k] = 0.f;
    const int end = s1 + K - 1;
    for (int p0 = s0; p0 < end; p0 += UB) {
      Raw<T, V> g[UB];
#pragma unroll
      for (int r = 0; r < UB; ++r) {
        x.load(p0 + r, win[KP - 1 + r]);
        dy.load(p0 + r, g[r]);
      }
#pragma unroll
      for (int r = 0; r < UB; ++r) {
        const int p = p0 + r;
        float e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = bias[k];
        if (!linear)
#pragma unroll
          for (int j = 0; j < KP; ++j)
            if (EXACT || j >= skip)
#pragma unroll
              for (int k = 0; k < V; ++k) e[k] = fmaf(w[j][k], win[r + j][k], e[k]);
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = p < len ? g[r][k] * act_grad<KIND>(e[k], a.act) : 0.f;
#pragma unroll
        for (int j = 0; j < KP - 1; ++j)
#pragma unroll
          for (int k = 0; k < V; ++k) ew[j][k] = ew[j + 1][k];
#pragma unroll
        for (int k = 0; k < V; ++k) ew[KP - 1][k] = e[k];
        const bool own = p < s1 && p < len;  // (0 times infinity is not 0)
#pragma unroll
        for (int j = 0; j < KP; ++j)
          if (EXACT || j >= skip)
#pragma unroll
            for (int k = 0; k < V; ++k) dw[j][k] = own ? fmaf(e[k], win[r + j][k], dw[j][k]) : dw[j][k];
#pragma unroll
        for (int k = 0; k < V; ++k) db[k] += own ? e[k] : 0.f;
        const int s = p - K + 1;
        float o[V];
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = 0.f;
#pragma unroll
        for (int j = 0; j < KP; ++j)  // tap j with e_{p - j}
          if (EXACT || j < K)
#pragma unroll
            for (int k = 0; k < V; ++k)
              o[k] = fmaf(EXACT ? w[j][k] : wl[EXACT ? 0 : j][k], ew[KP - 1 - j][k], o[k]);
        if (a.dxT && s < s1 && s < len && s >= len - (K - 1)) {
          Raw<T, V> v;
          v.load((const T*)a.dxT + ((long)(s - len + K - 1) * a.B + b) * a.D + c);
#pragma unroll
          for (int k = 0; k < V; ++k) o[k] += v[k];
        }
        T* at = s < 0 ? (T*)a.dx0 + ((long)(s + K - 1) * a.B + b) * a.D + c
              : s < len ? dx.base + s * dx.step
                        : (T*)a.dx + ((long)s * a.B + b) * a.D + c;
        if (s < s1 && (s >= s0 || (s0 == 0 && a.dx0))) store_vec<T, V>(at, o);
      }
#pragma unroll
      for (int j = 0; j < KP - 1; ++j) win[j] = win[UB + j];
    }
  }
  // the slab [K + 1][D] of this workgroup row
#pragma unroll
  for (int j = 0; j <= KP; ++j) {
    if (j < KP && !EXACT && j < skip) continue;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) red[ty][cl * V + k] = j < KP ? dw[j < KP ? j : 0][k] : db[k];
    __syncthreads();
    for (int i = threadIdx.x; i < CX * V; i += 256) {
      const int ch = blockIdx.x * CX * V + i;
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < JY; ++r) sum += red[r][i];
      if (ch < a.D) a.part[((long)blockIdx.y * (K + 1) + (j < KP ? j - skip : K)) * a.D + ch] = sum;
    }
  }
}

// dw [K][D], dbias [D]: the sum over the slabs, 32 columns x 8 rows a workgroup
__global__ void __launch_bounds__(256)
param_grad_k(const float* __restrict__ p, int S, int K, int D, float* dw, float* db, int acc_w,
             int acc_b) {
  __shared__ float red[8][33];
  const long total = (long)(K + 1) * D;
  const int cl = threadIdx.x % 32, r0 = threadIdx.x / 32;
  const long i = (long)blockIdx.x * 32 + cl;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (i < total)
    for (int r = r0; r < S; r += 32)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (r + 8 * k < S) s[k] += p[(long)(r + 8 * k) * total + i];
  red[r0][cl] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (r0 || i >= total) return;
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) sum += red[r][cl];
  const bool isw = i < (long)K * D;
  float* out = isw ? dw : db;
  if (!out) return;
  out += isw ? i : i - (long)K * D;
  *out = (isw ? acc_w : acc_b) ? *out + sum : sum;
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

// y [T][B][D] = x with the rows at or past each sequence's length zero, whatever they
// hold: a wave a row.
template <typename T, int V>
__global__ void __launch_bounds__(256) mask_rows_k(const T* __restrict__ x, long ldx, const int* __restrict__ len,
                                                   T* __restrict__ y, long rows, int B, int D) {
  for (long row = (long)blockIdx.x * 4 + threadIdx.x / 64; row < rows; row += (long)gridDim.x * 4) {
    const bool on = row / B < len[row % B];
    for (int c = threadIdx.x % 64 * V; c < D; c += 64 * V) {
      Raw<T, V> v;
      float f[V];
      if (on) v.load(x + row * ldx + c);
      else v.zero();
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = v[k];
      store_vec<T, V>(y + row * D + c, f);
    }
  }
}

inline bool bad(const Args& a) {
  return a.T <= 0 || a.B <= 0 || a.D <= 0 || a.K < 1 || a.K > KMAX;
}

// Positions of a thread's run: long runs read few rows twice, short ones fill the
// card (2048 waves; 874 x 16 x 1600 bf16 values: 22.5 us forward and 45.1 backward,
// with 1024 waves 27.0 and 60.8, with 4096 24.2 and 50.4).  A launch has at most
// 65535 runs.
inline int run_of(long T, long lanes) {
  int run = 64;
  while (run > 8 && lanes * ceil_div(T, run) < 2048 * 64 && ceil_div(T, run / 2) < 65000) run /= 2;
  return run;
}

constexpr int BV = 4, BCX = 32;  // backward: channels of a vector, vectors of a workgroup row

inline int bwd_slabs(int T, int B, int D, int run) {
  const long rows = ceil_div((long)B * ceil_div(T, run), 256 / BCX);
  const long most = ceil_div(2048, ceil_div(D, BCX * BV));
  return (int)(rows < most ? rows : most);
}

}  // namespace cconv
}  // namespace kfb

using namespace kfb;

#define KFB_CCONV_VEC(vec, WIDE, V, ...)         \
  if (vec) { constexpr int V = WIDE; __VA_ARGS__; } \
  else { constexpr int V = 1; __VA_ARGS__; }

// filter lengths: 2, 3 and 4 with everything unrolled, the others inside 8
#define KFB_CCONV_TAPS(K, KP, EXACT, ...)                                  \
  switch (K) {                                                             \
    case 2: { constexpr int KP = 2; constexpr bool EXACT = true; __VA_ARGS__; break; } \
    case 3: { constexpr int KP = 3; constexpr bool EXACT = true; __VA_ARGS__; break; } \
    case 4: { constexpr int KP = 4; constexpr bool EXACT = true; __VA_ARGS__; break; } \
    default: { constexpr int KP = 8; constexpr bool EXACT = false; __VA_ARGS__; break; } \
  }

KFB_API long kfb_cconv_bwd_ws(int T, int B, int D, int K) {
  if (T <= 0 || B <= 0 || D <= 0 || K <= 0) return 0;
  return (long)cconv::bwd_slabs(T, B, D, cconv::run_of(T, (long)ceil_div(D, cconv::BV) * B)) * (K + 1) * D;
}

KFB_API hipError_t kfb_cconv_fwd(int dtype, int vec, const void* x, long ldx, const void* x0,
                                 const float* w, const float* bias, const int* len, void* y,
                                 void* xT, int T, int B, int D, int K, int act, int reverse,
                                 hipStream_t stream) {
  cconv::Args a{};
  a.x = x; a.ldx = ldx; a.x0 = x0; a.w = w; a.bias = bias; a.len = len; a.y = y; a.xT = xT;
  a.T = T; a.B = B; a.D = D; a.K = K; a.act = act_of(act); a.reverse = reverse;
  if (cconv::bad(a)) return hipErrorInvalidValue;
  KFB_DISPATCH_DTYPE(dtype, E, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    KFB_CCONV_VEC(vec, 16 / sizeof(E), V, {
      const long lanes = (long)D / V * B;
      const int run = cconv::run_of(T, lanes), runs = ceil_div(T, run);
      if (runs > 65534 || lanes > (1l << 31)) return hipErrorInvalidValue;
      KFB_CCONV_TAPS(K, KP, EXACT, {
        hipLaunchKernelGGL((cconv::fwd_k<E, V, KIND, KP, EXACT>),
                           dim3(ceil_div(lanes, 256), runs + (xT && K > 1 ? 1 : 0)), dim3(256), 0,
                           stream, a, run, runs);
      });
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
  if (cconv::bad(a) || !ws) return hipErrorInvalidValue;
  const int run = cconv::run_of(T, (long)ceil_div(D, cconv::BV) * B), runs = ceil_div(T, run);
  const int S = cconv::bwd_slabs(T, B, D, run);
  KFB_DISPATCH_DTYPE(dtype, E, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    KFB_CCONV_VEC(vec, cconv::BV, V, {
      // the same slabs for any vector width
      KFB_CCONV_TAPS(K, KP, EXACT, {
        hipLaunchKernelGGL((cconv::bwd_k<E, V, KIND, KP, EXACT, cconv::BCX>),
                           dim3(ceil_div(D, cconv::BCX * V), S), dim3(256), 0, stream, a, run, runs);
      });
    });
  }));
  hipLaunchKernelGGL(cconv::param_grad_k, dim3(ceil_div((long)(K + 1) * D, 32)), dim3(256), 0,
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
    KFB_CCONV_VEC(vec, 16 / sizeof(E), V, {
      hipLaunchKernelGGL((cconv::step_k<E, V, KIND>), dim3(ceil_div((long)D / V * B, 256)), dim3(256),
                         0, stream, a, (E*)state);
    });
  }));
  return hipGetLastError();
}

KFB_API hipError_t kfb_mask_rows(int dtype, int vec, const void* x, long ldx, const int* len, void* y,
                                 int T, int B, int D, hipStream_t stream) {
  if (T <= 0 || B <= 0 || D <= 0 || !len) return hipErrorInvalidValue;
  const long rows = (long)T * B, wgs = (rows + 3) / 4;
  KFB_DISPATCH_DTYPE(dtype, E, KFB_CCONV_VEC(vec, 16 / sizeof(E), V, {
    hipLaunchKernelGGL((cconv::mask_rows_k<E, V>), dim3((unsigned)(wgs < 65536 ? wgs : 65536)), dim3(256), 0,
                       stream, (const E*)x, ldx, len, (E*)y, rows, B, D);
  }));
  return hipGetLastError();
}
