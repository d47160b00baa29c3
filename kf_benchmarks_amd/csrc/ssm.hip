// Selective state space scan over time-major sequences [T][B][D] with N states
// per channel, h [B][N][D] fp32:
//   dt = softplus(delta + bias)            (or delta + bias)
//   h_t = exp(dt A) h_{t-1} + dt x B_t
//   y   = (sum_n C_t h_t + skip x) silu(z)
// A [N][D], skip, bias [D] fp32; B, C [T][B][N] of x's type.  Position s of a
// sequence is time s, or len - 1 - s in reverse; rows at or past a sequence's
// length leave the state alone, give y = 0 and take no gradient.
//
// A workgroup owns 64 channels (lanes) of one sequence; its waves share the N
// states (NS each), so B and C are the same for a whole wave and come through
// scalar loads, from a copy in fp32 that is laid out per wave (prep_k).  A tile
// of TQ steps is staged in LDS as (dt, dt x), the waves walk it with their
// states in registers and leave their part of sum_n C h in LDS, and the tile's
// elementwise end is again one pass over (step, channel).
#include "act.h"

namespace kfb {
namespace ssm {

struct Args {
  const void *x, *delta, *z, *bm, *cm, *dy;
  long ldx, ldd, ldz, ldb, ldc, ldy;  // elements from row (t, b) to the next
  const float *A, *skip, *bias;
  const int* len;
  const float* h0;   // [B][N][D] or null: zero
  float* hT;         // [B][N][D] or null
  float* hs;         // [tiles][B][N][D], the state before each tile, or null
  float* bc;         // [B][W][Tp][2 NS], B then C of a wave's states
  void* y;
  // backward
  void *dx, *ddelta, *dz;
  const float* dhT;  // [B][N][D] or null
  float* dh0;        // [B][N][D] or null
  float* pbc;        // [D / 64][T * B][2 N]
  float* pch;        // [B][N + 2][D], dA | dskip | dbias of a sequence
  int T, B, D, N, W, Tp, softplus, reverse;
};

template <int V> struct Pack { float v[V]; };

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return a.len ? min(max(a.len[b], 0), a.T) : a.T;
}

// the row of position s
__device__ __forceinline__ long row_of(const Args& a, int b, int s, int len) {
  const int t = a.reverse && s < len ? len - 1 - s : s;
  return (long)t * a.B + b;
}

// B and C in fp32, per wave, zero past a sequence's end and past N (a row that
// must not count may hold NaN).
template <typename T, int NS>
__global__ void __launch_bounds__(256) prep_k(Args a) {
  const long total = (long)a.B * a.W * a.Tp * 2 * NS;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const int j = (int)(i % (2 * NS));
    long q = i / (2 * NS);
    const int s = (int)(q % a.Tp);
    q /= a.Tp;
    const int w = (int)(q % a.W), b = (int)(q / a.W);
    const int n = w * NS + (j % NS), len = seq_len(a, b);
    float v = 0.f;
    if (n < a.N && s < len) {
      const long row = row_of(a, b, s, len);
      v = j < NS ? to_f32(((const T*)a.bm)[row * a.ldb + n]) : to_f32(((const T*)a.cm)[row * a.ldc + n]);
    }
    a.bc[i] = v;
  }
}

template <typename T, int V, int NS, int TQ>
__global__ void __launch_bounds__(512) scan_fwd_k(Args a) {
  extern __shared__ float lds[];
  float2* du = (float2*)lds;           // [TQ][64]
  float* yp = lds + TQ * 64 * 2;       // [W][TQ][64]
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, d0 = blockIdx.x * 64, d = d0 + lane;
  const int len = seq_len(a, b), nt = a.W * 64;
  float A2[NS], h[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w * NS + i;
    const bool on = n < a.N && d < a.D;
    A2[i] = on ? a.A[(long)n * a.D + d] * LOG2E : 0.f;
    h[i] = on && a.h0 ? a.h0[((long)b * a.N + n) * a.D + d] : 0.f;
  }
  const float* __restrict__ bcw = a.bc + ((long)b * a.W + w) * a.Tp * 2 * NS;
  for (int s0 = 0; s0 < a.T; s0 += TQ) {
    for (int i = threadIdx.x; i < TQ * 64 / V; i += nt) {
      const int r = i / (64 / V), cl = i % (64 / V) * V, c = d0 + cl, s = s0 + r;
      float xv[V], dv[V];
#pragma unroll
      for (int k = 0; k < V; ++k) xv[k] = dv[k] = 0.f;
      if (s < len && c < a.D) {
        const long row = row_of(a, b, s, len);
        load_vec<T, V>((const T*)a.x + row * a.ldx + c, xv);
        load_vec<T, V>((const T*)a.delta + row * a.ldd + c, dv);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float raw = dv[k] + (a.bias ? a.bias[c + k] : 0.f);
          dv[k] = a.softplus ? softplusf(raw) : raw;
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) du[r * 64 + cl + k] = make_float2(dv[k], dv[k] * xv[k]);
    }
    if (a.hs && d < a.D) {
      float* hs = a.hs + ((long)(s0 / TQ) * a.B + b) * a.N * a.D + d;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (w * NS + i < a.N) hs[(long)(w * NS + i) * a.D] = h[i];
    }
    __syncthreads();
    const float* __restrict__ bct = bcw + (long)s0 * 2 * NS;
#pragma unroll 4
    for (int r = 0; r < TQ; ++r) {
      const float2 u = du[r * 64 + lane];
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        h[i] = fmaf(__builtin_amdgcn_exp2f(u.x * A2[i]), h[i], u.y * bct[r * 2 * NS + i]);
        v = fmaf(bct[r * 2 * NS + NS + i], h[i], v);
      }
      yp[(w * TQ + r) * 64 + lane] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TQ * 64 / V; i += nt) {
      const int r = i / (64 / V), cl = i % (64 / V) * V, c = d0 + cl, s = s0 + r;
      if (s >= a.T || c >= a.D) continue;
      const long row = row_of(a, b, s, len);
      float v[V], xv[V], zv[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = 0.f;
      if (s < len) {
        for (int q = 0; q < a.W; ++q) {
          const Pack<V> p = *(const Pack<V>*)(yp + (q * TQ + r) * 64 + cl);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] += p.v[k];
        }
        if (a.skip) {
          load_vec<T, V>((const T*)a.x + row * a.ldx + c, xv);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = fmaf(a.skip[c + k], xv[k], v[k]);
        }
        if (a.z) {
          load_vec<T, V>((const T*)a.z + row * a.ldz + c, zv);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] *= siluf(zv[k]);
        }
      }
      store_vec<T, V>((T*)a.y + row * a.D + c, v);
    }
  }
  if (a.hT && d < a.D)
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (w * NS + i < a.N) a.hT[((long)b * a.N + w * NS + i) * a.D + d] = h[i];
}

// Backward: the tiles from the last to the first, each one first forward again
// from its saved state (the TQ states and decays stay in registers), then back:
//   g = C e + a_{t+1} g_{t+1},  e = dy silu(z)
//   p = sum_n g B, q = sum_n g A a h_{t-1}:  dx = dt p + skip e, ddt = q + x p
//   dA = sum_t g dt a h_{t-1};  dB = sum_d g dt x;  dC = sum_d e h.
// dB and dC are summed over the wave's 64 channels here and over the channel
// blocks by bc_grad_k, dA, dskip and dbias over the sequences by
// param_grad_k: no atomics, the same sums on every run.
template <typename T, int V, int NS, int TQ>
__global__ void __launch_bounds__(512) scan_bwd_k(Args a) {
  extern __shared__ float lds[];
  float* sd = lds;                         // [TQ][64] dt
  float* sx = sd + TQ * 64;                // [TQ][64] dt x
  float* se = sx + TQ * 64;                // [TQ][64] e
  float* yp = se + TQ * 64;                // [W][TQ][64]
  float2* pq = (float2*)(yp + a.W * TQ * 64);  // [W][TQ][64]
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, d0 = blockIdx.x * 64, d = d0 + lane;
  const int len = seq_len(a, b), nt = a.W * 64;
  float A1[NS], carry[NS], dA[NS];
  constexpr int CH = V;  // channels of a thread in the elementwise passes
  float gskip[CH], gbias[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) gskip[k] = gbias[k] = 0.f;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w * NS + i;
    const bool on = n < a.N && d < a.D;
    A1[i] = on ? a.A[(long)n * a.D + d] : 0.f;
    carry[i] = on && a.dhT ? a.dhT[((long)b * a.N + n) * a.D + d] : 0.f;
    dA[i] = 0.f;
  }
  const float* __restrict__ bcw = a.bc + ((long)b * a.W + w) * a.Tp * 2 * NS;
  const int ntile = a.Tp / TQ;
  for (int tile = ntile - 1; tile >= 0; --tile) {
    const int s0 = tile * TQ;
    for (int i = threadIdx.x; i < TQ * 64 / V; i += nt) {
      const int r = i / (64 / V), cl = i % (64 / V) * V, c = d0 + cl, s = s0 + r;
      float xv[V], dv[V], ev[V], zv[V];
#pragma unroll
      for (int k = 0; k < V; ++k) xv[k] = dv[k] = ev[k] = 0.f;
      if (s < len && c < a.D) {
        const long row = row_of(a, b, s, len);
        load_vec<T, V>((const T*)a.x + row * a.ldx + c, xv);
        load_vec<T, V>((const T*)a.delta + row * a.ldd + c, dv);
        load_vec<T, V>((const T*)a.dy + row * a.ldy + c, ev);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float raw = dv[k] + (a.bias ? a.bias[c + k] : 0.f);
          dv[k] = a.softplus ? softplusf(raw) : raw;
        }
        if (a.z) {
          load_vec<T, V>((const T*)a.z + row * a.ldz + c, zv);
#pragma unroll
          for (int k = 0; k < V; ++k) ev[k] *= siluf(zv[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        sd[r * 64 + cl + k] = dv[k];
        sx[r * 64 + cl + k] = dv[k] * xv[k];
        se[r * 64 + cl + k] = ev[k];
      }
    }
    float hb[NS], H[TQ][NS], dec[TQ][NS];
    const float* hs = a.hs + ((long)tile * a.B + b) * a.N * a.D + d;
#pragma unroll
    for (int i = 0; i < NS; ++i)
      hb[i] = w * NS + i < a.N && d < a.D ? hs[(long)(w * NS + i) * a.D] : 0.f;
    __syncthreads();
    const float* __restrict__ bct = bcw + (long)s0 * 2 * NS;
#pragma unroll
    for (int r = 0; r < TQ; ++r) {
      const float dt = sd[r * 64 + lane], dtx = sx[r * 64 + lane];
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        dec[r][i] = __builtin_amdgcn_exp2f(dt * (A1[i] * LOG2E));
        H[r][i] = fmaf(dec[r][i], r ? H[r - 1][i] : hb[i], dtx * bct[r * 2 * NS + i]);
        v = fmaf(bct[r * 2 * NS + NS + i], H[r][i], v);
      }
      if (a.z) yp[(w * TQ + r) * 64 + lane] = v;
    }
    float dAt[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) dAt[i] = 0.f;
#pragma unroll
    for (int r = TQ - 1; r >= 0; --r) {
      const float dt = sd[r * 64 + lane], dtx = sx[r * 64 + lane], e = se[r * 64 + lane];
      float p = 0.f, q = 0.f, red[2 * NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const float g = fmaf(bct[r * 2 * NS + NS + i], e, carry[i]);
        p = fmaf(g, bct[r * 2 * NS + i], p);
        red[i] = g * dtx;
        red[NS + i] = e * H[r][i];
        carry[i] = g * dec[r][i];
        const float k = carry[i] * (r ? H[r - 1][i] : hb[i]);
        q = fmaf(k, A1[i], q);
        dAt[i] = fmaf(k, dt, dAt[i]);
      }
      pq[(w * TQ + r) * 64 + lane] = make_float2(p, q);
      const int s = s0 + r;
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) red[i] = wave_sum(red[i]);
      if (s < a.T && lane == 0) {
        float* out = a.pbc + ((long)blockIdx.x * a.T * a.B + row_of(a, b, s, len)) * 2 * a.N;
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (w * NS + i < a.N) {
            out[w * NS + i] = red[i];
            out[a.N + w * NS + i] = red[NS + i];
          }
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) dA[i] += dAt[i];
    __syncthreads();
    for (int i = threadIdx.x; i < TQ * 64 / V; i += nt) {
      const int r = i / (64 / V), cl = i % (64 / V) * V, c = d0 + cl, s = s0 + r;
      if (s >= a.T || c >= a.D) continue;
      const long row = row_of(a, b, s, len);
      float ox[V], od[V], oz[V];
#pragma unroll
      for (int k = 0; k < V; ++k) ox[k] = od[k] = oz[k] = 0.f;
      if (s < len) {
        float xv[V], dv[V], zv[V], gv[V];
        load_vec<T, V>((const T*)a.x + row * a.ldx + c, xv);
        load_vec<T, V>((const T*)a.delta + row * a.ldd + c, dv);
        if (a.z) {
          load_vec<T, V>((const T*)a.z + row * a.ldz + c, zv);
          load_vec<T, V>((const T*)a.dy + row * a.ldy + c, gv);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float p = 0.f, q = 0.f, v = 0.f;
          for (int u = 0; u < a.W; ++u) {
            const float2 t = pq[(u * TQ + r) * 64 + cl + k];
            p += t.x;
            q += t.y;
            if (a.z) v += yp[(u * TQ + r) * 64 + cl + k];
          }
          const float sk = a.skip ? a.skip[c + k] : 0.f;
          const float e = se[r * 64 + cl + k], dt = sd[r * 64 + cl + k];
          ox[k] = fmaf(dt, p, sk * e);
          float dd = fmaf(xv[k], p, q);
          if (a.softplus) dd *= sigmoidf(dv[k] + (a.bias ? a.bias[c + k] : 0.f));
          od[k] = dd;
          if (a.z) oz[k] = gv[k] * fmaf(sk, xv[k], v) * dsiluf(zv[k]);
          gskip[k] = fmaf(e, xv[k], gskip[k]);
          gbias[k] += dd;
        }
      }
      store_vec<T, V>((T*)a.dx + row * a.D + c, ox);
      store_vec<T, V>((T*)a.ddelta + row * a.D + c, od);
      if (a.z) store_vec<T, V>((T*)a.dz + row * a.D + c, oz);
    }
    __syncthreads();
  }
  float* pch = a.pch + (long)b * (a.N + 2) * a.D;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w * NS + i;
    if (n < a.N && d < a.D) {
      pch[(long)n * a.D + d] = dA[i];
      if (a.dh0) a.dh0[((long)b * a.N + n) * a.D + d] = carry[i];
    }
  }
  // dskip, dbias: thread i holds V channels (i % (64 / V)) of some rows
  const int ncol = 64 / V, nrow = nt / ncol;
  float* rs = lds;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    rs[(threadIdx.x / ncol) * 64 + threadIdx.x % ncol * V + k] = gskip[k];
    rs[(nrow + threadIdx.x / ncol) * 64 + threadIdx.x % ncol * V + k] = gbias[k];
  }
  __syncthreads();
  if (w == 0 && d < a.D) {
    float u = 0.f, v = 0.f;
    for (int r = 0; r < nrow; ++r) {
      u += rs[r * 64 + lane];
      v += rs[(nrow + r) * 64 + lane];
    }
    pch[(long)a.N * a.D + d] = u;
    pch[(long)(a.N + 1) * a.D + d] = v;
  }
}

// dB, dC [T * B][N]: the sum over the channel blocks of pbc [nblk][rows][2 N]
template <typename T>
__global__ void __launch_bounds__(256)
bc_grad_k(const float* __restrict__ p, int nblk, long rows, int N, T* __restrict__ db,
          T* __restrict__ dc) {
  const long total = rows * 2 * N;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    float s = 0.f;
    for (int k = 0; k < nblk; ++k) s += p[k * total + i];
    const long row = i / (2 * N);
    const int n = (int)(i % (2 * N));
    (n < N ? db : dc)[row * N + (n < N ? n : n - N)] = from_f32<T>(s);
  }
}

// dA [N][D], dskip, dbias [D]: the sum over the slabs of pch [S][N + 2][D]
__global__ void __launch_bounds__(256)
param_grad_k(const float* __restrict__ p, int S, int N, int D, float* dA, float* dskip,
             float* dbias, int acc_a, int acc_s, int acc_b) {
  const long total = (long)(N + 2) * D;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float s = 0.f;
  for (int k = 0; k < S; ++k) s += p[k * total + i];
  const int n = (int)(i / D);
  float* out = n < N ? dA : n == N ? dskip : dbias;
  const int acc = n < N ? acc_a : n == N ? acc_s : acc_b;
  if (!out) return;
  out += n < N ? i : i % D;
  *out = acc ? *out + s : s;
}

// One token: state [B][N][D] in place.  64 channels x 4 waves, wave w the
// states w, w + 4, ...
template <typename T>
__global__ void __launch_bounds__(256) step_k(Args a, float* __restrict__ state) {
  __shared__ float yp[4][64];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int b = blockIdx.y, d = blockIdx.x * 64 + lane;
  const bool on = d < a.D;
  float x = 0.f, dt = 0.f, v = 0.f;
  if (on) {
    x = to_f32(((const T*)a.x)[b * a.ldx + d]);
    dt = to_f32(((const T*)a.delta)[b * a.ldd + d]) + (a.bias ? a.bias[d] : 0.f);
    if (a.softplus) dt = softplusf(dt);
    float* h = state + (long)b * a.N * a.D + d;
#pragma unroll 4
    for (int n = w; n < a.N; n += 4) {
      const float B = to_f32(((const T*)a.bm)[b * a.ldb + n]);
      const float C = to_f32(((const T*)a.cm)[b * a.ldc + n]);
      const float e = __builtin_amdgcn_exp2f(dt * (a.A[(long)n * a.D + d] * LOG2E));
      const float u = fmaf(e, h[(long)n * a.D], dt * x * B);
      h[(long)n * a.D] = u;
      v = fmaf(C, u, v);
    }
  }
  yp[w][lane] = v;
  __syncthreads();
  if (w == 0 && on) {
    v = yp[0][lane] + yp[1][lane] + yp[2][lane] + yp[3][lane];
    if (a.skip) v = fmaf(a.skip[d], x, v);
    if (a.z) v *= siluf(to_f32(((const T*)a.z)[b * a.ldz + d]));
    ((T*)a.y)[(long)b * a.D + d] = from_f32<T>(v);
  }
}

struct Plan {
  int ns, tq, W, Tp, tiles;
};

inline Plan plan(int T, int N) {
  Plan p;
  p.ns = N <= 32 ? 4 : 8;
  p.tq = N <= 32 ? 16 : 8;
  p.W = ceil_div(N, p.ns);
  p.tiles = ceil_div(T, p.tq);
  p.Tp = p.tiles * p.tq;
  return p;
}

inline bool bad(const Args& a) {
  return a.T <= 0 || a.B <= 0 || a.D <= 0 || a.N <= 0 || a.N > 64 || a.B > 65535;
}

}  // namespace ssm
}  // namespace kfb

using namespace kfb;

#define KFB_SSM_CONFIG(ns, NS, TQ, ...)              \
  if (ns == 4) { constexpr int NS = 4, TQ = 16; __VA_ARGS__; } \
  else { constexpr int NS = 8, TQ = 8; __VA_ARGS__; }

KFB_API int kfb_ssm_max_states() { return 64; }

// Floats of: the fp32 copy of B and C (what = 0), the saved states of a
// training forward (1), the backward's workspace (2).
KFB_API long kfb_ssm_floats(int what, int T, int B, int D, int N) {
  const ssm::Plan p = ssm::plan(T, N);
  switch (what) {
    case 0: return (long)B * p.W * p.Tp * 2 * p.ns;
    case 1: return (long)p.tiles * B * N * D;
    case 2: return (long)ceil_div(D, 64) * T * B * 2 * N + (long)B * (N + 2) * D;
    default: return -1;
  }
}

KFB_API hipError_t kfb_ssm_scan_fwd(int dtype, int V, const void* x, long ldx, const void* delta,
                                    long ldd, const void* z, long ldz, const void* bm, long ldb,
                                    const void* cm, long ldc, const float* A, const float* skip,
                                    const float* bias, const int* len, const float* h0, float* hT,
                                    float* hs, float* bc, void* y, int T, int B, int D, int N,
                                    int softplus, int reverse, hipStream_t stream) {
  const ssm::Plan p = ssm::plan(T, N > 0 ? N : 1);
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.bm = bm; a.cm = cm;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldb = ldb; a.ldc = ldc;
  a.A = A; a.skip = skip; a.bias = bias; a.len = len; a.h0 = h0; a.hT = hT; a.hs = hs; a.bc = bc;
  a.y = y;
  a.T = T; a.B = B; a.D = D; a.N = N; a.W = p.W; a.Tp = p.Tp;
  a.softplus = softplus; a.reverse = reverse;
  if (ssm::bad(a) || (V != 1 && V != 4)) return hipErrorInvalidValue;
  const dim3 grid(ceil_div(D, 64), B);
  KFB_DISPATCH_DTYPE(dtype, E, {
    KFB_SSM_CONFIG(p.ns, NS, TQ, {
      const long total = (long)B * p.W * p.Tp * 2 * NS;
      hipLaunchKernelGGL((ssm::prep_k<E, NS>), dim3(ceil_div(total < (1l << 22) ? total : (1l << 22), 256)),
                         dim3(256), 0, stream, a);
      const size_t shm = (size_t)(2 + p.W) * TQ * 64 * sizeof(float);
      if (V == 4)
        hipLaunchKernelGGL((ssm::scan_fwd_k<E, 4, NS, TQ>), grid, dim3(p.W * 64), shm, stream, a);
      else
        hipLaunchKernelGGL((ssm::scan_fwd_k<E, 1, NS, TQ>), grid, dim3(p.W * 64), shm, stream, a);
    });
  });
  return hipGetLastError();
}

KFB_API hipError_t kfb_ssm_scan_bwd(int dtype, int V, const void* dy, long ldy, const void* x,
                                    long ldx, const void* delta, long ldd, const void* z, long ldz,
                                    const float* A, const float* skip, const float* bias,
                                    const int* len, const float* hs, float* bc, const float* dhT,
                                    float* dh0, void* dx, void* ddelta, void* dz, void* db,
                                    void* dc, float* dA, float* dskip, float* dbias, int acc_a,
                                    int acc_skip, int acc_bias, float* ws, int T, int B, int D,
                                    int N, int softplus, int reverse, hipStream_t stream) {
  const ssm::Plan p = ssm::plan(T, N > 0 ? N : 1);
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.dy = dy;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldy = ldy;
  a.A = A; a.skip = skip; a.bias = bias; a.len = len; a.hs = const_cast<float*>(hs); a.bc = bc;
  a.dhT = dhT; a.dh0 = dh0; a.dx = dx; a.ddelta = ddelta; a.dz = dz;
  a.T = T; a.B = B; a.D = D; a.N = N; a.W = p.W; a.Tp = p.Tp;
  a.softplus = softplus; a.reverse = reverse;
  if (ssm::bad(a) || (V != 1 && V != 4) || !ws || !hs) return hipErrorInvalidValue;
  const int nblk = ceil_div(D, 64);
  const long rows = (long)T * B;
  a.pbc = ws;
  a.pch = ws + (long)nblk * rows * 2 * N;
  const dim3 grid(nblk, B);
  KFB_DISPATCH_DTYPE(dtype, E, {
    KFB_SSM_CONFIG(p.ns, NS, TQ, {
      size_t shm = (size_t)(3 + 3 * p.W) * TQ * 64 * sizeof(float);
      if (shm < (size_t)2 * 64 * p.W * V * sizeof(float)) shm = (size_t)2 * 64 * p.W * V * sizeof(float);
      if (V == 4)
        hipLaunchKernelGGL((ssm::scan_bwd_k<E, 4, NS, TQ>), grid, dim3(p.W * 64), shm, stream, a);
      else
        hipLaunchKernelGGL((ssm::scan_bwd_k<E, 1, NS, TQ>), grid, dim3(p.W * 64), shm, stream, a);
    });
    hipLaunchKernelGGL((ssm::bc_grad_k<E>), dim3(ceil_div(rows * 2 * N < (1l << 22) ? rows * 2 * N : (1l << 22), 256)),
                       dim3(256), 0, stream, a.pbc, nblk, rows, N, (E*)db, (E*)dc);
  });
  hipLaunchKernelGGL(ssm::param_grad_k, dim3(ceil_div((long)(N + 2) * D, 256)), dim3(256), 0, stream,
                     a.pch, B, N, D, dA, dskip, dbias, acc_a, acc_skip, acc_bias);
  return hipGetLastError();
}

KFB_API hipError_t kfb_ssm_step(int dtype, const void* x, long ldx, const void* delta, long ldd,
                                const void* z, long ldz, const void* bm, long ldb, const void* cm,
                                long ldc, const float* A, const float* skip, const float* bias,
                                float* state, void* y, int B, int D, int N, int softplus,
                                hipStream_t stream) {
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.bm = bm; a.cm = cm;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldb = ldb; a.ldc = ldc;
  a.A = A; a.skip = skip; a.bias = bias; a.y = y;
  a.T = 1; a.B = B; a.D = D; a.N = N; a.softplus = softplus;
  if (ssm::bad(a)) return hipErrorInvalidValue;
  KFB_DISPATCH_DTYPE(dtype, E, {
    hipLaunchKernelGGL((ssm::step_k<E>), dim3(ceil_div(D, 64), B), dim3(256), 0, stream, a, state);
  });
  return hipGetLastError();
}
