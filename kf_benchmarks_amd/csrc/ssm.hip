// Selective state space scan over time-major sequences [T][B][D] with N states
// per channel, h [B][N][D] fp32:
//   dt = softplus(delta + bias)            (or delta + bias)
//   A = -exp(A)                            (with log_a, or as given)
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
// elementwise end is again one pass over (step, channel).  The next tile's rows are
// loaded while a tile is walked.
//
// Bound by the vector units: an exponential (8 cycles a wave) and four fused
// operations (4 cycles each) per state, 24 cycles, and about 60 operations a value
// around it; the bytes take a quarter to a half of that.  By its counters the walk of 874 x
// 16 x 1600 bf16 values with 16 states (115 us) keeps them busy for 83% of its time.
// Where B D / 64 workgroups do not fill the card, a sequence is cut into chunks: a first
// launch (ENDS, 73 us there, 72% busy) walks every chunk but the last from a zero state,
// and because the decays of a chunk multiply to exp(A sum dt), the state before a chunk
// follows from the earlier chunks' (end, sum dt) alone.
//
// Zeros that stand for nothing are selected, not multiplied by: a missing skip, the states
// that a wave does not have, the rows behind a sequence's end.  An infinite input then
// gives infinities where the formulas do, and in nothing else.
#include "act.h"
#include "raw.h"

#include <type_traits>

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
  float* pch;        // [B * nchunk][N + 2][D], dA | dskip | dbias of a chunk
  // chunks of tpc tiles: end state (backward: gradient before the chunk) from
  // zero [nchunk][B][N][D], sum of dt [nchunk][B][D]
  float *ends, *sums;
  int nchunk, tpc;
  int T, B, D, N, W, Tp, softplus, reverse, log_a;
  FastDiv by2n;
};

// The state from which wave w reads the saved states: its first one.  There are at least
// four waves, so some may have no state; these loads have no branch, so such a wave reads
// the last state, and what it reads is dropped.
__host__ __device__ inline int base_state(int w, int NS, int N) { return w * NS < N ? w * NS : N - 1; }

// Where state n of sequence b, channel d stands in [B][N][D].
__host__ __device__ inline long state_at(int b, int n, int N, int D, int d) {
  return ((long)b * N + n) * D + d;
}

// From a wave's base to its state i, of ns; for a state that it does not have, to the base.
__host__ __device__ inline long saved_at(int i, int ns, int D) { return i < ns ? (long)i * D : 0; }

// B and C as constant memory: uniform addresses become scalar loads
typedef const __attribute__((address_space(4))) float cfloat;

// B and C of UR steps for NS states, in scalar registers.  load() is given an
// address that the compiler does not know to be an earlier one: the loads are
// neither merged with others nor moved, so that a group is in flight while the one
// before it is worked on and no more than two are alive (64 of the 102 registers).
template <int NS, int UR> struct Group {
  float v[UR * 2 * NS];
  __device__ __forceinline__ void load(const float* p) {
    uintptr_t q = (uintptr_t)p;
    asm volatile("" : "+s"(q));
    cfloat* c = (cfloat*)q;
#pragma unroll
    for (int i = 0; i < UR * 2 * NS; ++i) v[i] = c[i];
    __builtin_amdgcn_sched_barrier(0x7ff);  // everything but scalar loads may pass
  }
  __device__ __forceinline__ float B(int k, int i) const { return v[k * 2 * NS + i]; }
  __device__ __forceinline__ float C(int k, int i) const { return v[k * 2 * NS + NS + i]; }
};

constexpr int BC_PAD = 64;  // floats behind bc: a group is fetched ahead

__device__ __forceinline__ float rate(const Args& a, long i) {
  return a.log_a ? -expf(a.A[i]) : a.A[i];
}

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return a.len ? min(max(a.len[b], 0), a.T) : a.T;
}

// the time of position s
__device__ __forceinline__ long time_of(const Args& a, int s, int len) {
  return a.reverse && s < len ? len - 1 - s : s;
}

__device__ __forceinline__ long row_of(const Args& a, int b, int s, int len) {
  return time_of(a, s, len) * a.B + b;
}

// (5 us for 874 x 16 rows of 16 states.)
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

// A thread's part of the elementwise passes over a tile: IT vectors of V channels,
// the same channels in each (the thread count is a multiple of 64 / V).
template <typename T, int V, int IT, int TQ> struct Part {
  int r[IT];  // its steps of the tile (TQ: none)
  int cl, c;  // its first channel: in the block, in the row
  bool on;

  __device__ __forceinline__ Part(const Args& a, int d0) {
    cl = threadIdx.x % (64 / V) * V;
    c = d0 + cl;
    on = c < a.D;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int q = (threadIdx.x + i * a.W * 64) / (64 / V);
      r[i] = q < TQ ? q : TQ;
    }
  }
};

// One sequence's rows of a [T][B] tensor: position s at p + s * step.  Loads are
// unconditional: a position or channel outside reads the last one inside (of an
// empty sequence: row 0), and what it gives is not used.
template <typename T, int V> struct Line {
  const T* p;
  long step;
  int last;

  __device__ __forceinline__ Line(const Args& a, const void* t, long ld, int b, int c, int len) {
    step = (long)a.B * ld;
    p = (const T*)t + (long)b * ld + (c < a.D ? c : a.D - V);
    last = len > 0 ? len - 1 : 0;
    if (a.reverse && len > 0) {
      p += last * step;
      step = -step;
    }
  }
  template <int IT> __device__ __forceinline__ void load(const int (&r)[IT], int s0, Raw<T, V> (&v)[IT]) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) v[i].load(p + min(s0 + r[i], last) * step);
  }
};

template <int V>
__device__ __forceinline__ void params(const float* p, int c, bool on, float (&v)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = on && p ? p[c + k] : 0.f;
}

// V neighbouring floats of LDS at once (V = 4: 16-byte aligned)
template <int V> struct alignas(4 * V) Quad {
  float v[V];
};
template <int V> __device__ __forceinline__ Quad<V> get(const float* p) { return *(const Quad<V>*)p; }
template <int V> __device__ __forceinline__ void put(float* p, const Quad<V>& q) { *(Quad<V>*)p = q; }

__device__ __forceinline__ float step_size(float raw, bool softplus) {
  const float v = softplusf(raw);  // (a select, not a branch: the flag is uniform)
  return softplus ? v : raw;
}

// h over ``n`` chunks j = from, from + by, ...: h = exp(A sum dt_j) h + end_j,
// eight chunks' values in flight.  The decays of a chunk may multiply to zero where no single one
// is zero, and zero times an infinite h is NaN: 2^-149 in its place leaves infinities as they are
// and at most 2^-21 of the largest finite h.
template <int NS>
__device__ __forceinline__ void join(const Args& a, int b, int dc, long bnd, long bn, int ns,
                                     const float (&A2)[NS], int from, int by, int n, float (&h)[NS]) {
  constexpr int Q = NS > 4 ? 4 : 8;
  for (int j0 = 0; j0 < n; j0 += Q) {
    float sum[Q], end[Q][NS];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = from + by * min(j0 + q, n - 1);
      sum[q] = a.sums[((long)j * a.B + b) * a.D + dc];
#pragma unroll
      for (int i = 0; i < NS; ++i) end[q][i] = i < ns ? a.ends[j * bn + bnd + (long)i * a.D] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (j0 + q < n)
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (i < ns) h[i] = fmaf(fmaxf(__builtin_amdgcn_exp2f(sum[q] * A2[i]), 0x1p-149f), h[i], end[q][i]);
  }
}

// v, or 0 from position len on (a mask takes one scalar register, a select two)
__device__ __forceinline__ float zero_from(float v, int s, int len) {
  return __builtin_bit_cast(float, __builtin_bit_cast(int, v) & (s - len) >> 31);
}

// The order in a tile is for the memory counter, which counts loads and stores in
// turn: the next tile's rows are fetched before the walk and used before y is stored,
// so that no wait for a load waits for a store just issued.
// ENDS: only the state after each chunk, from zero, and the chunk's sum of dt.
// PART: not every wave has NS states; those that it does not have stay zero by selection
// (zero times an infinite input or gradient is not).  (ENDS stores none of them.)
template <typename T, int V, int IT, int NS, int TQ, bool ENDS, bool PART>
__global__ void __launch_bounds__(512) scan_fwd_k(Args a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  constexpr int UR = 16 / NS < 4 ? 16 / NS : 4;  // steps of a group
  float *sd = lds, *sx = lds + TQ * 64;  // [TQ][64] dt, dt x
  float* yp = lds + TQ * 64 * 2;         // [W][TQ][64]
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, d0 = blockIdx.x * 64, d = d0 + lane, chunk = blockIdx.z;
  const int len = seq_len(a, b), ns = min(max(a.N - w * NS, 0), NS);  // states of this wave
  const bool ok = d < a.D;
  const int dc = ok ? d : a.D - 1;
  const long bnd = state_at(b, w * NS, a.N, a.D, dc), bn = (long)a.B * a.N * a.D;
  float A2[NS], h[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A2[i] = i < ns ? rate(a, (long)(w * NS + i) * a.D + dc) * LOG2E : 0.f;
    h[i] = i < ns && a.h0 && !ENDS ? a.h0[bnd + (long)i * a.D] : 0.f;
  }
  if constexpr (!ENDS) join<NS>(a, b, dc, bnd, bn, ns, A2, 0, 1, chunk, h);
  const float* bcw = a.bc + ((long)b * a.W + w) * a.Tp * 2 * NS;
  const Part<T, V, IT, TQ> me(a, d0);
  const Line<T, V> lx(a, a.x, a.ldx, b, me.c, len), ld(a, a.delta, a.ldd, b, me.c, len);
  const bool gate = !ENDS && a.z;
  const Line<T, V> lz(a, gate ? a.z : a.x, gate ? a.ldz : a.ldx, b, me.c, len);
  float bias[V], skip[V];
  params<V>(a.bias, me.c, me.on, bias);
  params<V>(a.skip, me.c, me.on, skip);
  Raw<T, V> nx[IT], nd[IT], nz[IT], cx[IT], cz[IT];
  const int s_end = min((chunk + 1) * a.tpc * TQ, a.Tp);
  auto fetch = [&](int s0) {
    lx.load(me.r, s0, nx);
    ld.load(me.r, s0, nd);
    if (!ENDS) lz.load(me.r, s0, nz);
  };
  auto stage = [&](int s0) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (me.r[i] < TQ) {
        const bool in = me.on && s0 + me.r[i] < len;
        const int at = me.r[i] * 64 + me.cl;
        Quad<V> qd, qx;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float dt = step_size(nd[i][k] + bias[k], a.softplus);
          qd.v[k] = in ? dt : 0.f;
          qx.v[k] = in ? dt * nx[i][k] : 0.f;
        }
        put(sd + at, qd);
        put(sx + at, qx);
      }
  };
  const long ystep = (long)a.B * a.D, ybase = (long)b * a.D + me.c;
  float sum_dt = 0.f;
  int s0 = chunk * a.tpc * TQ;
  Group<NS, UR> next;
  next.load(bcw + (long)s0 * 2 * NS);
  fetch(s0);
  stage(s0);
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    cx[i] = nx[i];
    cz[i] = nz[i];
  }
  __syncthreads();
  for (; s0 < s_end; s0 += TQ) {
    const bool more = s0 + TQ < s_end;
    fetch(more ? s0 + TQ : s0);
    if (!ENDS && a.hs && ok) {
      float* hs = a.hs + (long)(s0 / TQ) * bn + bnd;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (i < ns) hs[(long)i * a.D] = h[i];
    }
#pragma unroll
    for (int r0 = 0; r0 < TQ; r0 += UR) {
      const Group<NS, UR> bc = next;
      next.load(bcw + (long)(s0 + r0 + UR) * 2 * NS);
#pragma unroll
      for (int k = 0; k < UR; ++k) {
        const float2 u = make_float2(sd[(r0 + k) * 64 + lane], sx[(r0 + k) * 64 + lane]);
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float in = u.y * bc.B(k, i);
          h[i] = fmaf(__builtin_amdgcn_exp2f(u.x * A2[i]), h[i], PART && i >= ns ? 0.f : in);
          if (!ENDS) v = fmaf(bc.C(k, i), h[i], v);
        }
        if constexpr (ENDS) sum_dt += u.x;
        else yp[(w * TQ + r0 + k) * 64 + lane] = v;
      }
    }
    __syncthreads();
    if (more) stage(s0 + TQ);
    if constexpr (!ENDS) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = me.r[i], s = s0 + r;
        if (r < TQ) {
          float v[V];
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = a.skip ? skip[k] * cx[i][k] : 0.f;  // (not 0 * inf)
          const float* part = yp + r * 64 + me.cl;
#pragma unroll
          for (int q = 0; q < 4; ++q) {  // W >= 4
            const Quad<V> t = get<V>(part + q * TQ * 64);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += t.v[k];
          }
          for (int q = 4; q < a.W; ++q) {
            const Quad<V> t = get<V>(part + q * TQ * 64);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += t.v[k];
          }
          if (gate)
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] *= siluf(cz[i][k]);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = s < len ? v[k] : 0.f;
          if (s < a.T && me.on) store_vec<T, V>((T*)a.y + time_of(a, s, len) * ystep + ybase, v);
        }
        cx[i] = nx[i];
        cz[i] = nz[i];
      }
    }
    __syncthreads();
  }
  if constexpr (ENDS) {
    if (ok)
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (i < ns) a.ends[chunk * bn + bnd + (long)i * a.D] = h[i];
    if (w == 0 && ok) a.sums[((long)chunk * a.B + b) * a.D + d] = sum_dt;
  } else if (a.hT && chunk == a.nchunk - 1 && ok) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (i < ns) a.hT[bnd + (long)i * a.D] = h[i];
  }
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL,
                                                               0xf, 0xf, true));
}

// Sums over the wave's lanes of M = 2, 4, 8 or 16 values at once, halving the
// number of registers where it halves the lanes: 18 instructions for 8 values
// instead of 48.  Lane l ends up with the sum of value lane_value<M>(l).
template <int M> __device__ __forceinline__ float lanes_sum(float (&v)[M], int lane) {
  static_assert(M == 2 || M == 4 || M == 8 || M == 16, "2, 4, 8 or 16 values");
#pragma unroll
  for (int i = 0; i < M / 2; ++i) {  // lanes 0-31 | 32-63
    const auto q = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v[i]),
                                                    __builtin_bit_cast(unsigned, v[i + M / 2]), false, false);
    const unsigned lo = q[0], hi = q[1];  // (a bit_cast of q[1] itself takes element 0)
    v[i] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
  }
  constexpr int R = M / 4 > 0 ? M / 4 : 1;
#pragma unroll
  for (int i = 0; i < R; ++i) {  // even | odd rows of 16 (M = 2: the sum is left in the even ones)
    const auto q = __builtin_amdgcn_permlane16_swap(
        __builtin_bit_cast(unsigned, v[i]), M == 2 ? 0u : __builtin_bit_cast(unsigned, v[i + R < M ? i + R : 0]),
        false, false);
    const unsigned lo = q[0], hi = q[1];  // (a bit_cast of q[1] itself takes element 0)
    v[i] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
  }
  const bool b3 = lane & 8, b2 = lane & 4;
  if constexpr (M >= 8) {
#pragma unroll
    for (int i = 0; i < M / 8; ++i)  // lane ^ 8: row_ror:8
      v[i] = (b3 ? v[2 * i + 1] : v[2 * i]) + dpp<0x128>(b3 ? v[2 * i] : v[2 * i + 1]);
  } else {
    v[0] += dpp<0x128>(v[0]);
  }
  float s;
  if constexpr (M == 16) s = (b2 ? v[1] : v[0]) + dpp<0x141>(b2 ? v[0] : v[1]);  // lane ^ 7: row_half_mirror
  else s = v[0] + dpp<0x141>(v[0]);
  s += dpp<0xB1>(s);  // lane ^ 1
  s += dpp<0x4E>(s);  // lane ^ 2
  return s;
}

template <int M> __device__ __forceinline__ int lane_value(int l) {
  const int b2 = l >> 2 & 1, b3 = l >> 3 & 1, row = l >> 4;
  switch (M) {
    case 2: return row >> 1;
    case 4: return (row & 1) + 2 * (row >> 1);
    case 8: return b3 + 2 * (row & 1) + 4 * (row >> 1);
    default: return b3 + 2 * b2 + 4 * (row & 1) + 8 * (row >> 1);
  }
}

// Backward.  The tiles of a chunk from the last to the first, each one first
// forward again from its saved state (the TQ states and decays stay in registers),
// then back:
//   g = C e + a_{t+1} g_{t+1},  e = dy silu(z)
//   p = sum_n g B, q = sum_n g A a h_{t-1}:  dx = dt p + skip e, ddt = q + x p
//   dA = sum_t g dt a h_{t-1};  dB = sum_d g dt x;  dC = sum_d e h.
// dB and dC are summed over the wave's 64 channels here and over the channel
// blocks by bc_grad_k, dA, dskip and dbias over the chunks by param_grad_k: no
// atomics, the same sums on every run.  Bound by the vector units too: 70
// instructions a step of 4 states (19 of them the sums over lanes), 1840 a wave and tile,
// at two waves a SIMD (H and dec take 128 registers): 874 x 16 x 1600 values take
// 519 us, the vector units busy for 52% of it.  Tiles of 8 steps (three waves a SIMD), decays computed again instead of
// kept, and two states a wave were no faster (550 to 890 us).
// ENDS: only the gradient before each chunk, from zero behind it, and sum dt.
// PART: as in scan_fwd_k (and all tiles in the loop for the last ones: fewer kernels).
template <typename T, int V, int IT, int NS, int TQ, bool ENDS, bool PART>
__global__ void __launch_bounds__(512) scan_bwd_k(Args a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int WN = a.W * NS;
  constexpr int UR = 8 / NS < 4 ? 8 / NS : 4;
  float *sd = lds, *sx = lds + TQ * 64, *se = lds + TQ * 64 * 2;  // [TQ][64] dt, dt x, e
  float* sbc = se + TQ * 64;                                      // [TQ][2 WN] and a lane's rest
  float* pp = sbc + TQ * 2 * WN + 64;                             // [W][TQ][64]: p, q, sum_n C h
  float *pq = pp + a.W * TQ * 64, *yp = pq + a.W * TQ * 64;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = blockIdx.y, d0 = blockIdx.x * 64, d = d0 + lane;
  const int chunk = ENDS ? blockIdx.z + 1 : blockIdx.z;
  const int len = seq_len(a, b), nt = a.W * 64, ns = min(max(a.N - w * NS, 0), NS);
  const bool ok = d < a.D;
  const int dc = ok ? d : a.D - 1;
  const long bnd = state_at(b, w * NS, a.N, a.D, dc), bn = (long)a.B * a.N * a.D;
  const long saved = state_at(b, base_state(w, NS, a.N), a.N, a.D, dc);
  float A1[NS], carry[NS], dA[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A1[i] = i < ns && ok ? rate(a, (long)(w * NS + i) * a.D + dc) : 0.f;
    carry[i] = i < ns && ok && a.dhT && !ENDS ? a.dhT[bnd + (long)i * a.D] : 0.f;
    dA[i] = 0.f;
  }
  if constexpr (!ENDS) {
    float A2[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) A2[i] = A1[i] * LOG2E;
    join<NS>(a, b, dc, bnd, bn, ok ? ns : 0, A2, a.nchunk - 1, -1, a.nchunk - 1 - chunk, carry);
  }
  const float* bcw = a.bc + ((long)b * a.W + w) * a.Tp * 2 * NS;
  const Part<T, V, IT, TQ> me(a, d0);
  const bool gate = a.z;
  const Line<T, V> lx(a, a.x, a.ldx, b, me.c, len), ld(a, a.delta, a.ldd, b, me.c, len),
      ly(a, a.dy, a.ldy, b, me.c, len), lz(a, gate ? a.z : a.x, gate ? a.ldz : a.ldx, b, me.c, len);
  float bias[V], skip[V], gskip[V], gbias[V];
  params<V>(a.bias, me.c, me.on, bias);
  params<V>(a.skip, me.c, me.on, skip);
#pragma unroll
  for (int k = 0; k < V; ++k) gskip[k] = gbias[k] = 0.f;
  Raw<T, V> nx[IT], nd[IT], ny[IT], nz[IT], cx[IT], cd[IT], cy[IT], cz[IT];
  float hb[NS], hn[NS];  // the state before this tile and before the next one
  auto fetch = [&](int s0) {
    if (!ENDS) lx.load(me.r, s0, nx);
    ld.load(me.r, s0, nd);
    ly.load(me.r, s0, ny);
    lz.load(me.r, s0, nz);
    if (!ENDS) {
      const float* hs = a.hs + (long)(s0 / TQ) * bn + saved;
#pragma unroll
      for (int i = 0; i < NS; ++i) hn[i] = hs[saved_at(i, ns, a.D)];
    }
  };
  auto stage = [&](int s0) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (me.r[i] < TQ) {
        const bool in = me.on && s0 + me.r[i] < len;
        const int at = me.r[i] * 64 + me.cl;
        float e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = ny[i][k];
        if (gate)
#pragma unroll
          for (int k = 0; k < V; ++k) e[k] *= siluf(nz[i][k]);
        Quad<V> qd, qx, qe;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float dt = step_size(nd[i][k] + bias[k], a.softplus);
          qd.v[k] = in ? dt : 0.f;
          qx.v[k] = in && !ENDS ? dt * nx[i][k] : 0.f;
          qe.v[k] = in ? e[k] : 0.f;
        }
        put(sd + at, qd);
        if (!ENDS) put(sx + at, qx);
        put(se + at, qe);
      }
      cx[i] = nx[i];
      cd[i] = nd[i];
      cy[i] = ny[i];
      cz[i] = nz[i];
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) hb[i] = i < ns && ok ? hn[i] : 0.f;
  };
  // where a lane's sum of lanes_sum goes in a row of sbc; a lane whose sum is
  // another lane's too writes behind the rows (no branch in the walk)
  const int val = lane_value<2 * NS>(lane);
  const bool writer = (lane & (32 / NS - 1)) == 0;
  const int col = !writer ? TQ * 2 * WN + lane : val < NS ? w * NS + val : WN + w * NS + val - NS;
  const int row = writer ? 2 * WN : 0;
  const int t0 = chunk * a.tpc, t1 = min(t0 + a.tpc, a.Tp / TQ);
  // outputs of time t: ybase + t ystep; pbc of this block and sequence: t bstep
  const long ystep = (long)a.B * a.D, ybase = (long)b * a.D + me.c, bstep = (long)a.B * 2 * a.N;
  float* pbc = a.pbc + ((long)blockIdx.x * a.T * a.B + b) * 2 * a.N;
  float sum_dt = 0.f;
  Group<NS, UR> next;
  next.load(bcw + (long)(ENDS ? t1 * TQ - UR : (t1 - 1) * TQ) * 2 * NS);
  fetch((t1 - 1) * TQ);
  stage((t1 - 1) * TQ);
  __syncthreads();
  // One tile; tail: with rows behind the sequence's end, which add nothing to dA by selection
  // (their zeros times an infinite last state are not zero).  In every tile that takes 7%
  // longer, in a loop of its own 2%.
  auto back = [&](int tile, auto tail) {
    const int s0 = tile * TQ;
    const bool more = tile > t0;
    if constexpr (ENDS) {
      fetch(more ? s0 - TQ : s0);
#pragma unroll
      for (int r0 = TQ - UR; r0 >= 0; r0 -= UR) {
        const Group<NS, UR> bc = next;
        next.load(bcw + (long)max(s0 + r0 - UR, 0) * 2 * NS);
#pragma unroll
        for (int k = UR - 1; k >= 0; --k) {
          const float dt = sd[(r0 + k) * 64 + lane], e = se[(r0 + k) * 64 + lane];
          sum_dt += dt;
#pragma unroll
          for (int i = 0; i < NS; ++i)
            carry[i] = fmaf(bc.C(k, i), e, carry[i]) * __builtin_amdgcn_exp2f(dt * (A1[i] * LOG2E));
        }
      }
      __syncthreads();
      if (more) stage(s0 - TQ);
    } else {
      float H[TQ][NS], dec[TQ][NS], dAt[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) dAt[i] = 0.f;
#pragma unroll
      for (int r0 = 0; r0 < TQ; r0 += UR) {
        const Group<NS, UR> bc = next;
        if (r0 + UR < TQ) next.load(bcw + (long)(s0 + r0 + UR) * 2 * NS);
#pragma unroll
        for (int k = 0; k < UR; ++k) {
          const int r = r0 + k;
          const float2 u = make_float2(sd[r * 64 + lane], sx[r * 64 + lane]);
          float v = 0.f;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            dec[r][i] = __builtin_amdgcn_exp2f(u.x * (A1[i] * LOG2E));
            const float in = u.y * bc.B(k, i);
            H[r][i] = fmaf(dec[r][i], r ? H[r - 1][i] : hb[i], PART && i >= ns ? 0.f : in);
            v = fmaf(bc.C(k, i), H[r][i], v);
          }
          yp[(w * TQ + r) * 64 + lane] = v;
        }
      }
#pragma unroll
      for (int r0 = TQ - UR; r0 >= 0; r0 -= UR) {
        const Group<NS, UR> bc = next;
        // the group before; behind a tile's first one comes the earlier tile's first
        next.load(bcw + (long)max(r0 ? s0 + r0 - UR : s0 - TQ, 0) * 2 * NS);
#pragma unroll
        for (int k = UR - 1; k >= 0; --k) {
          const int r = r0 + k;
          const float2 u = make_float2(sd[r * 64 + lane], sx[r * 64 + lane]);
          const float e = se[r * 64 + lane];
          float p = 0.f, q = 0.f, red[2 * NS];
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            const float full = fmaf(bc.C(k, i), e, carry[i]), g = PART && i >= ns ? 0.f : full;
            p = fmaf(g, bc.B(k, i), p);
            red[i] = g * u.y;
            red[NS + i] = e * H[r][i];
            carry[i] = g * dec[r][i];
            float t = carry[i] * (r ? H[r - 1][i] : hb[i]);
            if (tail) t = zero_from(t, s0 + r, len);
            q = fmaf(t, A1[i], q);
            dAt[i] = fmaf(t, u.x, dAt[i]);
          }
          pp[(w * TQ + r) * 64 + lane] = p;
          pq[(w * TQ + r) * 64 + lane] = q;
          const float s = lanes_sum<2 * NS>(red, lane);
          sbc[col + r * row] = s;
        }
      }
      fetch(more ? s0 - TQ : s0);  // here, where H and dec have left their registers
#pragma unroll
      for (int i = 0; i < NS; ++i) dA[i] += dAt[i];
      __syncthreads();
      float ox[IT][V], od[IT][V], oz[IT][V];
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = me.r[i];
        if (r >= TQ) continue;
        const bool in = s0 + r < len;
        const int at = r * 64 + me.cl;
        float p[V], q[V], v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] = q[k] = v[k] = 0.f;
        auto add = [&](int u) {
          const Quad<V> tp = get<V>(pp + u * TQ * 64 + at), tq = get<V>(pq + u * TQ * 64 + at),
                        tv = get<V>(yp + u * TQ * 64 + at);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            p[k] += tp.v[k];
            q[k] += tq.v[k];
            v[k] += tv.v[k];
          }
        };
#pragma unroll
        for (int u = 0; u < 4; ++u) add(u);  // W >= 4
        for (int u = 4; u < a.W; ++u) add(u);
        const Quad<V> me_d = get<V>(sd + at), me_e = get<V>(se + at);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float x = in ? cx[i][k] : 0.f, e = me_e.v[k];
          const float sg = sigmoidf(cd[i][k] + bias[k]), dd = fmaf(x, p[k], q[k]);
          ox[i][k] = in ? fmaf(me_d.v[k], p[k], a.skip ? skip[k] * e : 0.f) : 0.f;
          od[i][k] = in ? (a.softplus ? dd * sg : dd) : 0.f;
          v[k] = a.skip ? fmaf(skip[k], x, v[k]) : v[k];
          gskip[k] = fmaf(e, x, gskip[k]);
          gbias[k] += od[i][k];
        }
        if (gate)
#pragma unroll
          for (int k = 0; k < V; ++k) oz[i][k] = in ? cy[i][k] * v[k] * dsiluf(cz[i][k]) : 0.f;
      }
      // (a thread stages the elements that it has just read)
      if (more) stage(s0 - TQ);
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int s = s0 + me.r[i];
        if (me.r[i] < TQ && s < a.T && me.on) {
          const long at = time_of(a, s, len) * ystep + ybase;
          store_vec<T, V>((T*)a.dx + at, ox[i]);
          store_vec<T, V>((T*)a.ddelta + at, od[i]);
          if (gate) store_vec<T, V>((T*)a.dz + at, oz[i]);
        }
      }
      for (int i = threadIdx.x; i < TQ * 2 * a.N; i += nt) {
        const int r = a.by2n.div(i), j = i - r * 2 * a.N, s = s0 + r;
        if (s < a.T)
          pbc[time_of(a, s, len) * bstep + j] =
              s < len ? sbc[r * 2 * WN + (j < a.N ? j : WN + j - a.N)] : 0.f;  // (not 0 * inf)
      }
    }
    __syncthreads();
  };
  int tile = t1 - 1;
  if constexpr (!ENDS)
    for (; tile >= t0 && (PART || (tile + 1) * TQ > len); --tile) back(tile, std::true_type{});
  if constexpr (!PART)
    for (; tile >= t0; --tile) back(tile, std::false_type{});
  if constexpr (ENDS) {
    if (ok)
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (i < ns) a.ends[chunk * bn + bnd + (long)i * a.D] = carry[i];
    if (w == 0 && ok) a.sums[((long)chunk * a.B + b) * a.D + d] = sum_dt;
    return;
  }
  float* pch = a.pch + ((long)chunk * a.B + b) * (a.N + 2) * a.D;
  if (ok)
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (i < ns) {
        pch[(long)(w * NS + i) * a.D + d] = dA[i];
        if (a.dh0 && chunk == 0) a.dh0[bnd + (long)i * a.D] = carry[i];
      }
  // dskip, dbias: a thread holds V channels of some rows
  const int nrow = nt / (64 / V), mine = threadIdx.x / (64 / V);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    lds[mine * 64 + me.cl + k] = gskip[k];
    lds[(nrow + mine) * 64 + me.cl + k] = gbias[k];
  }
  __syncthreads();
  if (w == 0 && ok) {
    float u = 0.f, v = 0.f;
    for (int r = 0; r < nrow; ++r) {
      u += lds[r * 64 + lane];
      v += lds[(nrow + r) * 64 + lane];
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
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < nblk; k += 4)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < nblk) s[u] += p[(k + u) * total + i];
    const long row = i / (2 * N);
    const int n = (int)(i % (2 * N));
    (n < N ? db : dc)[row * N + (n < N ? n : n - N)] = from_f32<T>((s[0] + s[1]) + (s[2] + s[3]));
  }
}

// dA [N][D], dskip, dbias [D]: the sum over the slabs of pch [S][N + 2][D], 32
// columns x 8 rows a workgroup
__global__ void __launch_bounds__(256)
param_grad_k(const float* __restrict__ p, int S, int N, int D, const float* log_a, float* dA,
             float* dskip, float* dbias, int acc_a, int acc_s, int acc_b) {
  __shared__ float red[8][33];
  const long total = (long)(N + 2) * D;
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
  const int n = (int)(i / D);
  float* out = n < N ? dA : n == N ? dskip : dbias;
  const int acc = n < N ? acc_a : n == N ? acc_s : acc_b;
  if (!out) return;
  if (n < N && log_a) sum *= -expf(log_a[i]);
  out += n < N ? i : i % D;
  *out = acc ? *out + sum : sum;
}

// One token: state [B][N][D] in place.  64 channels x 4 waves, wave w the
// states w, w + 4, ...  64 x 16 x 1600 states, 13 MB read and written: 6.0 us
// (2.2 TB/s; an empty launch alone is 3.5).
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
      const float e = __builtin_amdgcn_exp2f(dt * (rate(a, (long)n * a.D + d) * LOG2E));
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
  int fc, bc;  // chunks of the forward and of the backward
};

// A sequence is cut where its workgroups alone leave the card idle (fewer than
// ``alone``), into ``want`` workgroups of at least 4 tiles.  Forward at 874 steps of
// 1600 channels, 16 states: 16 sequences (400 workgroups) 255 us whole, 226 in 800
// workgroups, 183 in 2000; 32 sequences (800) 286 us whole, 341 in 1600.  Backward,
// two workgroups a compute unit: 16 sequences 535 us whole, 600 in 2000.
inline int chunks_of(long wgs, int tiles, long alone, long want) {
  long c = wgs >= alone ? 1 : want / wgs;
  if (c > tiles / 4) c = tiles / 4;
  return (int)(c < 1 ? 1 : c > 65535 ? 65535 : c);
}

inline Plan plan(int T, int B, int D, int N) {
  Plan p;
  p.ns = N <= 4 ? 1 : N <= 8 ? 2 : N <= 32 ? 4 : 8;
  p.tq = N <= 32 ? 16 : 8;
  p.W = ceil_div(N, p.ns);
  if (p.W < 4) p.W = 4;  // the elementwise passes want the threads
  p.tiles = ceil_div(T, p.tq);
  p.Tp = p.tiles * p.tq;
  const long wgs = (long)ceil_div(D, 64) * B;
  p.fc = chunks_of(wgs, p.tiles, 640, 2048);
  p.bc = chunks_of(wgs, p.tiles, 256, 512);
  return p;
}

// tiles of a chunk; the count may come out smaller than asked for
inline void cut(Args& a, const Plan& p, int chunks) {
  a.tpc = ceil_div(p.tiles, chunks);
  a.nchunk = ceil_div(p.tiles, a.tpc);
}

inline bool bad(const Args& a) {
  return a.T <= 0 || a.B <= 0 || a.D <= 0 || a.N <= 0 || a.N > 64 || a.B > 65535 ||
         a.T > INT32_MAX - 64;
}

}  // namespace ssm
}  // namespace kfb

using namespace kfb;

// NS states a wave and tiles of TQ steps; V channels a vector, IT vectors a
// thread: 4 to 8 waves hold a tile.
#define KFB_SSM_VEC(v, V, IT, one, ...)                    \
  if (v == 4) { constexpr int V = 4, IT = 1; __VA_ARGS__; } \
  else { constexpr int V = 1, IT = one; __VA_ARGS__; }

#define KFB_SSM_CONFIG(p, v, V, IT, NS, TQ, ...)                                                          \
  switch (p.ns) {                                                                                         \
    case 1: { constexpr int NS = 1, TQ = 16; KFB_SSM_VEC(v, V, IT, 4, __VA_ARGS__) break; }                \
    case 2: { constexpr int NS = 2, TQ = 16; KFB_SSM_VEC(v, V, IT, 4, __VA_ARGS__) break; }                \
    case 4: { constexpr int NS = 4, TQ = 16; KFB_SSM_VEC(v, V, IT, 4, __VA_ARGS__) break; }                \
    default: { constexpr int NS = 8, TQ = 8; KFB_SSM_VEC(v, V, IT, 2, __VA_ARGS__) break; }                \
  }

// Floats of: the fp32 copy of B and C and the forward's chunk ends (what = 0),
// the saved states of a training forward (1), the backward's workspace (2).
KFB_API long kfb_ssm_floats(int what, int T, int B, int D, int N) {
  if (T <= 0 || B <= 0 || D <= 0 || N <= 0) return 0;
  const ssm::Plan p = ssm::plan(T, B, D, N);
  const long state = (long)B * N * D, chunk = state + (long)B * D;
  switch (what) {
    case 0: return (long)B * p.W * p.Tp * 2 * p.ns + ssm::BC_PAD + (p.fc > 1 ? p.fc * chunk : 0);
    case 1: return (long)p.tiles * state;
    case 2: return (long)ceil_div(D, 64) * T * B * 2 * N + (long)B * p.bc * (N + 2) * D +
                   (p.bc > 1 ? p.bc * chunk : 0);
    default: return -1;
  }
}

// The furthest element of the saved states that the backward reads: every wave's in
// the last tile of the last sequence and channel.
KFB_API long kfb_ssm_furthest_state(int T, int B, int D, int N) {
  if (T <= 0 || B <= 0 || D <= 0 || N <= 0 || N > 64) return -1;
  const ssm::Plan p = ssm::plan(T, B, D, N);
  long most = -1;
  for (int w = 0; w < p.W; ++w)
    for (int i = 0; i < p.ns; ++i) {
      const int own = N - w * p.ns, ns = own < 0 ? 0 : own < p.ns ? own : p.ns;
      const long at = (long)(p.tiles - 1) * B * N * D + ssm::state_at(B - 1, ssm::base_state(w, p.ns, N), N, D, D - 1) +
                      ssm::saved_at(i, ns, D);
      if (at > most) most = at;
    }
  return most;
}

KFB_API hipError_t kfb_ssm_scan_fwd(int dtype, int V_, const void* x, long ldx, const void* delta,
                                    long ldd, const void* z, long ldz, const void* bm, long ldb,
                                    const void* cm, long ldc, const float* A, const float* skip,
                                    const float* bias, const int* len, const float* h0, float* hT,
                                    float* hs, float* bc, void* y, int T, int B, int D, int N,
                                    int softplus, int reverse, int log_a, hipStream_t stream) {
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.bm = bm; a.cm = cm;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldb = ldb; a.ldc = ldc;
  a.A = A; a.skip = skip; a.bias = bias; a.len = len; a.h0 = h0; a.hT = hT; a.hs = hs; a.bc = bc;
  a.y = y;
  a.T = T; a.B = B; a.D = D; a.N = N; a.softplus = softplus; a.reverse = reverse; a.log_a = log_a;
  a.by2n = FastDiv(N > 0 ? 2 * N : 1);
  if (ssm::bad(a) || (V_ != 1 && V_ != 4)) return hipErrorInvalidValue;
  const ssm::Plan p = ssm::plan(T, B, D, N);
  a.W = p.W; a.Tp = p.Tp;
  ssm::cut(a, p, p.fc);
  a.ends = bc + (long)B * p.W * p.Tp * 2 * p.ns + ssm::BC_PAD;
  a.sums = a.ends + (long)p.fc * B * N * D;
  KFB_DISPATCH_DTYPE(dtype, E, KFB_SSM_CONFIG(p, V_, V, IT, NS, TQ, {
    const long total = (long)B * p.W * p.Tp * 2 * NS;
    hipLaunchKernelGGL((ssm::prep_k<E, NS>), dim3(ceil_div(total < (1l << 22) ? total : (1l << 22), 256)),
                       dim3(256), 0, stream, a);
    const size_t shm = (size_t)(2 + p.W) * TQ * 64 * sizeof(float);
    dim3 grid(ceil_div(D, 64), B, a.nchunk - 1);
    if (grid.z)
      hipLaunchKernelGGL((ssm::scan_fwd_k<E, V, IT, NS, TQ, true, false>), grid, dim3(p.W * 64),
                         2 * TQ * 64 * sizeof(float), stream, a);
    grid.z = a.nchunk;
    if (N == p.W * NS)
      hipLaunchKernelGGL((ssm::scan_fwd_k<E, V, IT, NS, TQ, false, false>), grid, dim3(p.W * 64), shm, stream, a);
    else
      hipLaunchKernelGGL((ssm::scan_fwd_k<E, V, IT, NS, TQ, false, true>), grid, dim3(p.W * 64), shm, stream, a);
  }));
  return hipGetLastError();
}

KFB_API hipError_t kfb_ssm_scan_bwd(int dtype, int V_, const void* dy, long ldy, const void* x,
                                    long ldx, const void* delta, long ldd, const void* z, long ldz,
                                    const float* A, const float* skip, const float* bias,
                                    const int* len, const float* hs, float* bc, const float* dhT,
                                    float* dh0, void* dx, void* ddelta, void* dz, void* db,
                                    void* dc, float* dA, float* dskip, float* dbias, int acc_a,
                                    int acc_skip, int acc_bias, float* ws, int T, int B, int D,
                                    int N, int softplus, int reverse, int log_a, hipStream_t stream) {
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.dy = dy;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldy = ldy;
  a.A = A; a.skip = skip; a.bias = bias; a.len = len; a.hs = const_cast<float*>(hs); a.bc = bc;
  a.dhT = dhT; a.dh0 = dh0; a.dx = dx; a.ddelta = ddelta; a.dz = dz;
  a.T = T; a.B = B; a.D = D; a.N = N; a.softplus = softplus; a.reverse = reverse; a.log_a = log_a;
  a.by2n = FastDiv(N > 0 ? 2 * N : 1);
  if (ssm::bad(a) || (V_ != 1 && V_ != 4) || !ws || !hs) return hipErrorInvalidValue;
  const ssm::Plan p = ssm::plan(T, B, D, N);
  a.W = p.W; a.Tp = p.Tp;
  ssm::cut(a, p, p.bc);
  const int nblk = ceil_div(D, 64);
  const long rows = (long)T * B;
  a.pbc = ws;
  a.pch = ws + (long)nblk * rows * 2 * N;
  a.ends = a.pch + (long)B * p.bc * (N + 2) * D;
  a.sums = a.ends + (long)p.bc * B * N * D;
  KFB_DISPATCH_DTYPE(dtype, E, {
    KFB_SSM_CONFIG(p, V_, V, IT, NS, TQ, {
      size_t shm = sizeof(float) * ((size_t)(3 + 3 * p.W) * TQ * 64 + (size_t)TQ * 2 * p.W * NS + 64);
      const size_t last = sizeof(float) * 2 * 64 * p.W * V;
      if (shm < last) shm = last;
      dim3 grid(nblk, B, a.nchunk - 1);
      if (grid.z)
        hipLaunchKernelGGL((ssm::scan_bwd_k<E, V, IT, NS, TQ, true, false>), grid, dim3(p.W * 64),
                           3 * TQ * 64 * sizeof(float), stream, a);
      grid.z = a.nchunk;
      if (N == p.W * NS)
        hipLaunchKernelGGL((ssm::scan_bwd_k<E, V, IT, NS, TQ, false, false>), grid, dim3(p.W * 64), shm, stream, a);
      else
        hipLaunchKernelGGL((ssm::scan_bwd_k<E, V, IT, NS, TQ, false, true>), grid, dim3(p.W * 64), shm, stream, a);
    });
    hipLaunchKernelGGL((ssm::bc_grad_k<E>), dim3(ceil_div(rows * 2 * N < (1l << 22) ? rows * 2 * N : (1l << 22), 256)),
                       dim3(256), 0, stream, a.pbc, nblk, rows, N, (E*)db, (E*)dc);
  });
  hipLaunchKernelGGL(ssm::param_grad_k, dim3(ceil_div((long)(N + 2) * D, 32)), dim3(256), 0, stream,
                     a.pch, B * a.nchunk, N, D, log_a ? A : nullptr, dA, dskip, dbias, acc_a, acc_skip, acc_bias);
  return hipGetLastError();
}

KFB_API hipError_t kfb_ssm_step(int dtype, const void* x, long ldx, const void* delta, long ldd,
                                const void* z, long ldz, const void* bm, long ldb, const void* cm,
                                long ldc, const float* A, const float* skip, const float* bias,
                                float* state, void* y, int B, int D, int N, int softplus,
                                int log_a, hipStream_t stream) {
  ssm::Args a{};
  a.x = x; a.delta = delta; a.z = z; a.bm = bm; a.cm = cm;
  a.ldx = ldx; a.ldd = ldd; a.ldz = ldz; a.ldb = ldb; a.ldc = ldc;
  a.A = A; a.skip = skip; a.bias = bias; a.y = y;
  a.T = 1; a.B = B; a.D = D; a.N = N; a.softplus = softplus; a.log_a = log_a;
  if (ssm::bad(a)) return hipErrorInvalidValue;
  KFB_DISPATCH_DTYPE(dtype, E, {
    hipLaunchKernelGGL((ssm::step_k<E>), dim3(ceil_div(D, 64), B), dim3(256), 0, stream, a, state);
  });
  return hipGetLastError();
}
