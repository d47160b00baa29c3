// Group norm with an activation on channels-last activations [N][HW][C]:
// group g of image n is HW rows x cpg = C / G channels, M = HW cpg values,
//   mu = mean, r = 1 / sqrt(var + eps), xh = (x - mu) r,
//   y = act(gamma xh + beta);
//   e = dy act'(gamma xh + beta), dbeta = sum e, dgamma = sum e xh,
//   dx = r (gamma e - (s1 + xh s2) / M), s1 = sum_g gamma e, s2 = sum_g gamma e xh.
// The backward recomputes xh and the activation from x: nothing but mu and r
// is stored.  All sums are fp32; the variance is that of the centred values.
//
// Bound by HBM.  A workgroup covers whole groups, at least 128 bytes of
// neighbouring channels, in 16-byte vectors: thread = (image, row, vector column).
//   * resident (gn_fwd_tile_k, gn_bwd_tile_k): the rows of an image fit the
//     workgroup's registers, so x (and dy) are read once and one launch does all
//     (32 x 28 x 28 x 512 bf16 in 32 groups: 16.5 us, 3.1 TB/s; 32 x 14 x 14 x 1024:
//     11.2 us forward, 14.9 backward);
//   * split: statistics of row chunks, then an apply pass that merges them in
//     its prologue (images too large for one workgroup; the second read comes
//     from the last-level cache while the tensor is below its 256 MB).  32 x 56 x
//     56 x 256 bf16 in 32 groups, 51 MB a tensor: statistics 13.7 us, y 23.6,
//     backward sums 22.5, dx 35.0 (3.8, 4.3, 4.6 and 4.4 TB/s; a copy: 5.2);
//   * rows (group_norm_rows.hip): one row an image, groups held by lanes;
//   * gn_*_any_k: one workgroup per image and group (backward: up to 2048, each a
//     slab of channel sums), for groups wider than 512 vectors (every image and
//     group of the split case above this way: 480 us, not 95).
#include "group_norm.h"

namespace kfb {
namespace gn {

constexpr int NT = 256;

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
template <typename T, int KIND>
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
      y[r * a.C + c] = from_f32<T>(act_fwd<KIND>(fmaf((to_f32(x[r * a.C + c]) - mu) * rs, ga, be), a.act));
  }
  }
}

// (images slab, slab + slabs, ... of a group, whose channel sums are added up in the slab)
template <typename T, int KIND>
__global__ void __launch_bounds__(NT) gn_bwd_any_k(Args a, int tc, int slabs) {
  __shared__ float red[NT / 64], colp[NT], colq[NT];
  const int c0 = threadIdx.x % tc, r0 = threadIdx.x / tc, rp = NT / tc;
  const int g = blockIdx.x % a.G, slab = blockIdx.x / a.G;
  for (long n = slab; n < a.N; n += slabs) {
  const long id = n * a.G + g;
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
        const float e = to_f32(dy[r * a.C + c]) * act_grad<KIND>(fmaf(xh, ga, be), a.act);
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
      float* at = a.part + (long)slab * 2 * a.C + ch;
      at[0] = n == slab ? q : at[0] + q;
      at[a.C] = n == slab ? p : at[a.C] + p;
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
      const float e = to_f32(dy[r * a.C + c]) * act_grad<KIND>(fmaf(xh, ga, be), a.act);
      dx[r * a.C + c] = from_f32<T>(rs * (fmaf(ga, e, -s1) - xh * s2));
    }
  }
  }
}

// ---------------------------------------------------------------- tiled kernels
// A tile: sp images (resident) or one (split) x rows x cb channels.
struct Tile {
  int ncol;   // vector columns of a workgroup
  int rp;     // rows in parallel
  int sp;     // images in parallel
  int cb;     // channels of a workgroup, whole groups
  int gb;     // groups of a workgroup
  int nblk;   // column blocks
  int nchunk; // row chunks of an image
  int rows;   // rows of a chunk
  int fold;   // every vector lies in one group: reduce it before LDS
  int glw;    // LDS values of a group and row
  int lp;     // lanes that sum a group, a power of two
  int nt;     // threads
  long total; // tiles
  FastDiv dcol, drp, dglw, dcpg, dgb;
};

// Where a thread stands in tile ``id``.
struct At {
  int col, r, s, q, c0, cbw, gbw, c;  // c: its first channel
  long n, row0;
  bool on;
};

template <int V>
__device__ __forceinline__ At place(const Args& a, const Tile& t, long id) {
  At p;
  const int tid = threadIdx.x;
  p.q = t.dcol.div(tid);
  p.col = tid - p.q * t.ncol;
  p.s = t.drp.div(p.q);
  p.r = p.q - p.s * t.rp;
  const int blk = (int)(id % t.nblk);
  id /= t.nblk;
  p.c0 = blk * t.cb;
  p.cbw = min(t.cb, a.C - p.c0);
  p.gbw = t.dcpg.div(p.cbw);
  p.row0 = id % t.nchunk * t.rows;
  p.n = id / t.nchunk * t.sp + p.s;
  p.c = p.c0 + p.col * V;
  p.on = p.s < t.sp && p.col * V < p.cbw && p.n < a.N;
  return p;
}

// tot[image * gb + group] = sum over the rows and the group's channels of the
// threads' v.  LDS values of a thread: one per vector (fold) or one per channel.
template <int V, int VG>
__device__ __forceinline__ void group_reduce(const Tile& t, const At& p, float* buf, float* tot,
                                             const float (&v)[V]) {
  const int tid = threadIdx.x, rowlen = t.ncol * VG;
  __syncthreads();
  if (p.q < t.sp * t.rp) {
    if constexpr (VG == 1) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[i];
      buf[p.q * rowlen + p.col] = s;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) buf[p.q * rowlen + p.col * V + i] = v[i];
    }
  }
  __syncthreads();
  const int j = tid & (t.lp - 1), per = t.nt / t.lp, n = t.rp * t.glw;
  for (int pr = tid / t.lp; pr < t.sp * t.gb; pr += per) {
    const int s = t.dgb.div(pr), gl = pr - s * t.gb;
    float sum = 0.f;
    if (gl < p.gbw) {
      const float* b = buf + s * t.rp * rowlen + gl * t.glw;
      for (int e = j; e < n; e += t.lp) {
        const int rr = t.dglw.div(e);
        sum += b[rr * rowlen + e - rr * t.glw];
      }
    }
    for (int o = t.lp >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (j == 0) tot[pr] = sum;
  }
  __syncthreads();
}

// The values of a thread's groups out of a table: VG = 1 where every vector lies
// in one group (fold), else one for each of its V channels.
template <int V, int VG>
__device__ __forceinline__ void of_groups(const Tile& t, const At& p, const float* tab,
                                          float (&v)[VG]) {
#pragma unroll
  for (int i = 0; i < VG; ++i) v[i] = p.on ? tab[p.s * t.gb + t.dcpg.div(p.col * V + i)] : 0.f;
}

// mean and 1 / std of a thread's groups
template <int V, int VG>
__device__ __forceinline__ void load_stats(const Args& a, const Tile& t, const At& p,
                                           float (&mu)[VG], float (&rs)[VG]) {
  const int g0 = t.dcpg.div(p.c0);
#pragma unroll
  for (int i = 0; i < VG; ++i) {
    const long g = p.n * a.G + g0 + t.dcpg.div(p.col * V + i);
    mu[i] = p.on ? a.mean[g] : 0.f;
    rs[i] = p.on ? a.rstd[g] : 0.f;
  }
}

// Rows of a chunk in registers (K vectors a thread): mean, then the centred
// squares, and where the chunk is the image also y.  part: (mean, M2) of the
// chunks [N][nchunk][G], or null when resident.
template <typename T, int V, int VG, int KIND, int K>
__global__ void __launch_bounds__(512) gn_fwd_tile_k(Args a, Tile t, float2* __restrict__ part) {
  extern __shared__ float lds[];
  float* tot = lds;
  float* buf = lds + t.sp * t.gb;
  for (long id = blockIdx.x; id < t.total; id += gridDim.x) {
    const At p = place<V>(a, t, id);
    const int rows = p.on ? (int)min((long)t.rows, a.HW - p.row0) : 0;
    const T* __restrict__ x = (const T*)a.x + (p.n * a.HW + p.row0) * a.C + p.c;
    Raw<T, V> raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows) raw[k].load(x + (long)(p.r + k * t.rp) * a.C);
    float mu[VG], v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows)
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += raw[k][i];
    const float inv = 1.f / ((float)min((long)t.rows, a.HW - p.row0) * a.cpg);
    group_reduce<V, VG>(t, p, buf, tot, v);
    of_groups<V, VG>(t, p, tot, mu);
    const float mu_g = (int)threadIdx.x < t.sp * t.gb ? tot[threadIdx.x] * inv : 0.f;
#pragma unroll
    for (int i = 0; i < VG; ++i) mu[i] *= inv;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = raw[k][i] - mu[i % VG];
          v[i] = fmaf(d, d, v[i]);
        }
    // (tot is rewritten behind group_reduce's first barrier)
    group_reduce<V, VG>(t, p, buf, tot, v);
    if ((int)threadIdx.x < t.sp * t.gb) {
      // thread i: group i % gb of image i / gb (sp gb <= threads, host-checked)
      const int s = t.dgb.div(threadIdx.x), gl = threadIdx.x - s * t.gb;
      const long n = p.n - p.s + s;
      const long g = t.dcpg.div(p.c0) + gl;
      if (n < a.N && gl < p.gbw) {
        if (part) {
          part[(n * t.nchunk + p.row0 / t.rows) * a.G + g] = make_float2(mu_g, tot[threadIdx.x]);
        } else {
          a.mean[n * a.G + g] = mu_g;
          a.rstd[n * a.G + g] = 1.f / sqrtf(tot[threadIdx.x] * inv + a.eps);
        }
      }
    }
    if (!part) {
      float sc[V], be[V], m2[VG];
      load_params<V>(a.gamma, p.c, p.on, 1.f, sc);
      load_params<V>(a.beta, p.c, p.on, 0.f, be);
      of_groups<V, VG>(t, p, tot, m2);
      T* __restrict__ y = (T*)a.y + (p.n * a.HW + p.row0) * a.C + p.c;
#pragma unroll
      for (int i = 0; i < VG; ++i) m2[i] = 1.f / sqrtf(m2[i] * inv + a.eps);
#pragma unroll
      for (int i = 0; i < V; ++i) sc[i] *= m2[i % VG];
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (p.r + k * t.rp < rows) {
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i)
            o[i] = act_fwd<KIND>(fmaf(raw[k][i] - mu[i % VG], sc[i], be[i]), a.act);
          store_vec<T, V>(y + (long)(p.r + k * t.rp) * a.C, o);
        }
    }
  }
}

// Split forward, second pass: the chunks' statistics are merged as
//   mean = sum n_i mean_i / M,  M2 = sum M2_i + n_i (mean_i - mean)^2
// (16 lanes a group), then y for a row chunk (its own chunking).
template <typename T, int V, int VG, int KIND>
__global__ void __launch_bounds__(512)
gn_apply_k(Args a, Tile t, const float2* __restrict__ part, int pchunk, int prows) {
  extern __shared__ float lds[];
  float* mean = lds;
  float* rstd = lds + t.gb;
  for (long id = blockIdx.x; id < t.total; id += gridDim.x) {
    const At p = place<V>(a, t, id);
    const long n = id / t.nblk / t.nchunk;
    const int g0 = t.dcpg.div(p.c0);
    __syncthreads();
    const int j = threadIdx.x & 15;
    for (int gl = threadIdx.x >> 4; gl < t.gb; gl += t.nt >> 4) {
      const float2* q = part + n * pchunk * a.G + g0 + gl;
      float s = 0.f, m2 = 0.f;
      const float inv = 1.f / ((float)a.HW * a.cpg);
      if (gl < p.gbw)
        for (int i = j; i < pchunk; i += 16)
          s = fmaf((float)min((long)prows, a.HW - (long)i * prows) * a.cpg, q[(long)i * a.G].x, s);
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
      s *= inv;
      if (gl < p.gbw)
        for (int i = j; i < pchunk; i += 16) {
          const float2 u = q[(long)i * a.G];
          const float d = u.x - s;
          m2 += fmaf((float)min((long)prows, a.HW - (long)i * prows) * a.cpg * d, d, u.y);
        }
      for (int o = 8; o > 0; o >>= 1) m2 += __shfl_xor(m2, o, 64);
      const float rs = 1.f / sqrtf(m2 * inv + a.eps);
      if (j == 0) {
        mean[gl] = s;
        rstd[gl] = rs;
        if (p.row0 == 0 && gl < p.gbw) {
          a.mean[n * a.G + g0 + gl] = s;
          a.rstd[n * a.G + g0 + gl] = rs;
        }
      }
    }
    __syncthreads();
    if (!p.on) continue;
    float mu[VG], rs[VG], sc[V], be[V];
    of_groups<V, VG>(t, p, mean, mu);
    of_groups<V, VG>(t, p, rstd, rs);
    load_params<V>(a.gamma, p.c, true, 1.f, sc);
    load_params<V>(a.beta, p.c, true, 0.f, be);
#pragma unroll
    for (int i = 0; i < V; ++i) sc[i] *= rs[i % VG];
    const long base = (p.n * a.HW + p.row0) * a.C + p.c;
    const int rows = (int)min((long)t.rows, a.HW - p.row0);
    const T* __restrict__ x = (const T*)a.x + base;
    T* __restrict__ y = (T*)a.y + base;
    constexpr int U = 4;
    for (int r = p.r; r < rows; r += U * t.rp) {
      Raw<T, V> raw[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) raw[k].load(x + (long)(r + k * t.rp) * a.C);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) {
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i)
            o[i] = act_fwd<KIND>(fmaf(raw[k][i] - mu[i % VG], sc[i], be[i]), a.act);
          store_vec<T, V>(y + (long)(r + k * t.rp) * a.C, o);
        }
    }
  }
}

// out[c] = sum over a tile's images and rows of v, for the cbw channels at c0.
template <int V>
__device__ __forceinline__ void channel_reduce(const Tile& t, const At& p, float* buf,
                                               const float (&v)[V], float* __restrict__ out) {
  const int rowlen = t.ncol * V;
  __syncthreads();
  if (p.q < t.sp * t.rp)
#pragma unroll
    for (int i = 0; i < V; ++i) buf[p.q * rowlen + p.col * V + i] = v[i];
  __syncthreads();
  for (int c = threadIdx.x; c < p.cbw; c += t.nt) {
    float s = 0.f;
    for (int q = 0; q < t.sp * t.rp; ++q) s += buf[q * rowlen + c];
    out[c] = s;
  }
}

// Resident backward: x and dy of whole images in registers.  The channel sums
// of all tiles of a workgroup go to its slab of part [slabs][2][C].
template <typename T, int V, int VG, int KIND, int K>
__global__ void __launch_bounds__(512) gn_bwd_tile_k(Args a, Tile t) {
  extern __shared__ float lds[];
  float* tot = lds;
  float* tot2 = lds + t.sp * t.gb;
  float* buf = lds + 2 * t.sp * t.gb;
  const float inv = 1.f / ((float)a.HW * a.cpg);
  float cp[V], cq[V], ga[V], be[V];
  const At p0 = place<V>(a, t, blockIdx.x);  // gridDim.x is a multiple of nblk: one column block
  load_params<V>(a.gamma, p0.c, p0.col * V < p0.cbw, 1.f, ga);
  load_params<V>(a.beta, p0.c, p0.col * V < p0.cbw, 0.f, be);
#pragma unroll
  for (int i = 0; i < V; ++i) cp[i] = cq[i] = 0.f;
  for (long id = blockIdx.x; id < t.total; id += gridDim.x) {
    const At p = place<V>(a, t, id);
    const int rows = p.on ? (int)a.HW : 0;
    const long base = p.n * a.HW * a.C + p.c;
    const T* __restrict__ x = (const T*)a.x + base;
    const T* __restrict__ dy = (const T*)a.dy + base;
    Raw<T, V> rx[K], rd[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows) {
        rx[k].load(x + (long)(p.r + k * t.rp) * a.C);
        rd[k].load(dy + (long)(p.r + k * t.rp) * a.C);
      }
    float mu[VG], rs[VG], sp[V], sq[V];
    load_stats<V, VG>(a, t, p, mu, rs);
#pragma unroll
    for (int i = 0; i < V; ++i) sp[i] = sq[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows) {
        float e[V], xh[V];
        grad_terms<T, V, VG, KIND>(a, rx[k], rd[k], mu, rs, ga, be, e, xh);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sp[i] += e[i];
          sq[i] = fmaf(e[i], xh[i], sq[i]);
        }
      }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      cp[i] += sp[i];
      cq[i] += sq[i];
      sp[i] *= ga[i];
      sq[i] *= ga[i];
    }
    group_reduce<V, VG>(t, p, buf, tot, sp);
    group_reduce<V, VG>(t, p, buf, tot2, sq);
    float s1[VG], s2[VG];
    of_groups<V, VG>(t, p, tot, s1);
    of_groups<V, VG>(t, p, tot2, s2);
    T* __restrict__ dx = (T*)a.y + base;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (p.r + k * t.rp < rows) {
        float e[V], xh[V];
        grad_terms<T, V, VG, KIND>(a, rx[k], rd[k], mu, rs, ga, be, e, xh);
#pragma unroll
        for (int i = 0; i < V; ++i)
          e[i] = rs[i % VG] * (fmaf(ga[i], e[i], -s1[i % VG] * inv) - xh[i] * (s2[i % VG] * inv));
        store_vec<T, V>(dx + (long)(p.r + k * t.rp) * a.C, e);
      }
  }
  float* out = a.part + (long)(blockIdx.x / t.nblk) * 2 * a.C + p0.c0;
  channel_reduce<V>(t, p0, buf, cq, out);
  channel_reduce<V>(t, p0, buf, cp, out + a.C);
}

// Split backward, first pass: a row chunk's channel sums into part
// [N * nchunk][2][C] and its (s1, s2) into gpart [N * nchunk][G].
template <typename T, int V, int VG, int KIND>
__global__ void __launch_bounds__(512) gn_bwd_sums_k(Args a, Tile t, float2* __restrict__ gpart) {
  extern __shared__ float lds[];
  float *tot = lds, *tot2 = lds + t.gb, *buf = lds + 2 * t.gb;
  for (long id = blockIdx.x; id < t.total; id += gridDim.x) {
    const At p = place<V>(a, t, id);
    float sp[V], sq[V], mu[VG], rs[VG], ga[V], be[V];
    load_params<V>(a.gamma, p.c, p.on, 1.f, ga);
    load_params<V>(a.beta, p.c, p.on, 0.f, be);
    load_stats<V, VG>(a, t, p, mu, rs);
#pragma unroll
    for (int i = 0; i < V; ++i) sp[i] = sq[i] = 0.f;
    const long base = (p.n * a.HW + p.row0) * a.C + p.c;
    const int rows = p.on ? (int)min((long)t.rows, a.HW - p.row0) : 0;
    const T* __restrict__ x = (const T*)a.x + base;
    const T* __restrict__ dy = (const T*)a.dy + base;
    constexpr int U = 4;
    for (int r = p.r; r < rows; r += U * t.rp) {
      Raw<T, V> rx[U], rd[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) {
          rx[k].load(x + (long)(r + k * t.rp) * a.C);
          rd[k].load(dy + (long)(r + k * t.rp) * a.C);
        }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) {
          float e[V], xh[V];
          grad_terms<T, V, VG, KIND>(a, rx[k], rd[k], mu, rs, ga, be, e, xh);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            sp[i] += e[i];
            sq[i] = fmaf(e[i], xh[i], sq[i]);
          }
        }
    }
    const long slab = id / t.nblk;
    float* out = a.part + slab * 2 * a.C + p.c0;
    channel_reduce<V>(t, p, buf, sq, out);
    channel_reduce<V>(t, p, buf, sp, out + a.C);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sp[i] *= ga[i];
      sq[i] *= ga[i];
    }
    group_reduce<V, VG>(t, p, buf, tot, sp);
    group_reduce<V, VG>(t, p, buf, tot2, sq);
    if ((int)threadIdx.x < p.gbw)
      gpart[slab * a.G + t.dcpg.div(p.c0) + threadIdx.x] = make_float2(tot[threadIdx.x], tot2[threadIdx.x]);
  }
}

// dgamma / dbeta = sum over the slabs of part [S][2][C], in a fixed order: the
// same sum on every run.  16 of the 2 C columns x blockDim / 16 rows a workgroup.
struct ParamGrad {
  const float* part;
  float *dgamma, *dbeta;
  long S;
  int C, acc_g, acc_b, blocks;
};

__device__ __forceinline__ void param_grad(const ParamGrad& q, int block, float* red) {
  const int nt = blockDim.x, cl = threadIdx.x % 16, r0 = threadIdx.x / 16, nr = nt / 16;
  const int c = block * 16 + cl;
  constexpr int U = 8;
  float s[U];
#pragma unroll
  for (int k = 0; k < U; ++k) s[k] = 0.f;
  if (c < 2 * q.C)
    for (long r = r0; r < q.S; r += U * nr)
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + nr * k < q.S) s[k] += q.part[(r + nr * k) * 2 * q.C + c];
  red[threadIdx.x] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (r0 == 0 && c < 2 * q.C) {
    float sum = 0.f;
    for (int r = 0; r < nr; ++r) sum += red[r * 16 + cl];
    float* out = c < q.C ? q.dgamma : q.dbeta;
    const int acc = c < q.C ? q.acc_g : q.acc_b, i = c < q.C ? c : c - q.C;
    if (out) out[i] = acc ? out[i] + sum : sum;
  }
}

__global__ void __launch_bounds__(1024) gn_param_grad_k(ParamGrad q) {
  __shared__ float red[1024];
  param_grad(q, blockIdx.x, red);
}

// Split backward, second pass: the first q.blocks workgroups sum dgamma and
// dbeta; the others merge (s1, s2) of their groups and write dx.
template <typename T, int V, int VG, int KIND>
__global__ void __launch_bounds__(512)
gn_bwd_apply_k(Args a, Tile t, const float2* __restrict__ gpart, int pchunk, ParamGrad q) {
  extern __shared__ float lds[];
  if ((int)blockIdx.x < q.blocks) {
    param_grad(q, blockIdx.x, lds);
    return;
  }
  float *s1 = lds, *s2 = lds + t.gb;
  const float inv = 1.f / ((float)a.HW * a.cpg);
  for (long id = blockIdx.x - q.blocks; id < t.total; id += gridDim.x - q.blocks) {
    const At p = place<V>(a, t, id);
    const long n = id / t.nblk / t.nchunk;
    const int g0 = t.dcpg.div(p.c0);
    __syncthreads();
    const int j = threadIdx.x & 15;
    for (int gl = threadIdx.x >> 4; gl < t.gb; gl += t.nt >> 4) {
      float u = 0.f, v = 0.f;
      if (gl < p.gbw)
        for (int i = j; i < pchunk; i += 16) {
          const float2 w = gpart[(n * pchunk + i) * a.G + g0 + gl];
          u += w.x;
          v += w.y;
        }
      for (int o = 8; o > 0; o >>= 1) {
        u += __shfl_xor(u, o, 64);
        v += __shfl_xor(v, o, 64);
      }
      if (j == 0) {
        s1[gl] = u * inv;
        s2[gl] = v * inv;
      }
    }
    __syncthreads();
    if (!p.on) continue;
    float sp[VG], sq[VG], mu[VG], rs[VG], ga[V], be[V];
    of_groups<V, VG>(t, p, s1, sp);
    of_groups<V, VG>(t, p, s2, sq);
    load_params<V>(a.gamma, p.c, true, 1.f, ga);
    load_params<V>(a.beta, p.c, true, 0.f, be);
    load_stats<V, VG>(a, t, p, mu, rs);
    const long base = (p.n * a.HW + p.row0) * a.C + p.c;
    const int rows = (int)min((long)t.rows, a.HW - p.row0);
    const T* __restrict__ x = (const T*)a.x + base;
    const T* __restrict__ dy = (const T*)a.dy + base;
    T* __restrict__ dx = (T*)a.y + base;
    constexpr int U = 4;
    for (int r = p.r; r < rows; r += U * t.rp) {
      Raw<T, V> rx[U], rd[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) {
          rx[k].load(x + (long)(r + k * t.rp) * a.C);
          rd[k].load(dy + (long)(r + k * t.rp) * a.C);
        }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * t.rp < rows) {
          float e[V], xh[V];
          grad_terms<T, V, VG, KIND>(a, rx[k], rd[k], mu, rs, ga, be, e, xh);
#pragma unroll
          for (int i = 0; i < V; ++i)
            e[i] = rs[i % VG] * (fmaf(ga[i], e[i], -sp[i % VG]) - xh[i] * sq[i % VG]);
          store_vec<T, V>(dx + (long)(r + k * t.rp) * a.C, e);
        }
    }
  }
}

// ------------------------------------------------------------------- host rules
// most vectors a thread holds (forward: x, backward: x and dy each), most threads
constexpr int KF = 16, KB = 8, NTMAX = 512;

enum How : int { ANY, RESIDENT, SPLIT, ROWS };

struct Plan {
  How how;
  int V, K;
  Tile t;       // resident, or the statistics pass of the split
  Tile apply;   // split: the apply pass
  int slabs;    // resident and any: slabs of channel sums of the backward
  long ws;      // floats
};

inline int pow2_floor(int v) {
  int p = 1;
  while (2 * p <= v) p *= 2;
  return p;
}

inline void finish(Tile& t, int V, int C, int cpg) {
  t.gb = t.cb / cpg;
  t.nblk = ceil_div(C, t.cb);
  t.fold = cpg % V == 0;
  t.glw = t.fold ? cpg / V : cpg;
  const int pairs = t.sp * t.gb;
  t.lp = pairs >= t.nt ? 1 : pow2_floor(t.nt / pairs);
  if (t.lp > 64) t.lp = 64;
  t.dcol = FastDiv(t.ncol);
  t.drp = FastDiv(t.rp);
  t.dglw = FastDiv(t.glw);
  t.dcpg = FastDiv(cpg);
  t.dgb = FastDiv(t.gb);
}

// The column block: whole groups, whole vectors, at least ``bytes`` of each row.
inline int column_block(int C, int cpg, int V, int esz, int bytes) {
  int unit = cpg;
  while (unit % V) unit += cpg;  // V is 8, 4, 2 or 1
  int cb = unit;
  while (cb * esz < bytes && cb < C) cb += unit;
  return cb < C ? cb : C;
}

inline Plan plan(int dtype, long N, long HW, int C, int G, int V, bool bwd) {
  const int esz = dtype == F32 ? 4 : 2, cpg = C / G;
  Plan p{};
  p.V = V;
  p.how = ANY;
  // slabs that fill the card, whatever the number of images (one 8192-wide group, 20000 bf16
  // rows: 1170 us; 1590 with 1024 workgroups, 1436 with a slab for each row)
  p.slabs = (int)(N < ceil_div(2048, G) ? N : ceil_div(2048, G));
  p.ws = bwd ? (long)p.slabs * 2 * C : 0;
  if (rows_take(dtype, N, HW, C, G, V)) {
    p.how = ROWS;
    p.ws = bwd ? rows_slabs(dtype, N, C, G, V) * 2 * C : 0;
    return p;
  }
  Tile& t = p.t;
  t.cb = column_block(C, cpg, V, esz, 128);
  t.ncol = t.cb / V;
  if (t.ncol > NTMAX) return p;
  // resident: the smallest workgroup whose registers hold an image's rows
  for (t.nt = 256; t.nt <= NTMAX; t.nt *= 2) {
    if (t.ncol > t.nt) continue;
    const int lanes = t.nt / t.ncol;
    if (HW > (long)lanes * (bwd ? KB : KF)) continue;
    // rows in parallel: all of them, or as many as leave no vector idle
    p.K = 2;
    while ((long)lanes * p.K < HW) p.K *= 2;
    t.rp = HW < lanes ? (int)HW : lanes;
    if (HW < lanes) p.K = 2;
    t.sp = lanes / t.rp;
    if (t.sp > N) t.sp = (int)N;
    t.nchunk = 1;
    t.rows = (int)HW;
    finish(t, V, C, cpg);
    while (t.sp * t.gb > t.nt) {
      --t.sp;
      finish(t, V, C, cpg);
    }
    if (t.sp < 1) return p;
    t.total = (long)ceil_div(N, t.sp) * t.nblk;
    p.how = RESIDENT;
    // a slab of channel sums per workgroup row: enough workgroups to fill the card
    const long per = t.total / t.nblk;
    const long most = ceil_div(2048, t.nblk);
    p.slabs = (int)(per < most ? per : most);
    p.ws = bwd ? (long)p.slabs * 2 * C : 0;
    return p;
  }
  // split
  t.cb = column_block(C, cpg, V, esz, 512);
  t.ncol = t.cb / V;
  t.nt = t.ncol > 256 ? 512 : 256;
  if (t.ncol > t.nt) return p;
  t.rp = t.nt / t.ncol;
  t.sp = 1;
  finish(t, V, C, cpg);
  if (t.gb > t.nt) return p;
  p.how = SPLIT;
  p.apply = t;
  p.K = 16;
  // workgroups that fill the card: fewer mean longer chunks and fewer partial
  // sums to merge (32 x 56 x 56 x 256, with channel sums merged by the apply pass:
  // 2048 of them took 41 us for y and 73 for dx; 1024, with group sums: 24 and 35)
  const long want = 1024;
  // forward statistics: chunks that fit the registers
  while (!bwd && p.K > 4 && N * t.nblk * ceil_div(HW, (long)t.rp * p.K) < want) p.K /= 2;
  long chunks = ceil_div(want, N * t.nblk);
  const long least = ceil_div(HW, 4l * t.rp);  // at least 4 vectors a thread
  if (chunks > least) chunks = least;
  auto set = [&](Tile& u, long rows) {
    u.rows = (int)rows;
    u.nchunk = ceil_div(HW, rows);
    u.total = N * u.nchunk * u.nblk;
  };
  set(t, bwd ? ceil_div(HW, chunks) : (long)t.rp * p.K);
  set(p.apply, ceil_div(HW, chunks));
  p.ws = bwd ? N * t.nchunk * (2 * C + 2 * G) : N * t.nchunk * G * 2;
  return p;
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

namespace kfb {
namespace gn {

// a launch holds fewer than 2^32 threads: the workgroups loop over the rest
inline dim3 tiles_grid(const Tile& t) { return dim3((unsigned)(t.total < (1l << 21) ? t.total : 1l << 21)); }

inline bool bad(long N, long HW, int C, int G) {
  return N <= 0 || HW <= 0 || C <= 0 || G <= 0 || C % G || HW > INT32_MAX;
}

// widest vector that C and the addresses (joined by or) allow: 16 bytes, 4 bytes or one value
inline int vec(int dtype, int C, uintptr_t at) {
  const int esz = dtype == F32 ? 4 : 2;
  if (C % (16 / esz) == 0 && at % 16 == 0) return 16 / esz;
  return esz == 2 && C % 2 == 0 && at % 4 == 0 ? 2 : 1;
}

}  // namespace gn
}  // namespace kfb

#define KFB_GN_VEC(T, v, fold, V, VG, ...)                                            \
  if (v > 2) {                                                                        \
    constexpr int V = 16 / sizeof(T);                                                 \
    if (fold) { constexpr int VG = 1; __VA_ARGS__; }                                   \
    else { constexpr int VG = V; __VA_ARGS__; }                                        \
  } else if (v == 2 && sizeof(T) == 2) {                                              \
    constexpr int V = 2;                                                              \
    if (fold) { constexpr int VG = 1; __VA_ARGS__; }                                   \
    else { constexpr int VG = V; __VA_ARGS__; }                                        \
  } else { constexpr int V = 1, VG = 1; __VA_ARGS__; }

#define KFB_GN_K(k, K, ...)                               \
  switch (k) {                                            \
    case 2: { constexpr int K = 2; __VA_ARGS__; break; }  \
    case 4: { constexpr int K = 4; __VA_ARGS__; break; }  \
    case 8: { constexpr int K = 8; __VA_ARGS__; break; }  \
    default: { constexpr int K = 16; __VA_ARGS__; break; } \
  }

// Workspace (floats) of the forward and of the backward; at: the tensors' addresses joined
// by or, of which the last four bits count.
KFB_API long kfb_gn_fwd_ws(int dtype, long N, long HW, int C, int G, int at) {
  return gn::bad(N, HW, C, G) ? 0 : gn::plan(dtype, N, HW, C, G, gn::vec(dtype, C, at & 15), false).ws;
}

KFB_API long kfb_gn_bwd_ws(int dtype, long N, long HW, int C, int G, int at) {
  return gn::bad(N, HW, C, G) ? 0 : gn::plan(dtype, N, HW, C, G, gn::vec(dtype, C, at & 15), true).ws;
}

KFB_API hipError_t kfb_gn_fwd(int dtype, const void* x, void* y, long N, long HW, int C, int G,
                              const float* gamma, const float* beta, float eps, int act,
                              float* mean, float* rstd, float* ws, hipStream_t stream) {
  if (gn::bad(N, HW, C, G)) return hipErrorInvalidValue;
  gn::Args a{x, nullptr, y, gamma, beta, mean, rstd, nullptr, N, HW, C, G, C / G, eps, act_of(act)};
  const gn::Plan p = gn::plan(dtype, N, HW, C, G, gn::vec(dtype, C, (uintptr_t)x | (uintptr_t)y), false);
  if (p.how == gn::ROWS) return gn::rows_fwd(dtype, a, p.V, stream);
  KFB_DISPATCH_DTYPE(dtype, T, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    if (p.how == gn::ANY) {
      hipLaunchKernelGGL((gn::gn_fwd_any_k<T, KIND>), gn::groups_grid(N, G), dim3(gn::NT), 0, stream, a,
                         gn::columns(C / G));
    } else {
      KFB_GN_VEC(T, p.V, p.t.fold, V, VG, {
        const size_t shm = sizeof(float) * ((size_t)p.t.sp * p.t.gb + (size_t)p.t.nt * VG);
        float2* part = p.how == gn::SPLIT ? (float2*)ws : nullptr;
        KFB_GN_K(p.K, K, {
          hipLaunchKernelGGL((gn::gn_fwd_tile_k<T, V, VG, KIND, K>), gn::tiles_grid(p.t),
                             dim3(p.t.nt), shm, stream, a, p.t, part);
        });
        if (part)
          hipLaunchKernelGGL((gn::gn_apply_k<T, V, VG, KIND>), gn::tiles_grid(p.apply),
                             dim3(p.apply.nt), 2 * sizeof(float) * p.apply.gb, stream, a, p.apply,
                             part, p.t.nchunk, p.t.rows);
      });
    }
  }));
  return hipGetLastError();
}

KFB_API hipError_t kfb_gn_bwd(int dtype, const void* dy, const void* x, void* dx, long N, long HW,
                              int C, int G, const float* gamma, const float* beta, int act,
                              const float* mean, const float* rstd, float* dgamma, float* dbeta,
                              int acc_gamma, int acc_beta, float* ws, hipStream_t stream) {
  if (gn::bad(N, HW, C, G) || !ws) return hipErrorInvalidValue;
  gn::Args a{x, dy, dx, gamma, beta, (float*)mean, (float*)rstd, ws, N, HW, C, G, C / G, 0.f, act_of(act)};
  const gn::Plan p = gn::plan(dtype, N, HW, C, G, gn::vec(dtype, C, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx), true);
  gn::ParamGrad q{ws, dgamma, dbeta, N, C, acc_gamma, acc_beta, ceil_div(2 * C, 16)};
  const bool params = dgamma || dbeta;
  bool done = false;
  if (p.how == gn::ROWS) {
    q.S = gn::rows_slabs(dtype, N, C, G, p.V);
    const hipError_t err = gn::rows_bwd(dtype, a, p.V, stream);
    if (err != hipSuccess) return err;
  } else
  KFB_DISPATCH_DTYPE(dtype, T, KFB_DISPATCH_ACT(a.act.kind, KIND, {
    if (p.how == gn::ANY) {
      q.S = p.slabs;
      hipLaunchKernelGGL((gn::gn_bwd_any_k<T, KIND>), dim3((unsigned)p.slabs * G), dim3(gn::NT), 0,
                         stream, a, gn::columns(C / G), p.slabs);
    } else {
      KFB_GN_VEC(T, p.V, p.t.fold, V, VG, {
        const size_t buf = sizeof(float) * ((size_t)p.t.nt * V + 2 * (size_t)p.t.sp * p.t.gb);
        if (p.how == gn::RESIDENT) {
          q.S = p.slabs;
          KFB_GN_K(p.K, K, {
            if constexpr (K <= gn::KB)
              hipLaunchKernelGGL((gn::gn_bwd_tile_k<T, V, VG, KIND, K>),
                                 dim3((unsigned)(p.slabs * p.t.nblk)), dim3(p.t.nt), buf, stream, a,
                                 p.t);
          });
        } else {
          q.S = N * p.t.nchunk;
          float2* gpart = (float2*)(ws + q.S * 2 * C);
          hipLaunchKernelGGL((gn::gn_bwd_sums_k<T, V, VG, KIND>), gn::tiles_grid(p.t), dim3(p.t.nt),
                             buf, stream, a, p.t, gpart);
          if (!params) q.blocks = 0;
          dim3 grid = gn::tiles_grid(p.apply);
          grid.x += q.blocks;
          size_t shm = 2 * sizeof(float) * (size_t)p.apply.gb;
          if (shm < sizeof(float) * p.apply.nt) shm = sizeof(float) * p.apply.nt;
          hipLaunchKernelGGL((gn::gn_bwd_apply_k<T, V, VG, KIND>), grid, dim3(p.apply.nt), shm, stream,
                             a, p.apply, gpart, p.t.nchunk, q);
          done = true;
        }
      });
    }
  }));
  if (params && !done)
    hipLaunchKernelGGL(gn::gn_param_grad_k, dim3(q.blocks), dim3(1024), 0, stream, q);
  return hipGetLastError();
}
