// Group norm over channels-last rows with an activation, forward and backward: any number of groups, none / ReLU / SiLU / GELU,
// statistics over an item's valid rows.
//
//   group (b, g): n = len[b] * C / G values;  xh = (x - mean) rstd,  z = xh gamma + beta,  y = act(z);  rows >= len[b] give 0
//   backward: dz = dy act'(z);  dbeta = sum dz, dgamma = sum dz xh;  with d = dz gamma and the group's means m1 = mean d,
//   m2 = mean d xh:  dx = rstd (d - m1 - xh m2)
//
// Bound by memory.  Two forms:
//   * fused: a block owns a slab of whole groups of one item and keeps its values in registers between the statistics and the
//     output, so x (and dy) is read once;
//   * split (items too long for that, or too few of them): row chunks leave per-channel sums, a small launch joins them per
//     group, a third writes the output.  x is read twice.
// Statistics: a thread sums (x - K) and (x - K)^2 of its channel, K = the chunk's first row -- a channel's offset, which may be
// large against its spread, is gone before the squares are formed; (count, mean, M2) triples are then joined pairwise exactly.
// Everything is summed in a fixed order in 32 bits; there are no atomics.
#include "common.h"

namespace {

struct GArgs {
  const void *x, *dy;
  void* out;                                             // y or dx
  const float *gamma, *beta;
  float* stats;                                          // [B, G, 2] mean, rstd
  float* ws;
  float *dgamma, *dbeta;
  const int64_t* len;
  int64_t xb, xl, db, dl, ob, ol;                        // item and row strides of x, dy, out
  int B, L, C, G, cg, chunks, rows, slab;                // rows: rows per chunk; slab: channels per block
  float eps;
};

__device__ __forceinline__ int gn_len(const int64_t* len, int b, int L) {
  if (!len) return L;
  const int64_t n = len[b];
  return n < 0 ? 0 : (n > L ? L : (int)n);
}

template <int ACT> __device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == STYLER_ACT_RELU) return fmaxf(z, 0.f);
  if constexpr (ACT == STYLER_ACT_SILU) return z / (1.f + __expf(-z));
  if constexpr (ACT == STYLER_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == STYLER_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == STYLER_ACT_SILU) {
    const float t = 1.f / (1.f + __expf(-z));
    return t * (1.f + z * (1.f - t));
  }
  if constexpr (ACT == STYLER_ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.3989422804014327f * __expf(-0.5f * z * z);
  return 1.f;
}

// V consecutive channels, kept as loaded
template <bool B16, int V> struct Raw {
  uint32_t w[B16 ? (V + 1) / 2 : V];
  __device__ __forceinline__ void load(const void* base, int64_t idx) {
    const char* p = reinterpret_cast<const char*>(base) + idx * (B16 ? 2 : 4);
    constexpr int BY = V * (B16 ? 2 : 4);
    if constexpr (BY == 16) { const uint4 u = *reinterpret_cast<const uint4*>(p); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
    else if constexpr (BY == 8) { const uint2 u = *reinterpret_cast<const uint2*>(p); w[0] = u.x; w[1] = u.y; }
    else if constexpr (BY == 4) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (B16 ? (V + 1) / 2 : V); ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (B16) return __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __uint_as_float(w[i]);
  }
};
template <bool B16, int V> __device__ __forceinline__ void put(void* base, int64_t idx, const float (&f)[V]) {
  char* p = reinterpret_cast<char*>(base) + idx * (B16 ? 2 : 4);
  constexpr int BY = V * (B16 ? 2 : 4);
  if constexpr (B16 && V == 1) *reinterpret_cast<uint16_t*>(p) = (uint16_t)f32_to_bf16_bits(f[0]);
  else {
    uint32_t w[BY / 4];
#pragma unroll
    for (int i = 0; i < BY / 4; ++i) w[i] = B16 ? cvt_pk_bf16_rne(f[(2 * i) % V], f[(2 * i + 1) % V]) : __float_as_uint(f[i % V]);
    if constexpr (BY == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (BY == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

// Sums over the block's rl row lanes (thread = row lane * cv + column): column sums of a in sa, of b in sb [cv * V] on return.
// red: T * V floats, used for a and then for b.  Two steps each: T / (cv * V) partial sums per channel, then those.
template <int V, int T>
__device__ __forceinline__ void col_sum(const float (&a)[V], float* red, float* sa, int cv, int rl, bool on) {
  const int tid = threadIdx.x, W = cv * V;
  if (on) {
    float* r = red + tid / cv * W + tid % cv * V;
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = a[i];
  }
  __syncthreads();
  const int parts = max(1, min(rl, T / W)), per = (rl + parts - 1) / parts;
  for (int j = tid; j < W * parts; j += T) {             // a (channel, part) pair is one thread's
    const int c = j % W, p = j / W;
    float x = 0.f;
    for (int r = p * per; r < min(rl, (p + 1) * per); ++r) x += red[r * W + c];
    if (p * per < rl) red[p * per * W + c] = x;          // the first of this thread's own rows
  }
  __syncthreads();
  for (int c = tid; c < W; c += T) {
    float x = 0.f;
    for (int r = 0; r < rl; r += per) x += red[r * W + c];
    sa[c] = x;
  }
  __syncthreads();
}
template <int V, int T>
__device__ __forceinline__ void col_sums(const float (&a)[V], const float (&b)[V], float* red, float* sa, float* sb, int cv, int rl, bool on) {
  col_sum<V, T>(a, red, sa, cv, rl, on);
  col_sum<V, T>(b, red, sb, cv, rl, on);
}

// join (n, mean, M2) of two sets
__device__ __forceinline__ void join(float& n, float& mean, float& m2, float n2, float mean2, float m22) {
  const float t = n + n2;
  if (n2 == 0.f) return;
  const float d = mean2 - mean, f = n2 / t;
  mean += d * f;
  m2 += m22 + d * d * n * f;
  n = t;
}

// ------------------------------------------------------------------------------------------------------------- fused
// grid (slabs, B).  Thread = (row lane, column of V channels); it holds rows rl, rl + RL, ... (at most IT) in registers.
template <bool B16, int V, int ACT, int IT, int T, bool BWD>
__global__ __launch_bounds__(T) void gn_slab_kernel(GArgs a) {
  extern __shared__ float sh[];
  const int b = blockIdx.y, c0 = blockIdx.x * a.slab, tid = threadIdx.x;
  const int W = min(a.slab, a.C - c0), cv = W / V, RL = T / cv, rl = tid / cv, col = tid - rl * cv;
  const bool on = rl < RL;
  const int n = gn_len(a.len, b, a.L), c = c0 + col * V;
  float* red = sh;                                       // max(T V, 2 slab)
  float* sa = sh + max(T * V, 2 * a.slab);               // slab
  float* sb = sa + a.slab;                               // slab
  float* gm = sb + a.slab;                               // 2 * groups of the slab
  Raw<B16, V> xr[IT], gr[BWD ? IT : 1];
  const int64_t x0 = b * a.xb + c, g0 = b * a.db + c, o0 = b * a.ob + c;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int t = rl + i * RL;
    if (on && t < n) {
      xr[i].load(a.x, x0 + t * a.xl);
      if constexpr (BWD) gr[i].load(a.dy, g0 + t * a.dl);
    } else {
      xr[i].zero();
      if constexpr (BWD) gr[i].zero();
    }
  }
  float s[V], q[V], K[V];
  const int ng = W / a.cg, gl0 = c0 / a.cg;
  if constexpr (!BWD) {
    Raw<B16, V> k0;
    if (on && n > 0) k0.load(a.x, x0); else k0.zero();
#pragma unroll
    for (int j = 0; j < V; ++j) { K[j] = k0.get(j); s[j] = 0.f; q[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (rl + i * RL < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) { const float d = xr[i].get(j) - K[j]; s[j] += d; q[j] = fmaf(d, d, q[j]); }
      }
    col_sums<V, T>(s, q, red, sa, sb, cv, RL, on);
    // channel c: mean = K + s / n, M2 = q - s^2 / n; the group's channels joined in order
    if (tid < cv) {                                      // (row lane 0 holds K of its channels)
#pragma unroll
      for (int j = 0; j < V; ++j) red[tid * V + j] = K[j];
    }
    __syncthreads();
    for (int g = tid; g < ng; g += T) {
      float N = 0.f, mean = 0.f, m2 = 0.f;
      const float fn = (float)n;
      if (n > 0)
        for (int j = g * a.cg; j < (g + 1) * a.cg; ++j) {
          const float sm = sa[j] / fn;
          join(N, mean, m2, fn, red[j] + sm, fmaxf(0.f, sb[j] - sa[j] * sm));
        }
      const float rstd = n > 0 ? rsqrtf(m2 / N + a.eps) : 0.f;
      gm[2 * g] = mean;
      gm[2 * g + 1] = rstd;
      if (a.stats) {
        float* st = a.stats + ((int64_t)b * a.G + gl0 + g) * 2;
        st[0] = mean;
        st[1] = rstd;
      }
    }
    __syncthreads();
  } else {
    for (int g = tid; g < ng; g += T) {
      const float* st = a.stats + ((int64_t)b * a.G + gl0 + g) * 2;
      gm[2 * g] = st[0];
      gm[2 * g + 1] = st[1];
    }
    __syncthreads();
  }
  if (!BWD && !on) return;
  float ga[V], be[V], mean[V], rstd[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int g = on ? (col * V + j) / a.cg : 0;
    ga[j] = on ? a.gamma[c + j] : 0.f;
    be[j] = on ? a.beta[c + j] : 0.f;
    mean[j] = gm[2 * g];
    rstd[j] = gm[2 * g + 1];
  }
  if constexpr (!BWD) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = rl + i * RL;
      if (t >= a.L) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = t < n ? act_of<ACT>((xr[i].get(j) - mean[j]) * rstd[j] * ga[j] + be[j]) : 0.f;
      put<B16, V>(a.out, o0 + t * a.ol, y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) { s[j] = 0.f; q[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (rl + i * RL < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = (xr[i].get(j) - mean[j]) * rstd[j];
          const float dz = gr[i].get(j) * act_slope<ACT>(xh * ga[j] + be[j]);
          s[j] += dz;
          q[j] = fmaf(dz, xh, q[j]);
        }
      }
    col_sums<V, T>(s, q, red, sa, sb, cv, RL, on);
    for (int j = tid; j < W; j += T) {                   // this item's share of the parameter gradients
      a.ws[((int64_t)b * a.C + c0 + j) * 2] = sa[j];
      a.ws[((int64_t)b * a.C + c0 + j) * 2 + 1] = sb[j];
    }
    for (int g = tid; g < ng; g += T) {
      float m1 = 0.f, m2 = 0.f;
      for (int j = g * a.cg; j < (g + 1) * a.cg; ++j) { m1 = fmaf(sa[j], a.gamma[c0 + j], m1); m2 = fmaf(sb[j], a.gamma[c0 + j], m2); }
      const float inv = n > 0 ? 1.f / ((float)n * a.cg) : 0.f;
      red[2 * g] = m1 * inv;
      red[2 * g + 1] = m2 * inv;
    }
    __syncthreads();
    if (!on) return;
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { const int g = (col * V + j) / a.cg; m1[j] = red[2 * g]; m2[j] = red[2 * g + 1]; }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = rl + i * RL;
      if (t >= a.L) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (xr[i].get(j) - mean[j]) * rstd[j];
        const float dz = gr[i].get(j) * act_slope<ACT>(xh * ga[j] + be[j]);
        y[j] = t < n ? rstd[j] * (dz * ga[j] - m1[j] - xh * m2[j]) : 0.f;
      }
      put<B16, V>(a.out, o0 + t * a.ol, y);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- split
// Per-channel sums of a chunk of rows.  grid (chunks, slabs, B); ws [B, chunks, C, 2]: forward (mean, M2), backward (sum dz, sum dz xh).
template <bool B16, int V, int ACT, bool BWD>
__global__ __launch_bounds__(256) void gn_sums_kernel(GArgs a) {
  extern __shared__ float sh[];
  constexpr int T = 256;
  const int b = blockIdx.z, c0 = blockIdx.y * a.slab, tid = threadIdx.x;
  const int W = min(a.slab, a.C - c0), cv = W / V, RL = T / cv, rl = tid / cv, col = tid - rl * cv, c = c0 + col * V;
  const bool on = rl < RL;
  const int n = gn_len(a.len, b, a.L), t0 = blockIdx.x * a.rows, t1 = min(n, t0 + a.rows);
  float* red = sh;
  float* sa = sh + T * V;
  float* sb = sa + a.slab;
  float* ws = a.ws + (((int64_t)b * a.chunks + blockIdx.x) * a.C + c0) * 2;
  if (t0 >= t1) {                                        // (the joining launch skips chunks without rows; the backward sums them)
    if (BWD) for (int j = tid; j < 2 * W; j += T) ws[j] = 0.f;
    return;
  }
  float s[V], q[V], K[V];
#pragma unroll
  for (int j = 0; j < V; ++j) { s[j] = 0.f; q[j] = 0.f; K[j] = 0.f; }
  const int64_t x0 = b * a.xb + c, g0 = b * a.db + c;
  if (on) {
    float ga[V], be[V], mean[V], rstd[V];
    if constexpr (BWD) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float* st = a.stats + ((int64_t)b * a.G + (c + j) / a.cg) * 2;
        ga[j] = a.gamma[c + j];
        be[j] = a.beta[c + j];
        mean[j] = st[0];
        rstd[j] = st[1];
      }
    } else {
      Raw<B16, V> k0;
      k0.load(a.x, x0 + t0 * a.xl);
#pragma unroll
      for (int j = 0; j < V; ++j) K[j] = k0.get(j);
    }
    constexpr int U = BWD ? 4 : 8;                       // rows in flight per thread
    for (int t = t0 + rl; t < t1; t += U * RL) {
      Raw<B16, V> xr[U], gr[BWD ? U : 1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = min(t + u * RL, t1 - 1);
        xr[u].load(a.x, x0 + r * a.xl);
        if constexpr (BWD) gr[u].load(a.dy, g0 + r * a.dl);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t + u * RL >= t1) break;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if constexpr (BWD) {
            const float xh = (xr[u].get(j) - mean[j]) * rstd[j];
            const float dz = gr[u].get(j) * act_slope<ACT>(xh * ga[j] + be[j]);
            s[j] += dz;
            q[j] = fmaf(dz, xh, q[j]);
          } else {
            const float d = xr[u].get(j) - K[j];
            s[j] += d;
            q[j] = fmaf(d, d, q[j]);
          }
        }
      }
    }
  }
  col_sums<V, T>(s, q, red, sa, sb, cv, RL, on);
  if constexpr (!BWD) {
    if (tid < cv) {
#pragma unroll
      for (int j = 0; j < V; ++j) red[tid * V + j] = K[j];
    }
    __syncthreads();
  }
  for (int j = tid; j < W; j += T) {
    if constexpr (BWD) {
      ws[2 * j] = sa[j];
      ws[2 * j + 1] = sb[j];
    } else {
      const float fn = (float)(t1 - t0), sm = sa[j] / fn;
      ws[2 * j] = red[j] + sm;
      ws[2 * j + 1] = fmaxf(0.f, sb[j] - sa[j] * sm);
    }
  }
}

// Join the chunks of group (b, g): grid (G, B), a block per group.  Forward: stats.  Backward: the group's two means -> gw [B, G, 2].
template <bool BWD>
__global__ __launch_bounds__(256) void gn_join_kernel(GArgs a, float* gw) {
  __shared__ float red[3][256];
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = gn_len(a.len, b, a.L);
  const int live = (n + a.rows - 1) / a.rows;
  float N = 0.f, x = 0.f, y = 0.f;
  for (int i = tid; i < live * a.cg; i += 256) {
    const int ch = i / a.cg, c = g * a.cg + i % a.cg;
    const float2 p = *reinterpret_cast<const float2*>(a.ws + (((int64_t)b * a.chunks + ch) * a.C + c) * 2);
    if constexpr (BWD) { x = fmaf(p.x, a.gamma[c], x); y = fmaf(p.y, a.gamma[c], y); }
    else join(N, x, y, (float)(min(n, (ch + 1) * a.rows) - ch * a.rows), p.x, p.y);
  }
  red[0][tid] = N; red[1][tid] = x; red[2][tid] = y;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) {
      if constexpr (BWD) { red[1][tid] += red[1][tid + o]; red[2][tid] += red[2][tid + o]; }
      else join(red[0][tid], red[1][tid], red[2][tid], red[0][tid + o], red[1][tid + o], red[2][tid + o]);
    }
    __syncthreads();
  }
  if (tid == 0) {
    float* st = (BWD ? gw : a.stats) + ((int64_t)b * a.G + g) * 2;
    if constexpr (BWD) {
      const float inv = n > 0 ? 1.f / ((float)n * a.cg) : 0.f;
      st[0] = red[1][0] * inv;
      st[1] = red[2][0] * inv;
    } else {
      st[0] = red[1][0];
      st[1] = n > 0 ? rsqrtf(red[2][0] / red[0][0] + a.eps) : 0.f;
    }
  }
}

// Elementwise part.  grid (chunks, slabs, B).
template <bool B16, int V, int ACT, bool BWD>
__global__ __launch_bounds__(256) void gn_write_kernel(GArgs a, const float* gw) {
  constexpr int T = 256;
  const int b = blockIdx.z, c0 = blockIdx.y * a.slab, tid = threadIdx.x;
  const int W = min(a.slab, a.C - c0), cv = W / V, RL = T / cv, rl = tid / cv, col = tid - rl * cv, c = c0 + col * V;
  if (rl >= RL) return;
  const int n = gn_len(a.len, b, a.L), t0 = blockIdx.x * a.rows, t1 = min(a.L, t0 + a.rows);
  float ga[V], be[V], mean[V], rstd[V], m1[V], m2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t g = ((int64_t)b * a.G + (c + j) / a.cg) * 2;
    ga[j] = a.gamma[c + j];
    be[j] = a.beta[c + j];
    mean[j] = a.stats[g];
    rstd[j] = a.stats[g + 1];
    if constexpr (BWD) { m1[j] = gw[g]; m2[j] = gw[g + 1]; }
  }
  const int64_t x0 = b * a.xb + c, g0 = b * a.db + c, o0 = b * a.ob + c;
  constexpr int U = 4;
  for (int t = t0 + rl; t < t1; t += U * RL) {
    Raw<B16, V> xr[U], gr[BWD ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = t + u * RL;
      if (r < n && r < t1) {
        xr[u].load(a.x, x0 + (int64_t)r * a.xl);
        if constexpr (BWD) gr[u].load(a.dy, g0 + (int64_t)r * a.dl);
      } else {
        xr[u].zero();
        if constexpr (BWD) gr[u].zero();
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = t + u * RL;
      if (r >= t1) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (xr[u].get(j) - mean[j]) * rstd[j];
        if constexpr (BWD) {
          const float dz = gr[u].get(j) * act_slope<ACT>(xh * ga[j] + be[j]);
          y[j] = r < n ? rstd[j] * (dz * ga[j] - m1[j] - xh * m2[j]) : 0.f;
        } else {
          y[j] = r < n ? act_of<ACT>(xh * ga[j] + be[j]) : 0.f;
        }
      }
      put<B16, V>(a.out, o0 + (int64_t)r * a.ol, y);
    }
  }
}

// dgamma, dbeta: the sums of `parts` rows of ws [parts, C, 2], a block per 32 channels (8 row lanes), in a fixed order.
__global__ __launch_bounds__(256) void gn_params_kernel(GArgs a, int64_t parts) {
  __shared__ float red[2][8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  float x = 0.f, y = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int64_t p = r; p < parts; p += 8) {
      const float2 v = *reinterpret_cast<const float2*>(a.ws + (p * a.C + c) * 2);
      x += v.x;
      y += v.y;
    }
  }
  red[0][r][threadIdx.x & 31] = x;
  red[1][r][threadIdx.x & 31] = y;
  __syncthreads();
  if (r == 0 && c < a.C) {
    for (int i = 1; i < 8; ++i) { x += red[0][i][threadIdx.x]; y += red[1][i][threadIdx.x]; }
    a.dbeta[c] = x;
    a.dgamma[c] = y;
  }
}

// ------------------------------------------------------------------------------------------------------------- host
int pow2_div(int64_t v, int cap) {
  int n = cap;
  while (n > 1 && v % n) n >>= 1;
  return n;
}
struct GPlan { bool fused; int v, slab, slabs, chunks, rows, it, T; };

int gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// bytes: of 16, what every row start and C divide; the plan depends on sizes alone besides it
GPlan gn_plan(int B, int L, int C, int G, int bf16, int v, bool bwd) {
  GPlan p = {};
  const int es = bf16 ? 2 : 4, cg = C / G;
  p.v = v;
  // fused: the narrowest slab of whole groups and whole pieces whose rows are >= 128 bytes (a memory line)
  const int64_t unit = (int64_t)cg / gcd(cg, v) * v;
  int64_t slab = unit * ((128 / es + unit - 1) / unit);
  if (slab > C) slab = C;
  const int64_t cv = slab / v;
  const int it_max = bwd ? 8 : 16;
  for (int T = 256; T <= 1024 && !p.fused; T *= 4) {
    if (cv > T || slab > 1024) continue;
    const int64_t it = (L + T / cv - 1) / (T / cv);
    if (it <= (T == 256 ? 4 : it_max)) {
      p.fused = true;
      p.T = T;
      p.it = it <= 4 ? 4 : it <= 8 ? 8 : 16;
    }
  }
  if (p.fused) {
    p.slab = (int)slab;
    p.slabs = (int)((C + slab - 1) / slab);
    return p;
  }
  const int wide = 256 * v;
  p.slab = C < wide ? C : wide;
  p.slabs = (C + p.slab - 1) / p.slab;
  // chunks: about 1024 blocks, at least 32 rows each
  int64_t ch = (1024 + (int64_t)B * p.slabs - 1) / ((int64_t)B * p.slabs);
  if (ch > (L + 31) / 32) ch = (L + 31) / 32;
  if (ch < 1) ch = 1;
  p.rows = (int)((L + ch - 1) / ch);
  p.chunks = (L + p.rows - 1) / p.rows;
  return p;
}
int gn_vec(const styler_gn_t* x, bool bwd) {
  const int es = x->bf16 ? 2 : 4;
  int v = pow2_div(x->C, 16 / es);
  const int64_t st[] = {x->xb, x->xl, x->ob, x->ol, bwd ? x->db : 0, bwd ? x->dl : 0};
  for (int64_t s : st) v = pow2_div(s, v);
  const uintptr_t p[] = {(uintptr_t)x->x, (uintptr_t)x->out, bwd ? (uintptr_t)x->dy : 0};
  for (uintptr_t q : p) v = pow2_div((int64_t)(q / es), v);
  return v;
}
int gn_check(const styler_gn_t* x, bool bwd) {
  if (!x || !x->x || !x->out || !x->gamma || !x->beta || x->B < 1 || x->L < 1 || x->C < 1 || x->G < 1 || x->C % x->G) return STYLER_EINVAL;
  if (x->B > 65535 || x->L > (1 << 30) || !(x->eps >= 0.f)) return STYLER_EINVAL;
  if (x->act != STYLER_ACT_NONE && x->act != STYLER_ACT_RELU && x->act != STYLER_ACT_SILU && x->act != STYLER_ACT_GELU) return STYLER_EINVAL;
  if (bwd && (!x->dy || !x->dgamma || !x->dbeta || !x->stats)) return STYLER_EINVAL;
  const uintptr_t es = x->bf16 ? 2 : 4;
  if ((uintptr_t)x->x % es || (uintptr_t)x->out % es || (uintptr_t)x->dy % es) return STYLER_EALIGN;
  return 0;
}
GArgs gn_args(const styler_gn_t* x, const GPlan& p) {
  GArgs a = {};
  a.x = x->x; a.dy = x->dy; a.out = x->out; a.gamma = x->gamma; a.beta = x->beta; a.stats = x->stats; a.dgamma = x->dgamma;
  a.dbeta = x->dbeta; a.len = x->len; a.xb = x->xb; a.xl = x->xl; a.db = x->db; a.dl = x->dl; a.ob = x->ob; a.ol = x->ol;
  a.B = x->B; a.L = x->L; a.C = x->C; a.G = x->G; a.cg = x->C / x->G; a.eps = x->eps;
  a.chunks = p.chunks; a.rows = p.rows; a.slab = p.slab;
  return a;
}

template <bool B16, int V, int ACT, bool BWD>
void gn_launch(const GArgs& a, const GPlan& p, float* gw, hipStream_t st) {
  if (p.fused) {
    const int red = p.T * V > 2 * p.slab ? p.T * V : 2 * p.slab;
    const size_t lds = (size_t)(red + 4 * p.slab) * 4;     // 56 KB at most
    const dim3 grid(p.slabs, a.B);
#define SLAB(IT, T) hipLaunchKernelGGL((gn_slab_kernel<B16, V, ACT, IT, T, BWD>), grid, dim3(T), lds, st, a)
    if (p.T == 256) SLAB(4, 256);
    else if (p.it == 4) SLAB(4, 1024);
    else if (p.it == 8) SLAB(8, 1024);
    else if constexpr (!BWD) SLAB(16, 1024);
#undef SLAB
    return;
  }
  const dim3 grid(p.chunks, p.slabs, a.B);
  const size_t lds = (size_t)(256 * V + 2 * p.slab) * 4;
  hipLaunchKernelGGL((gn_sums_kernel<B16, V, ACT, BWD>), grid, dim3(256), lds, st, a);
  hipLaunchKernelGGL((gn_join_kernel<BWD>), dim3(a.G, a.B), dim3(256), 0, st, a, gw);
  hipLaunchKernelGGL((gn_write_kernel<B16, V, ACT, BWD>), grid, dim3(256), 0, st, a, (const float*)gw);
}
template <bool B16, int V, bool BWD>
void gn_by_act(const GArgs& a, const GPlan& p, int act, float* gw, hipStream_t st) {
  if (act == STYLER_ACT_RELU) gn_launch<B16, V, STYLER_ACT_RELU, BWD>(a, p, gw, st);
  else if (act == STYLER_ACT_SILU) gn_launch<B16, V, STYLER_ACT_SILU, BWD>(a, p, gw, st);
  else if (act == STYLER_ACT_GELU) gn_launch<B16, V, STYLER_ACT_GELU, BWD>(a, p, gw, st);
  else gn_launch<B16, V, STYLER_ACT_NONE, BWD>(a, p, gw, st);
}
template <bool BWD>
void gn_dispatch(const GArgs& a, const GPlan& p, int bf16, int act, float* gw, hipStream_t st) {
  if (bf16) {
    if (p.v == 8) gn_by_act<true, 8, BWD>(a, p, act, gw, st);
    else if (p.v == 4) gn_by_act<true, 4, BWD>(a, p, act, gw, st);
    else if (p.v == 2) gn_by_act<true, 2, BWD>(a, p, act, gw, st);
    else gn_by_act<true, 1, BWD>(a, p, act, gw, st);
  } else {
    if (p.v == 4) gn_by_act<false, 4, BWD>(a, p, act, gw, st);
    else if (p.v == 2) gn_by_act<false, 2, BWD>(a, p, act, gw, st);
    else gn_by_act<false, 1, BWD>(a, p, act, gw, st);
  }
}

}  // namespace

// The largest any vector width needs (the width depends on addresses, which the caller may not have yet): per-channel sums of
// every chunk, the group means of the backward, and the forward's statistics where the caller keeps none.
extern "C" int64_t styler_groupnorm_act_workspace_bytes(int B, int L, int C, int G, int bf16, int bwd) {
  if (B < 1 || L < 1 || C < 1 || G < 1 || C % G) return 0;
  int64_t most = 0;
  for (int v = bf16 ? 8 : 4; v >= 1; v >>= 1) {
    if (C % v) continue;
    const GPlan p = gn_plan(B, L, C, G, bf16, v, bwd != 0);
    const int64_t n = p.fused ? (bwd ? (int64_t)B * C * 2 : 0) : (int64_t)B * p.chunks * C * 2;
    if (n > most) most = n;
  }
  return 4 * (most + 2 * (int64_t)B * G);
}

extern "C" int styler_groupnorm_act(const styler_gn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = gn_check(x, false)) return rc;
  if (!workspace || workspace_bytes < styler_groupnorm_act_workspace_bytes(x->B, x->L, x->C, x->G, x->bf16, 0) || ((uintptr_t)workspace & 15))
    return STYLER_EINVAL;
  const GPlan p = gn_plan(x->B, x->L, x->C, x->G, x->bf16, gn_vec(x, false), false);
  GArgs a = gn_args(x, p);
  if (!a.stats && !p.fused) a.stats = (float*)workspace;
  a.ws = (float*)workspace + 2 * (int64_t)x->B * x->G;
  gn_dispatch<false>(a, p, x->bf16, x->act, nullptr, (hipStream_t)stream);
  return launch_status();
}

extern "C" int styler_groupnorm_act_bwd(const styler_gn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = gn_check(x, true)) return rc;
  if (!workspace || workspace_bytes < styler_groupnorm_act_workspace_bytes(x->B, x->L, x->C, x->G, x->bf16, 1) || ((uintptr_t)workspace & 15))
    return STYLER_EINVAL;
  const GPlan p = gn_plan(x->B, x->L, x->C, x->G, x->bf16, gn_vec(x, true), true);
  GArgs a = gn_args(x, p);
  a.ws = (float*)workspace + 2 * (int64_t)x->B * x->G;
  gn_dispatch<true>(a, p, x->bf16, x->act, (float*)workspace, (hipStream_t)stream);
  hipLaunchKernelGGL(gn_params_kernel, dim3((x->C + 31) / 32), dim3(256), 0, (hipStream_t)stream, a,
                     (int64_t)x->B * (p.fused ? 1 : p.chunks));
  return launch_status();
}
