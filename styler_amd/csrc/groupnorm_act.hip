// Group norm over channels-last rows with an activation, forward and backward: any number of groups, none / ReLU / SiLU / GELU,
// statistics over an item's valid rows.
//
//   group (b, g): n = len[b] * C / G values;  xh = (x - mean) rstd,  z = xh gamma + beta,  y = act(z);  rows >= len[b] give 0
//   backward: dz = dy act'(z);  dbeta = sum dz, dgamma = sum dz xh;  with d = dz gamma and the group's means m1 = mean d,
//   m2 = mean d xh:  dx = rstd (d - m1 - xh m2)
//
// Two forms (kernel times of a trace).  8 x 16384 x 512 fp32, split: 62 + 8 + 85 us forward, 117 + 7 + 136 backward, bound by memory, 5.1
// TB/s over what the two passes move.  16 x 1000 x 320 bf16, fused: 11 us forward, 15 + 2 to 4 backward, one generation of 160 blocks: 96
// CUs have none, and on the others the vector unit is busy 0.62 and 0.76 of the time.
//   * fused: a block owns a slab of whole groups of one item and keeps its values in registers between the statistics and the
//     output, so x (and dy) is read once;
//   * split (items too long for that, or too few of them): row chunks leave per-channel sums, a small launch joins them per
//     group, a third writes the output.  x is read twice.
// Statistics: a thread sums (x - K) and (x - K)^2 of its channel, K = the mean of two of the chunk's rows -- a channel's offset, which
// may be large against its spread, is gone before the squares are formed; (count, mean, M2) triples are then joined pairwise exactly.
// (One row three deviations out would have nine tenths of the squares' sum cancel; four rows cost 0.3 us of 10.7.)
// Values enter as (x - mean), not folded into a multiply-add with -mean rstd: where a group hardly varies rstd is large, and the
// folded form keeps the rounding of mean rstd.  Everything is summed in a fixed order in 32 bits; there are no atomics.
#include "common.h"

namespace {

struct GArgs {
  const void *x, *dy;
  void* out;                                             // y or dx
  const float *gamma, *beta;
  float* stats;                                          // [B, G, 2] mean, rstd
  float *ws, *pw;                                        // chunk sums [B, chunks, C, 2]; item sums [B, C, 2] (backward)
  float *dgamma, *dbeta;
  const int64_t* len;
  int64_t xb, xl, db, dl, ob, ol;                        // item and row strides of x, dy, out
  int B, L, C, G, cg, chunks, rows, slab, slabs;         // rows: rows per chunk; slab: channels per block
  float eps;
};

// The kernels would be bound by their instructions with the library's erff and divisions (67 M values in 90 us leave 52
// instructions a value): one v_exp_f32 and one v_rcp_f32 a value instead.
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
// Phi(z) = (1 + erf(z / sqrt 2)) / 2, and e = exp(-z^2 / 2).  For z <= 0, Phi = e h(|z|) with h = erfcx / 2 as a polynomial in
// t = 1 / (1 + p |z| / sqrt 2) (the form of Hastings' approximations; coefficients fitted here to erfcx over [0, inf) in the
// norm max |exp(-x^2) err|: 2.6e-9), for z > 0, 1 - that.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.32f * 0.70710678118654752f, fabsf(z), 1.f));
  e = __builtin_amdgcn_exp2f(-0.72134752044448170f * (z * z));
  float h = 0.5f * -0.16305777512551112f;
  h = fmaf(h, t, 0.5f * 0.6326713090095979f);
  h = fmaf(h, t, 0.5f * -0.6115301283036071f);
  h = fmaf(h, t, 0.5f * 0.6121517059588323f);
  h = fmaf(h, t, 0.5f * -0.04181075739763211f);
  h = fmaf(h, t, 0.5f * 0.21519066395074074f);
  h = fmaf(h, t, 0.5f * 0.1756557856457516f);
  h = fmaf(h, t, 0.5f * 0.18072919626182787f);
  h *= t * e;
  return z > 0.f ? 1.f - h : h;
}
template <int ACT> __device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == STYLER_ACT_RELU) return z < 0.f ? 0.f : z;        // (a maximum would turn NaN into 0)
  if constexpr (ACT == STYLER_ACT_SILU) return z * sigmoid(z);
  if constexpr (ACT == STYLER_ACT_GELU) { float e; return z * normal_cdf(z, e); }
  return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == STYLER_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == STYLER_ACT_SILU) {
    const float t = sigmoid(z);
    return fmaf(z * t, 1.f - t, t);
  }
  if constexpr (ACT == STYLER_ACT_GELU) { float e; const float c = normal_cdf(z, e); return fmaf(z * 0.3989422804014327f, e, c); }
  return 1.f;
}

template <bool B16, int V> __device__ __forceinline__ void put(void* base, int64_t idx, const float (&f)[V]) {
  Raw<B16, V> r;
  r.set(f);
  r.store(base, idx);
}

// K of each channel: the mean of two of the n rows (0 of none), the same for all of a column's threads
template <bool B16, int V> __device__ __forceinline__ void shift_of(float (&K)[V], const void* x, int64_t at, int64_t ld, int n) {
  Raw<B16, V> k[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (n > 0) k[i].load(x, at + (i ? n / 2 : 0) * ld); else k[i].zero();
  }
#pragma unroll
  for (int j = 0; j < V; ++j) K[j] = 0.5f * k[0].get(j) + 0.5f * k[1].get(j);
}

// Sum over the lanes of a wave that hold the same column: lane & (cv - 1), cv a power of two up to 64.  The xor steps 32, 16 are
// half and row swaps, 8, 4, 2, 1 rotations and permutations inside sixteen lanes (all lanes agree modulo the steps done).
__device__ __forceinline__ float same_column_sum(float v, int cv) {
  if (cv <= 32) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  }
  if (cv <= 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (cv <= 8) v += dpp_f32<0x128>(v);
  if (cv <= 4) v += dpp_f32<0x124>(v);
  if (cv <= 2) v += dpp_f32<0x4E>(v);
  if (cv <= 1) v += dpp_f32<0xB1>(v);
  return v;
}
// Sums over the block's rl row lanes (thread = row lane * cv + column): column sums of a in sa, of b in sb [cv * V] on return.
// red: T * V floats.
template <int V, int T>
__device__ __forceinline__ void col_sums(const float (&a)[V], const float (&b)[V], float* red, float* sa, float* sb, int cv, int rl, bool on) {
  const int tid = threadIdx.x, W = cv * V;
  if (cv <= 32 && (cv & (cv - 1)) == 0) {                // columns repeat inside a wave: one partial row per wave
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = same_column_sum(a[i], cv), y = same_column_sum(b[i], cv);
      if (lane < cv) {
        red[wave * 2 * W + lane * V + i] = x;
        red[wave * 2 * W + W + lane * V + i] = y;
      }
    }
    __syncthreads();
    for (int c = tid; c < 2 * W; c += T) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < T / 64; ++w) x += red[w * 2 * W + c];
      (c < W ? sa : sb)[c < W ? c : c - W] = x;
    }
    __syncthreads();
    return;
  }
  // one array after the other; two steps each: partial sums of about sqrt(rl) rows (at most T / W a channel), then those.  (As many
  // partial sums as threads, added one after the other, are 204 terms for five channels: rstd was off by up to 1.9e-6.)
  int parts = 1;
  while (parts * parts < rl) ++parts;
  parts = max(1, min(parts, T / W));
  const int per = (rl + parts - 1) / parts;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if (on) {
      float* r = red + tid / cv * W + tid % cv * V;
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = q ? b[i] : a[i];
    }
    __syncthreads();
    if (parts > 1) {
      for (int j = tid; j < W * parts; j += T) {         // a (channel, part) pair is one thread's
        const int c = j % W, p = j / W;
        float x = 0.f;
        for (int r = p * per; r < min(rl, (p + 1) * per); ++r) x += red[r * W + c];
        if (p * per < rl) red[p * per * W + c] = x;      // the first of this thread's own rows
      }
      __syncthreads();
    }
    for (int c = tid; c < W; c += T) {
      float x = 0.f;
      for (int r = 0; r < rl; r += parts > 1 ? per : 1) x += red[r * W + c];
      (q ? sb : sa)[c] = x;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------------- fused
// Thread = (row lane, column of V channels); it holds rows rl, rl + RL, ... (at most IT) in registers.  The slabs of an item run
// on one XCD: their rows share memory lines where a slab is narrower than a line.
template <bool B16, int V, int ACT, int IT, int T, bool BWD>
__global__ __launch_bounds__(T) void gn_slab_kernel(GArgs a) {
  extern __shared__ float sh[];
  const int nx = blockIdx.x >> 3, b = nx / a.slabs * 8 + (blockIdx.x & 7);
  if (b >= a.B) return;
  const int c0 = nx % a.slabs * a.slab, tid = threadIdx.x, lane = tid & 63;
  const int W = min(a.slab, a.C - c0), cv = W / V, RL = T / cv, rl = tid / cv, col = tid - rl * cv;
  const bool on = rl < RL;
  const int n = clamp_len(a.len, b, a.L), c = c0 + col * V;
  float* red = sh;                                       // max(T V, slab)
  float* sa = sh + max(T * V, a.slab);                   // slab each
  float* sb = sa + a.slab;
  float* sk = sb + a.slab;
  float* gm = sk + a.slab;                               // 2 * groups of the slab
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
  float s[V], q[V];
  const int ng = W / a.cg, gl0 = c0 / a.cg;
  if constexpr (!BWD) {
    float K[V];
    shift_of<B16, V>(K, a.x, x0, a.xl, on ? n : 0);
#pragma unroll
    for (int j = 0; j < V; ++j) { s[j] = 0.f; q[j] = 0.f; }
    if (tid < cv) {                                      // (row lane 0)
#pragma unroll
      for (int j = 0; j < V; ++j) sk[tid * V + j] = K[j];
    }
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (on && rl + i * RL < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) { const float d = xr[i].get(j) - K[j]; s[j] += d; q[j] = fmaf(d, d, q[j]); }
      }
    col_sums<V, T>(s, q, red, sa, sb, cv, RL, on);
    // a wave per group: channel c has mean K + s / n and M2 = q - s^2 / n; all its channels have n values
    const float fn = (float)n;
    for (int g = tid >> 6; g < ng; g += T / 64) {
      float m = 0.f, m2 = 0.f;
      for (int j = g * a.cg + lane; j < (g + 1) * a.cg; j += 64) m += n > 0 ? sk[j] + sa[j] / fn : 0.f;
      const float mean = wave_sum(m) / (float)a.cg;
      for (int j = g * a.cg + lane; j < (g + 1) * a.cg; j += 64) {
        const float sm = n > 0 ? sa[j] / fn : 0.f, d = (sk[j] + sm) - mean;
        m2 += fmaxf(0.f, sb[j] - sa[j] * sm) + fn * d * d;
      }
      const float var = wave_sum(m2) / (fn * (float)a.cg), rstd = n > 0 ? 1.f / sqrtf(var + a.eps) : 0.f;
      if (lane == 0) {
        gm[2 * g] = n > 0 ? mean : 0.f;
        gm[2 * g + 1] = rstd;
        if (a.stats) {
          float* st = a.stats + ((int64_t)b * a.G + gl0 + g) * 2;
          st[0] = n > 0 ? mean : 0.f;
          st[1] = rstd;
        }
      }
    }
    __syncthreads();
    if (!on) return;
    float A[V], Z[V], mean[V];                           // z = A (x - mean) + Z
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int g = (col * V + j) / a.cg;
      mean[j] = gm[2 * g];
      A[j] = gm[2 * g + 1] * a.gamma[c + j];
      Z[j] = a.beta[c + j];
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = rl + i * RL;
      if (t >= a.L) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = t < n ? act_of<ACT>(fmaf(xr[i].get(j) - mean[j], A[j], Z[j])) : 0.f;
      put<B16, V>(a.out, o0 + t * a.ol, y);
    }
  } else {
    float ga[V], be[V], R[V], S[V];                      // xh = R (x - S)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float* st = a.stats + ((int64_t)b * a.G + (on ? (c + j) / a.cg : 0)) * 2;
      ga[j] = on ? a.gamma[c + j] : 0.f;
      be[j] = on ? a.beta[c + j] : 0.f;
      R[j] = st[1];
      S[j] = st[0];
      s[j] = 0.f;
      q[j] = 0.f;
    }
    float dz[IT][V];                                     // kept for the output: formed again there, 18.1 us instead of 16.2 (16 x 1000 x 320)
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (on && rl + i * RL < n) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = (xr[i].get(j) - S[j]) * R[j];
          dz[i][j] = gr[i].get(j) * act_slope<ACT>(fmaf(xh, ga[j], be[j]));
          s[j] += dz[i][j];
          q[j] = fmaf(dz[i][j], xh, q[j]);
        }
      }
    col_sums<V, T>(s, q, red, sa, sb, cv, RL, on);
    for (int j = tid; j < W; j += T)                     // this item's share of the parameter gradients
      *reinterpret_cast<float2*>(a.pw + ((int64_t)b * a.C + c0 + j) * 2) = make_float2(sa[j], sb[j]);
    const float count = (float)max(n, 1) * (float)a.cg;
    for (int g = tid >> 6; g < ng; g += T / 64) {
      float m1 = 0.f, m2 = 0.f;
      for (int j = g * a.cg + lane; j < (g + 1) * a.cg; j += 64) { m1 = fmaf(sa[j], a.gamma[c0 + j], m1); m2 = fmaf(sb[j], a.gamma[c0 + j], m2); }
      m1 = wave_sum(m1);
      m2 = wave_sum(m2);
      if (lane == 0) { gm[2 * g] = m1 / count; gm[2 * g + 1] = m2 / count; }
    }
    __syncthreads();
    if (!on) return;
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) { const int g = (col * V + j) / a.cg; m1[j] = gm[2 * g]; m2[j] = gm[2 * g + 1]; }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = rl + i * RL;
      if (t >= a.L) break;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (xr[i].get(j) - S[j]) * R[j];
        y[j] = t < n ? R[j] * (mul_rounded(dz[i][j], ga[j]) - m1[j] - xh * m2[j]) : 0.f;
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
  const int n = clamp_len(a.len, b, a.L), t0 = blockIdx.x * a.rows, t1 = min(n, t0 + a.rows);
  float* red = sh;
  float* sa = sh + T * V;
  float* sb = sa + a.slab;
  float* ws = a.ws + (((int64_t)b * a.chunks + blockIdx.x) * a.C + c0) * 2;
  if (t0 >= t1) return;                                  // (the joining launch skips chunks without rows)
  float s[V], q[V], K[V];
#pragma unroll
  for (int j = 0; j < V; ++j) { s[j] = 0.f; q[j] = 0.f; K[j] = 0.f; }
  const int64_t x0 = b * a.xb + c, g0 = b * a.db + c;
  if (on) {
    float ga[V], be[V], R[V], S[V];                      // xh = R (x - S)
    if constexpr (BWD) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float* st = a.stats + ((int64_t)b * a.G + (c + j) / a.cg) * 2;
        ga[j] = a.gamma[c + j];
        be[j] = a.beta[c + j];
        R[j] = st[1];
        S[j] = st[0];
      }
    } else {
      shift_of<B16, V>(K, a.x, x0 + t0 * a.xl, a.xl, t1 - t0);
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
            const float xh = (xr[u].get(j) - S[j]) * R[j];
            const float dz = gr[u].get(j) * act_slope<ACT>(fmaf(xh, ga[j], be[j]));
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

// Join the chunks of group (b, g): grid (G, B), a block per group, thread = (chunk lane, channel).  Forward, from (mean, M2) of
// n_i rows each: mean = sum n_i mean_i / N, then M2 = sum M2_i + n_i (mean_i - mean)^2 -> stats.  Backward: the channels' sums
// over the chunks -> pw [B, C, 2], and the group's two means -> gw [B, G, 2].
__device__ __forceinline__ float block_sum256(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
template <bool BWD>
__global__ __launch_bounds__(256) void gn_join_kernel(GArgs a, float* gw, float* pw) {
  __shared__ float red[2][256];
  const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = clamp_len(a.len, b, a.L), live = (n + a.rows - 1) / a.rows;
  const int cl = min(a.cg, 256), RL = 256 / cl, r0 = tid / cl, c = tid - r0 * cl;
  const float* ws = a.ws + (int64_t)b * a.chunks * a.C * 2;
  const float count = (float)max(n, 1) * (float)a.cg;
  float x = 0.f, y = 0.f;
  for (int c0 = 0; c0 < a.cg; c0 += cl) {                // (one turn unless a group has more than 256 channels)
    const int ch = g * a.cg + c0 + c;
    const bool on = r0 < RL && c0 + c < a.cg;
    float sx = 0.f, sy = 0.f;
    if (on) {
#pragma unroll 8
      for (int i = r0; i < live; i += RL) {
        const float2 p = *reinterpret_cast<const float2*>(ws + ((int64_t)i * a.C + ch) * 2);
        if constexpr (BWD) { sx += p.x; sy += p.y; }
        else sx = fmaf((float)(min(n, (i + 1) * a.rows) - i * a.rows), p.x, sx);
      }
    }
    if constexpr (BWD) {
      __syncthreads();
      red[0][tid] = sx;
      red[1][tid] = sy;
      __syncthreads();
      if (tid < cl && on) {
        for (int r = 1; r < RL; ++r) { sx += red[0][r * cl + c]; sy += red[1][r * cl + c]; }
        *reinterpret_cast<float2*>(pw + ((int64_t)b * a.C + ch) * 2) = make_float2(sx, sy);
        x = fmaf(sx, a.gamma[ch], x);
        y = fmaf(sy, a.gamma[ch], y);
      }
    } else {
      x += sx;
    }
  }
  __syncthreads();
  x = block_sum256(x, red[0]) / count;
  if constexpr (BWD) {
    y = block_sum256(y, red[1]) / count;
  } else {
    for (int c0 = 0; c0 < a.cg; c0 += cl) {
      if (r0 >= RL || c0 + c >= a.cg) continue;
#pragma unroll 8
      for (int i = r0; i < live; i += RL) {
        const float2 p = *reinterpret_cast<const float2*>(ws + ((int64_t)i * a.C + g * a.cg + c0 + c) * 2);
        const float d = p.x - x;
        y += fmaf((float)(min(n, (i + 1) * a.rows) - i * a.rows), d * d, p.y);
      }
    }
    y = 1.f / sqrtf(block_sum256(y, red[1]) / count + a.eps);
  }
  if (tid == 0) {
    float* st = (BWD ? gw : a.stats) + ((int64_t)b * a.G + g) * 2;
    st[0] = n > 0 ? x : 0.f;
    st[1] = n > 0 ? y : 0.f;
  }
}

// Elementwise part.  grid (chunks, slabs, B), walked from the end: the rows that the sums read last are those that the memory-side
// cache still holds.
template <bool B16, int V, int ACT, bool BWD>
__global__ __launch_bounds__(256) void gn_write_kernel(GArgs a, const float* gw) {
  constexpr int T = 256;
  const int b = a.B - 1 - blockIdx.z, c0 = blockIdx.y * a.slab, tid = threadIdx.x;
  const int W = min(a.slab, a.C - c0), cv = W / V, RL = T / cv, rl = tid / cv, col = tid - rl * cv, c = c0 + col * V;
  if (rl >= RL) return;
  const int n = clamp_len(a.len, b, a.L), t0 = (a.chunks - 1 - (int)blockIdx.x) * a.rows, t1 = min(a.L, t0 + a.rows);
  float ga[V], be[V], R[V], S[V], m1[V], m2[V];          // h = R (x - S); forward: R includes gamma
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int64_t g = ((int64_t)b * a.G + (c + j) / a.cg) * 2;
    ga[j] = a.gamma[c + j];
    be[j] = a.beta[c + j];
    R[j] = BWD ? a.stats[g + 1] : a.stats[g + 1] * ga[j];
    S[j] = a.stats[g];
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
        const float x = xr[u].get(j) - S[j];
        if constexpr (BWD) {
          const float h = x * R[j];
          const float dz = gr[u].get(j) * act_slope<ACT>(fmaf(h, ga[j], be[j]));
          y[j] = r < n ? R[j] * (mul_rounded(dz, ga[j]) - m1[j] - h * m2[j]) : 0.f;
        } else {
          y[j] = r < n ? act_of<ACT>(fmaf(x, R[j], be[j])) : 0.f;
        }
      }
      put<B16, V>(a.out, o0 + (int64_t)r * a.ol, y);
    }
  }
}

// dgamma, dbeta: the items' channel sums pw [B, C, 2] added in order.
__global__ __launch_bounds__(256) void gn_params_kernel(GArgs a, const float* pw) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float x = 0.f, y = 0.f;
#pragma unroll 8
  for (int b = 0; b < a.B; ++b) {
    const float2 v = *reinterpret_cast<const float2*>(pw + ((int64_t)b * a.C + c) * 2);
    x += v.x;
    y += v.y;
  }
  a.dbeta[c] = x;
  a.dgamma[c] = y;
}

// ------------------------------------------------------------------------------------------------------------- host
int pow2_div(int64_t v, int cap) {
  int n = cap;
  while (n > 1 && v % n) n >>= 1;
  return n;
}
struct GPlan { bool fused; int v, slab, slabs, chunks, rows, it, T; };

int gcd(int a, int b) { while (b) { const int t = a % b; a = b; b = t; } return a; }

// rows a thread of 1024 holds without spilling (the backward keeps x as loaded and dz in 32 bits)
constexpr int it_max(bool b16, int v, bool bwd) { return bwd ? (b16 && v == 8 ? 4 : 8) : 16; }

GPlan gn_plan(int B, int L, int C, int G, int bf16, int v, bool bwd) {
  GPlan p = {};
  const int es = bf16 ? 2 : 4, cg = C / G;
  p.v = v;
  // fused: a slab is whole groups and whole pieces, a memory line (128 bytes) wide where that gives 128 blocks, else down to 32
  // bytes (the lines that slabs share are then shared in one XCD's cache).  16 x 1000 x 320 bf16, forward / backward: 80 blocks
  // 13.7 / 16.3 us, 160 blocks 10.7 / 16.2, 320 blocks 12.9 / 22.8.  Blocks of 256 threads first, several of which share a CU: 12 x
  // 300 x 768 bf16, 384 blocks of 256 9.5 / 14.1, 132 blocks of 1024 10.9 / 17.6
  const int64_t unit = (int64_t)cg / gcd(cg, v) * v;
  for (int T = 256; T <= 1024 && !p.fused; T *= 4)
    for (int line = 128; line >= 32 && !p.fused; line >>= 1) {
      int64_t slab = unit * ((line / es + unit - 1) / unit);
      if (slab > C) slab = C;
      const int64_t cv = slab / v, slabs = (C + slab - 1) / slab;
      if (line > 32 && B * slabs < 128 && slab > unit) continue;
      if (cv > T || slab > 1024) continue;
      const int64_t it = (L + T / cv - 1) / (T / cv);
      if (it <= (T == 256 ? 4 : it_max(bf16 != 0, v, bwd))) {
        p.fused = true;
        p.T = T;
        p.it = it <= 4 ? 4 : it <= 8 ? 8 : 16;
        p.slab = (int)slab;
        p.slabs = (int)slabs;
      }
    }
  if (p.fused) return p;
  const int wide = 256 * v;
  p.slab = C < wide ? C : wide;
  p.slabs = (C + p.slab - 1) / p.slab;
  // chunks: about 4096 blocks, at least 32 rows each (8 x 16384 x 512 fp32, both sums: 512 blocks 228 us, 1024 200, 2048 197, 4096 181)
  int64_t ch = (4096 + (int64_t)B * p.slabs - 1) / ((int64_t)B * p.slabs);
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
  if (x->L > (1 << 30) || !(x->eps >= 0.f)) return STYLER_EINVAL;
  if (x->G > 1 << 22 || (x->C + 63) / 64 > 65535) return STYLER_EINVAL;                  // (grids: 65535 slabs, 2^32 threads)
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
  a.chunks = p.chunks; a.rows = p.rows; a.slab = p.slab; a.slabs = p.slabs;
  return a;
}

template <bool B16, int V, int ACT, bool BWD>
void gn_launch(const GArgs& a, const GPlan& p, float* gw, hipStream_t st) {
  if (p.fused) {
    const int red = p.T * V > p.slab ? p.T * V : p.slab;
    const size_t lds = (size_t)(red + 5 * p.slab) * 4;     // 52 KB at most
    const dim3 grid((unsigned)((a.B + 7) / 8 * 8 * p.slabs));
#define SLAB(IT, T) hipLaunchKernelGGL((gn_slab_kernel<B16, V, ACT, IT, T, BWD>), grid, dim3(T), lds, st, a)
    if (p.T == 256) SLAB(4, 256);
    else if (p.it == 4) SLAB(4, 1024);
    else if (p.it == 8) { if constexpr (it_max(B16, V, BWD) >= 8) SLAB(8, 1024); }
    else if constexpr (it_max(B16, V, BWD) >= 16) SLAB(16, 1024);
#undef SLAB
    return;
  }
  const dim3 grid(p.chunks, p.slabs, a.B);
  const size_t lds = (size_t)(256 * V + 2 * p.slab) * 4;
  hipLaunchKernelGGL((gn_sums_kernel<B16, V, ACT, BWD>), grid, dim3(256), lds, st, a);
  hipLaunchKernelGGL((gn_join_kernel<BWD>), dim3(a.G, a.B), dim3(256), 0, st, a, gw, a.pw);
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
// as many items a launch as a grid holds: 65535 in y and z, 2^32 threads in x
template <bool BWD>
void gn_run(const GArgs& all, const GPlan& p, int bf16, int act, float* gw, hipStream_t st) {
  const int64_t es = bf16 ? 2 : 4, step = p.fused ? ((int64_t)1 << 31) / ((int64_t)p.T * p.slabs) : 65528;
  for (int64_t b0 = 0; b0 < all.B; b0 += step) {
    GArgs a = all;
    a.B = (int)(all.B - b0 < step ? all.B - b0 : step);
    a.x = (const char*)all.x + b0 * all.xb * es;
    a.out = (char*)all.out + b0 * all.ob * es;
    if (BWD) { a.dy = (const char*)all.dy + b0 * all.db * es; a.pw = all.pw + 2 * b0 * all.C; }
    if (all.stats) a.stats = all.stats + 2 * b0 * all.G;
    if (!p.fused) a.ws = all.ws + 2 * b0 * p.chunks * all.C;
    if (all.len) a.len = all.len + b0;
    gn_dispatch<BWD>(a, p, bf16, act, BWD ? gw + 2 * b0 * all.G : nullptr, st);
  }
}

}  // namespace

// The largest any vector width needs (the width depends on addresses, which the caller may not have yet): per-channel sums of
// every chunk, the group means and items' sums of the backward, and the forward's statistics where the caller keeps none.
extern "C" int64_t styler_groupnorm_act_workspace_bytes(int B, int L, int C, int G, int bf16, int bwd) {
  if (B < 1 || L < 1 || C < 1 || G < 1 || C % G) return 0;
  int64_t most = 0;
  for (int v = bf16 ? 8 : 4; v >= 1; v >>= 1) {
    if (C % v) continue;
    const GPlan p = gn_plan(B, L, C, G, bf16, v, bwd != 0);
    const int64_t n = p.fused ? 0 : (int64_t)B * p.chunks * C * 2;
    if (n > most) most = n;
  }
  if (bwd) most += (int64_t)B * C * 2;
  return most ? 4 * (most + 2 * (int64_t)B * G) : 0;
}

extern "C" int styler_groupnorm_act(const styler_gn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = gn_check(x, false)) return rc;
  const int64_t need = styler_groupnorm_act_workspace_bytes(x->B, x->L, x->C, x->G, x->bf16, 0);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return STYLER_EINVAL;
  const GPlan p = gn_plan(x->B, x->L, x->C, x->G, x->bf16, gn_vec(x, false), false);
  GArgs a = gn_args(x, p);
  if (!a.stats && !p.fused) a.stats = (float*)workspace;
  a.ws = workspace ? (float*)workspace + 2 * (int64_t)x->B * x->G : nullptr;
  gn_run<false>(a, p, x->bf16, x->act, nullptr, (hipStream_t)stream);
  return launch_status();
}

extern "C" int styler_groupnorm_act_bwd(const styler_gn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = gn_check(x, true)) return rc;
  if (!workspace || workspace_bytes < styler_groupnorm_act_workspace_bytes(x->B, x->L, x->C, x->G, x->bf16, 1) || ((uintptr_t)workspace & 15))
    return STYLER_EINVAL;
  const GPlan p = gn_plan(x->B, x->L, x->C, x->G, x->bf16, gn_vec(x, true), true);
  GArgs a = gn_args(x, p);
  a.pw = (float*)workspace + 2 * (int64_t)x->B * x->G;
  a.ws = a.pw + 2 * (int64_t)x->B * x->C;
  gn_run<true>(a, p, x->bf16, x->act, (float*)workspace, (hipStream_t)stream);
  hipLaunchKernelGGL(gn_params_kernel, dim3((x->C + 255) / 256), dim3(256), 0, (hipStream_t)stream, a, (const float*)a.pw);
  return launch_status();
}
