// Rotary positions: the i-th pair of a head's first `rot` features is turned by pos * freq_i and scaled by `gain`; features
// past `rot` pass through.
//
//   half layout:        pair i = (i, i + rot / 2)          (y_a, y_b) = gain (x_a cos - x_b sin, x_b cos + x_a sin)
//   interleaved layout: pair i = (2 i, 2 i + 1)            inverse (the gradient, dx from dy): sin -> -sin
//
// Angles.  pos * freq is formed in 64 bits, in turns, and reduced to (-1/2, 1/2] there: a position of 200 000 is 30 000 turns,
// of which 32 bits keep three decimals.  The reduced angle goes to sincospi in 32 bits (no further reduction is needed).  A
// block forms the angles of its rows once, in LDS, one thread each; then all its threads stream the rows' heads.
//
// Bound by memory: every element is read and written once, in 16-byte pieces where layout and alignment allow.  4 x 8192 x 32 x
// 128 bf16: 98 us, 5.5 TB/s; 16 x 1000 x 4 x 64 fp32: 7.8 us (4.2 TB/s, start and end included); 32 rows of 10 heads: 3.4 us.
#include "common.h"

namespace {

struct RArgs {
  const void* x;
  void* y;
  const double* freq;
  const void* pos;
  int64_t xb, xl, xh, yb, yl, yh, posb;
  int64_t rows;
  int L, H, rot, nrot, nslot, rpb;
  uint32_t mslot, mhead;                                 // magic numbers of nslot and H
  int pos_kind;                                          // 0: the row index, 1: int64, 2: fp32
  float gain, sign;
};

// i / d by a multiplication: m = floor(2^32 / d) + 1 is exact for i d < 2^32 (the host sees to it); d = 1 has m = 0
__device__ __forceinline__ uint32_t div_magic(uint32_t i, uint32_t m) { return m ? __umulhi(i, m) : i; }

constexpr int UNROLL = 4;                                // items whose loads are in flight together
// A block covers rpb rows (item, position).  An item is one slot of one head: V pairs (half layout; interleaved: the V / 2 pairs
// of V consecutive features), or V features that pass through.  V: elements per access (interleaved and V = 1: the two elements
// of a pair are read one by one, as the half layout's are).
template <bool B16, bool INTER, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RArgs a) {
  constexpr int NP = INTER ? (V + 1) / 2 : V;
  constexpr bool WHOLE = INTER && V > 1;                 // an access holds whole pairs
  extern __shared__ __attribute__((aligned(16))) char sh[];
  int64_t* from = reinterpret_cast<int64_t*>(sh);                        // [rpb] where the rows start in x and in y
  int64_t* to = from + a.rpb;
  float2* turns = reinterpret_cast<float2*>(to + a.rpb);                 // [rpb][rot / 2] (cos, sin), gain and sign applied
  const int64_t r0 = (int64_t)blockIdx.x * a.rpb;
  const int nrow = (int)min((int64_t)a.rpb, a.rows - r0), half = a.rot >> 1;
  for (int r = threadIdx.x; r < nrow; r += 256) {
    const uint32_t row = (uint32_t)(r0 + r), b = row / (uint32_t)a.L, l = row - b * a.L;
    from[r] = b * a.xb + l * a.xl;
    to[r] = b * a.yb + l * a.yl;
  }
  __syncthreads();
  const uint32_t total = (uint32_t)nrow * a.H * a.nslot;
  Raw<B16, V> u[UNROLL], w[WHOLE ? 1 : UNROLL];
  int64_t at[UNROLL];                                    // where the item's first element goes in y
  int tr[UNROLL];                                        // index of the item's first pair in turns, -1: passes through
  auto fetch = [&](uint32_t i0) {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const uint32_t i = min(i0 + k * 256, total - 1);
      const uint32_t rh = div_magic(i, a.mslot), slot = i - rh * a.nslot, r = div_magic(rh, a.mhead), h = rh - r * a.H;
      const bool turned = (int)slot < a.nrot;
      const int d = turned ? slot * (INTER && V == 1 ? 2 : V) : a.rot + (slot - a.nrot) * V;
      const int64_t x0 = from[r] + h * a.xh + d;
      at[k] = to[r] + h * a.yh + d;
      tr[k] = turned ? r * half + (INTER ? d / 2 : d) : -1;
      u[k].load(a.x, x0);
      if constexpr (!WHOLE) w[k].load(a.x, x0 + (turned ? (INTER ? 1 : half) : 0));
    }
  };
  if (threadIdx.x < total) fetch(threadIdx.x);           // in flight while the angles are formed
  for (int i = threadIdx.x; i < nrow * half; i += 256) {
    const int r = i / half, p = i - r * half;
    const uint32_t row = (uint32_t)(r0 + r), b = row / (uint32_t)a.L, l = row - b * a.L;
    double pos = (double)l;
    if (a.pos_kind == 1) pos = (double)reinterpret_cast<const int64_t*>(a.pos)[b * a.posb + l];
    else if (a.pos_kind == 2) pos = (double)reinterpret_cast<const float*>(a.pos)[b * a.posb + l];
    const double t = pos * (a.freq[p] * 0.15915494309189533577);         // turns (1 / 2 pi)
    float sn, cs;
    sincospif(2.f * (float)(t - __builtin_rint(t)), &sn, &cs);
    turns[i] = make_float2(cs * a.gain, sn * a.gain * a.sign);
  }
  __syncthreads();
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += 256 * UNROLL) {
    if (i0 >= 256 * UNROLL) fetch(i0);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (i0 + k * 256 >= total) break;
      if (tr[k] < 0) {
        u[k].store(a.y, at[k]);
        continue;
      }
      float2 t[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) t[j] = turns[tr[k] + j];
      float y[V];
      if constexpr (WHOLE) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const float p = u[k].get(2 * j), q = u[k].get(2 * j + 1);
          y[2 * j] = p * t[j].x - q * t[j].y;
          y[2 * j + 1] = q * t[j].x + p * t[j].y;
        }
        u[k].set(y);
        u[k].store(a.y, at[k]);
      } else {
        float z[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float p = u[k].get(j), q = w[k].get(j);
          y[j] = p * t[j].x - q * t[j].y;
          z[j] = q * t[j].x + p * t[j].y;
        }
        u[k].set(y);
        w[k].set(z);
        u[k].store(a.y, at[k]);
        w[k].store(a.y, at[k] + (INTER ? 1 : half));
      }
    }
  }
}

}  // namespace

extern "C" int styler_rotary(const styler_rotary_t* p, void* stream) {
  if (!p || !p->x || !p->y || !p->freqs || p->B < 1 || p->L < 1 || p->H < 1 || p->D < 2) return STYLER_EINVAL;
  const int rot = p->rot, H = p->H, D = p->D, es = p->bf16 ? 2 : 4;
  if (rot < 2 || rot > D || (rot & 1) || D > 8192) return STYLER_EINVAL;         // (a row's angles: 32 KB of LDS at most)
  if ((int64_t)p->B * p->L > 0x7fffffff) return STYLER_EINVAL;
  if (p->pos_kind < 0 || p->pos_kind > 2 || (p->pos_kind != 0 && !p->pos)) return STYLER_EINVAL;
  if (((uintptr_t)p->x | (uintptr_t)p->y) % es) return STYLER_EALIGN;
  const int64_t st[] = {p->xb, p->xl, p->xh, p->yb, p->yl, p->yh};
  const bool copy = rot < D && !(p->x == p->y && p->xb == p->yb && p->xl == p->yl && p->xh == p->yh);
  // elements per access: the widest of 16, 8, 4, 2 bytes that divides every offset a thread forms
  int v = 16 / es;
  auto ok = [&](int n) {
    if (((uintptr_t)p->x | (uintptr_t)p->y) % (n * es)) return false;
    for (int64_t s : st) if (s % n) return false;
    if (p->interleaved ? rot % n : (rot / 2) % n) return false;
    return !(copy && D % n);
  };
  while (v > 1 && !ok(v)) v >>= 1;
  RArgs a = {};
  a.x = p->x; a.y = p->y; a.freq = p->freqs; a.pos = p->pos; a.xb = p->xb; a.xl = p->xl; a.xh = p->xh; a.yb = p->yb; a.yl = p->yl;
  a.yh = p->yh; a.posb = p->posb; a.rows = (int64_t)p->B * p->L; a.L = p->L; a.H = H; a.rot = rot; a.pos_kind = p->pos_kind;
  a.gain = p->gain; a.sign = p->inverse ? -1.f : 1.f;
  a.nrot = p->interleaved && v > 1 ? rot / v : rot / 2 / v;
  a.nslot = a.nrot + (copy ? (D - rot) / v : 0);
  const int64_t per_row = (int64_t)H * a.nslot;
  if (per_row * (H > a.nslot ? H : a.nslot) >= (int64_t)1 << 31) return STYLER_EINVAL;
  a.mslot = a.nslot == 1 ? 0 : (uint32_t)(((uint64_t)1 << 32) / a.nslot) + 1;
  a.mhead = H == 1 ? 0 : (uint32_t)(((uint64_t)1 << 32) / H) + 1;
  // rows per block: four items a thread, angles within 32 KB, and not fewer blocks than fill the chip several times over
  int64_t rpb = 1024 / per_row;
  if (rpb * (rot / 2) > 4096) rpb = 4096 / (rot / 2);
  while (rpb > 1 && a.rows / rpb < 768) rpb >>= 1;
  if (rpb < 1) rpb = 1;
  a.rpb = (int)rpb;
  const int64_t blocks = (a.rows + rpb - 1) / rpb;
  if (blocks > 0xffffff) return STYLER_EINVAL;                             // (2^32 threads a launch; 512 items a block: 17 GB of bf16 pairs)
  const size_t lds = (size_t)rpb * (rot / 2 * 8 + 16);
  hipStream_t s = (hipStream_t)stream;
#define GO(B16, I, V) hipLaunchKernelGGL((rotary_kernel<B16, I, V>), dim3((unsigned)blocks), dim3(256), lds, s, a)
  if (p->bf16) {
    if (p->interleaved) { if (v == 8) GO(true, true, 8); else if (v == 4) GO(true, true, 4); else if (v == 2) GO(true, true, 2); else GO(true, true, 1); }
    else { if (v == 8) GO(true, false, 8); else if (v == 4) GO(true, false, 4); else if (v == 2) GO(true, false, 2); else GO(true, false, 1); }
  } else {
    if (p->interleaved) { if (v == 4) GO(false, true, 4); else if (v == 2) GO(false, true, 2); else GO(false, true, 1); }
    else { if (v == 4) GO(false, false, 4); else if (v == 2) GO(false, false, 2); else GO(false, false, 1); }
  }
#undef GO
  return launch_status();
}
