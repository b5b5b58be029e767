// Rotary positions: the i-th pair of a head's first `rot` features is turned by pos * freq_i and scaled by `gain`; features
// past `rot` pass through.
//
//   half layout:        pair i = (i, i + rot / 2)          (y_a, y_b) = gain (x_a cos - x_b sin, x_b cos + x_a sin)
//   interleaved layout: pair i = (2 i, 2 i + 1)            inverse (the gradient, dx from dy): sin -> -sin
//
// Angles.  pos * freq is formed in 64 bits, in turns, and reduced to (-1/2, 1/2] there: a position of 200 000 is 30 000 turns,
// of which 32 bits keep three decimals.  The reduced angle goes to sincospi in 32 bits (no further reduction is needed).  A
// thread computes the angles of its pairs once and applies them to several heads.
//
// Bound by memory: every element is read and written once, in 16-byte pieces where layout and alignment allow.
#include "common.h"

namespace {

struct RArgs {
  const void* x;
  void* y;
  const double* freq;
  const void* pos;
  int64_t xb, xl, xh, yb, yl, yh, posb;
  int64_t rows;
  int L, H, D, rot, hpt, tpr, nrot, nslot, rpb;
  int pos_kind;                                          // 0: the row index, 1: int64, 2: fp32
  float gain, sign;
};

template <int N> struct Piece;                           // N 32-bit words
template <> struct Piece<4> { typedef uint4 T; };
template <> struct Piece<2> { typedef uint2 T; };
template <> struct Piece<1> { typedef uint32_t T; };

// V consecutive elements of a bf16 or fp32 row
template <bool B16, int V> struct Vec {
  static constexpr int BYTES = V * (B16 ? 2 : 4);
  float f[V];
  __device__ __forceinline__ void load(const void* base, int64_t idx) {
    if constexpr (B16 && V == 1) {
      f[0] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(base)[idx] << 16);
    } else {
      typename Piece<BYTES / 4>::T raw = *reinterpret_cast<const typename Piece<BYTES / 4>::T*>(reinterpret_cast<const char*>(base) + idx * (B16 ? 2 : 4));
      uint32_t w[BYTES / 4];
      __builtin_memcpy(w, &raw, BYTES);
#pragma unroll
      for (int i = 0; i < V; ++i)
        f[i] = B16 ? __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) : __uint_as_float(w[i < BYTES / 4 ? i : 0]);
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t idx) const {
    if constexpr (B16 && V == 1) {
      reinterpret_cast<uint16_t*>(base)[idx] = (uint16_t)f32_to_bf16_bits(f[0]);
    } else {
      uint32_t w[BYTES / 4];
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) w[i] = B16 ? cvt_pk_bf16_rne(f[(2 * i) % V], f[(2 * i + 1) % V]) : __float_as_uint(f[i % V]);
      typename Piece<BYTES / 4>::T raw;
      __builtin_memcpy(&raw, w, BYTES);
      *reinterpret_cast<typename Piece<BYTES / 4>::T*>(reinterpret_cast<char*>(base) + idx * (B16 ? 2 : 4)) = raw;
    }
  }
};

__device__ __forceinline__ void turn(double pos, double freq, float gain, float sign, float& c, float& s) {
  const double t = pos * (freq * 0.15915494309189533577);      // turns (1 / 2 pi)
  const float r = (float)(t - __builtin_rint(t));
  float sn, cs;
  sincospif(2.f * r, &sn, &cs);
  c = cs * gain;
  s = sn * gain * sign;
}

constexpr int UNROLL = 4;                                // heads whose loads are in flight together
// A block covers rpb rows (item, position), tpr threads a row; a thread has one slot of the row -- V pairs (half layout) or V / 2
// pairs (interleaved), or V features that pass through -- in hpt heads.  V: elements per access (interleaved and V = 1: the two
// elements of a pair are read one by one, as the half layout's are).
template <bool B16, bool INTER, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RArgs a) {
  constexpr int NP = INTER ? (V + 1) / 2 : V;
  constexpr bool WHOLE = INTER && V > 1;                 // an access holds whole pairs
  const int rib = threadIdx.x / a.tpr;
  const int64_t row = (int64_t)blockIdx.x * a.rpb + rib;
  if (rib >= a.rpb || row >= a.rows) return;
  const int b = (int)(row / a.L), l = (int)(row - (int64_t)b * a.L);
  const int h0 = blockIdx.y * a.hpt, h1 = min(a.H, h0 + a.hpt);
  const int64_t x0 = b * a.xb + l * a.xl, y0 = b * a.yb + l * a.yl;
  double pos = (double)l;
  if (a.pos_kind == 1) pos = (double)reinterpret_cast<const int64_t*>(a.pos)[b * a.posb + l];
  else if (a.pos_kind == 2) pos = (double)reinterpret_cast<const float*>(a.pos)[b * a.posb + l];
  for (int slot = threadIdx.x - rib * a.tpr; slot < a.nslot; slot += a.tpr) {
    if (slot >= a.nrot) {                                // features past rot
      const int d = a.rot + (slot - a.nrot) * V;
      for (int h = h0; h < h1; ++h) {
        Vec<B16, V> u;
        u.load(a.x, x0 + h * a.xh + d);
        u.store(a.y, y0 + h * a.yh + d);
      }
      continue;
    }
    const int d = slot * (INTER && V == 1 ? 2 : V), e = INTER ? d + 1 : d + a.rot / 2;     // e: where the second elements start
    float c[NP], s[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) turn(pos, a.freq[(INTER ? d / 2 : d) + i], a.gain, a.sign, c[i], s[i]);
    for (int h = h0; h < h1; h += UNROLL) {
      Vec<B16, V> u[UNROLL], w[WHOLE ? 1 : UNROLL];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        const int64_t p = x0 + (h + k < h1 ? h + k : h1 - 1) * a.xh;
        u[k].load(a.x, p + d);
        if constexpr (!WHOLE) w[k].load(a.x, p + e);
      }
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        if (h + k >= h1) break;
        const int64_t p = y0 + (h + k) * a.yh;
        if constexpr (WHOLE) {
          Vec<B16, V> r;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            r.f[2 * i] = u[k].f[2 * i] * c[i] - u[k].f[2 * i + 1] * s[i];
            r.f[2 * i + 1] = u[k].f[2 * i + 1] * c[i] + u[k].f[2 * i] * s[i];
          }
          r.store(a.y, p + d);
        } else {
          Vec<B16, V> r, q;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            r.f[i] = u[k].f[i] * c[i] - w[k].f[i] * s[i];
            q.f[i] = w[k].f[i] * c[i] + u[k].f[i] * s[i];
          }
          r.store(a.y, p + d);
          q.store(a.y, p + e);
        }
      }
    }
  }
}

}  // namespace

extern "C" int styler_rotary(const void* x, int64_t xb, int64_t xl, int64_t xh, void* y, int64_t yb, int64_t yl, int64_t yh,
                             const double* freqs, const void* pos, int64_t posb, int pos_kind, int B, int L, int H, int D, int rot,
                             int interleaved, int inverse, float gain, int bf16, void* stream) {
  if (!x || !y || !freqs || B < 1 || L < 1 || H < 1 || D < 2 || rot < 2 || rot > D || (rot & 1)) return STYLER_EINVAL;
  if (pos_kind < 0 || pos_kind > 2 || (pos_kind != 0 && !pos)) return STYLER_EINVAL;
  if ((int64_t)B * L > 0x7fffffff) return STYLER_EINVAL;
  const int es = bf16 ? 2 : 4;
  if (((uintptr_t)x | (uintptr_t)y) % es) return STYLER_EALIGN;
  // elements per access: the widest of 16, 8, 4, 2 bytes that divides every offset a thread forms
  int v = 16 / es;
  const bool copy = !(x == y && xb == yb && xl == yl && xh == yh) && rot < D;
  auto ok = [&](int n) {
    const int64_t bytes = (int64_t)n * es;
    if (((uintptr_t)x | (uintptr_t)y) % bytes) return false;
    const int64_t st[] = {xb, xl, xh, yb, yl, yh};
    for (int64_t s : st) if (s % n) return false;
    if (interleaved ? rot % n : (rot / 2) % n) return false;
    return !(copy && D % n);
  };
  while (v > 1 && !ok(v)) v >>= 1;
  RArgs a = {};
  a.x = x; a.y = y; a.freq = freqs; a.pos = pos; a.xb = xb; a.xl = xl; a.xh = xh; a.yb = yb; a.yl = yl; a.yh = yh; a.posb = posb;
  a.rows = (int64_t)B * L; a.L = L; a.H = H; a.D = D; a.rot = rot; a.pos_kind = pos_kind; a.gain = gain; a.sign = inverse ? -1.f : 1.f;
  a.nrot = interleaved && v > 1 ? rot / v : rot / 2 / v;
  a.nslot = a.nrot + (copy ? (D - rot) / v : 0);
  a.tpr = a.nslot < 256 ? a.nslot : 256;
  a.rpb = 256 / a.tpr;
  const int64_t blocks = (a.rows + a.rpb - 1) / a.rpb;
  // heads per thread: all eight share one set of angles once the rows alone fill the chip; a few rows are spread over the
  // heads instead
  a.hpt = H < 8 ? H : 8;
  while (a.hpt > 1 && blocks * ((H + a.hpt - 1) / a.hpt) < 512) a.hpt = (a.hpt + 1) / 2;
  const dim3 grid((unsigned)blocks, (unsigned)((H + a.hpt - 1) / a.hpt));
  hipStream_t st = (hipStream_t)stream;
#define GO(B16, I, V) hipLaunchKernelGGL((rotary_kernel<B16, I, V>), grid, dim3(256), 0, st, a)
  if (bf16) {
    if (interleaved) { if (v == 8) GO(true, true, 8); else if (v == 4) GO(true, true, 4); else if (v == 2) GO(true, true, 2); else GO(true, true, 1); }
    else { if (v == 8) GO(true, false, 8); else if (v == 4) GO(true, false, 4); else if (v == 2) GO(true, false, 2); else GO(true, false, 1); }
  } else {
    if (interleaved) { if (v == 4) GO(false, true, 4); else if (v == 2) GO(false, true, 2); else GO(false, true, 1); }
    else { if (v == 4) GO(false, false, 4); else if (v == 2) GO(false, false, 2); else GO(false, false, 1); }
  }
#undef GO
  return launch_status();
}
