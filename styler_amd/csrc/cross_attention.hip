// Attention between two sequences (queries of one, keys and values of the other), forward and backward, bf16 or fp32.
//
//   o[q, h] = sum_j p_j v[j, h / R],  p = softmax_j(scale q[q, h] . k[j, h / R]) over the keys j that are SEEN:
//   j < len[b] and not mask[b, j].  R = H / G query heads share a key head.  A query past q_len[b] and a query that sees no
//   key give 0 (lse = -inf).  With P_ij = exp(scale s_ij - lse_i) and delta_i = sum_d do_id o_id:
//   dv_j = sum_i P_ij do_i,  dS_ij = P_ij (do_i . v_j - delta_i),  dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   the sums over i running over the R heads of the group as well.
//
// Decomposition.  The R heads of a group and the queries are ONE row axis, m = q R + r (M = Lq R rows per item and key head):
// a single token of a grouped model fills R rows of a tile instead of one.  S^T = K Q^T on 32 x 32 matrix tiles, so a lane owns
// one row (column li = lane & 31 of S^T) and the 16 accumulator registers are 16 keys of it (keys (r&3) + 8 (r>>2) + 4 (lane>>5)):
// the softmax is a running maximum and sum per lane plus one exchange with lane ^ 32, and P never leaves its registers -- the
// product over the keys consumes them in place (bf16: packed in pairs, the other operand through the transposing LDS read;
// fp32: register r of both half waves IS the k pair of v_mfma_f32_32x32x2_f32).
//
// Tiles go memory -> LDS by DMA (buffer_load_dwordx4 ... lds), one tile ahead.  A lane whose key is not seen, or whose feature
// is past D (heads that are no multiple of the tile width), gives an offset past the descriptor: the DMA writes zeros, so
// nothing that stands in an unseen row (NaN, infinities) enters a product.  The 16-byte pieces of a row are permuted by the row
// index (Swz): both the row-wise ds_read_b128 and the transposing reads then touch distinct banks.
//
// Few rows: the four waves share the keys instead (key_blocks), and the key axis is cut into shares (make_plan) whose partial
// results a second launch joins.  fp32 with many rows: three bf16 planes (mma_planes).  Masks with many rows: xattn_order_kernel.
// The backward is two walks, rows over keys (dq) and keys over rows (dk, dv); each rebuilds P, nothing is added by atomics.
//
// Bounds, as measured (us of a call, one after another, without a profiler, which adds a tenth to the matrix-bound ones; TFLOP/s counts 4
// and 10 flops a pair, head and feature, not the second S and dP of the backward, 4 more):
//   forward 4 x 4096 x 4096, 16 heads of 128, bf16        519      1060 TFLOP/s: the matrix pipe at the clock this load leaves
//   forward, 2 tokens, 65537 keys, 8 heads of 128, bf16   110      5.2 TB/s in the tiles, then the join
//   forward, 32 tokens, 1500 keys, 4 key heads of 64       14      two launches by the host; 9.8 + 4.0 of the device: start, two or three
//                                                                  tiles a block (33 MB in all), join
//   training 8 x 2048 x 1500, 16 heads of 64, bf16        417      vector and matrix instructions one after the other (0.45 + 0.44 busy)
//   training 8 x 1203 x 1001, 8 heads of 64, fp32         321      six bf16 products for one (1142 / 6 = 190 TFLOP/s): those it forms, the
//                                                                  second S and dP among them, take 230; waits at the tiles' barriers
#include <type_traits>
#include "common.h"

namespace {

// Heads are padded to DT = 32, 64, 96 or 128 features; LDS rows are powers of two wide (banks, DMA).  96 leaves out a quarter of the
// products of 128 (heads of 80: training 8 x 16 heads, 2048 x 1500 bf16 890 -> 755 us, 11 x 2, 1059 x 699 fp32 254 -> 218; forward 4 x 16 /
// 4, 4096 x 4096 bf16 470 -> 420).
constexpr int stored(int dt) { return dt == 96 ? 128 : dt; }
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
constexpr uint32_t OOB = 0x80000000u;                  // past every descriptor's num_records
constexpr float LOG2E = 1.44269504088896f, LN2 = 0.693147180559945f;

struct XArgs {
  const void *q, *k, *v, *o, *dout;                    // dout / o: backward
  void *out, *dq, *dk, *dv;
  float* lse;                                          // [B, H, Lq]
  float *delta, *lse2;                                 // [B, H, Lq] (backward workspace); lse2: lse / ln 2, +inf for -inf
  float* part;                                         // partial results of a split launch
  const int64_t *len, *qlen;
  const uint8_t* mask;
  const int* order;                                    // [B, Lk] or null: the keys in the order of xattn_order_kernel
  int64_t qb, ql, qh, kb, kl, kh, vb, vl, vh, ob, ol, oh, gb, gl, gh;   // strides (elements): item, row, head; g: dout
  const void *t0, *t1;                                 // what tiles are made of: k and v, or (dk, dv) q and dout
  int64_t t0b, t0l, t0h, t0p, t1b, t1l, t1h, t1p;      // item, row, head, plane
  int64_t maskb;
  int B, Lq, Lk, H, G, R, D, nrt, splits, chunk, sort;
  float scale;
};

// Launch slot -> logical block.  Workgroups go to the eight XCDs round robin, each with its own L2, and blocks that read the same
// keys are neighbours in the logical order: runs of `chunk` logical blocks go to one XCD, run after run to the next.  (One eighth
// of the blocks each would give an XCD whole items: with ragged lengths the XCD of the longest item then worked alone.)
__device__ __forceinline__ int xcd_block(int total, int chunk) {
  const int n = blockIdx.x, i = n >> 3;
  const int v = ((i / chunk) * 8 + (n & 7)) * chunk + i % chunk;
  return v < total ? v : -1;
}

// Ragged batches are walked from the item with the most work (keys times queries) to the least, so that the last blocks are the
// shortest: item number `r` in that order.  Every wave finds it by itself -- lane i counts the items that come before item i,
// 3 B instructions.  Only for up to 16 items whose blocks' walks are long against that (8 x 1203 x 1001 fp32: 620 -> 570 us;
// 48 x 1000 x 133, sorted all the same: 74 -> 82).
__device__ __forceinline__ int item_at(const XArgs& a, int r, int lane) {
  if (!a.sort) return r;
  const int i = lane < a.B ? lane : 0;
  const float w = (float)clamp_len(a.len, i, a.Lk) * (float)clamp_len(a.qlen, i, a.Lq);
  int before = 0;
  for (int j = 0; j < a.B; ++j) {
    const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j));
    before += (x > w || (x == w && j < lane)) ? 1 : 0;
  }
  return __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.B && before == r));
}

// ---- LDS tiles: rows of DT elements, RB bytes ---------------------------------------------------------------------------------
// The 16-byte piece c of row r stands at piece c ^ swz(r).  256 bytes are the 64 banks once: rows narrower than that share a
// bank line, so the row index is divided by the rows per line first; its bits enter reversed, so that the four consecutive rows
// of a transposing read differ in the high piece bits (its 32 lanes read four neighbouring pieces of each of the four rows).
template <int RB> struct Swz {
  static constexpr int NCH = RB / 16 < 16 ? RB / 16 : 16, RPL = RB < 256 ? 256 / RB : 1;
  static constexpr int BITS = NCH == 16 ? 4 : (NCH == 8 ? 3 : (NCH == 4 ? 2 : 1));
  __device__ static constexpr uint32_t of(uint32_t row) {
    uint32_t x = row / RPL, r = 0;
    for (int i = 0; i < BITS; ++i) r |= ((x >> i) & 1u) << (BITS - 1 - i);
    return r;
  }
};

// Fill ROWS rows (a multiple of 32) of a tile: 1 KB per instruction, instruction i of a wave covers the rows
// (4 i + wave) RPI .. + RPI.  DmaLane: what a lane adds to the tile's base -- its row of the wave's first instruction and its
// (permuted) 16-byte piece; the permutation has a period of 16 rows, so it differs between instructions only where four of them
// cover fewer.  w: the bits of the rows that may be read (32 rows a word).
template <int RB> struct DmaLane {
  static constexpr int RPI = 1024 / RB, VAR = RPI * 4 >= 16 ? 1 : 16 / (RPI * 4);
  uint32_t off[VAR];
  int row;
  // pick: rows are found by their numbers (RowNumbers), off holds the piece alone
  __device__ __forceinline__ void init(int64_t ldbytes, int dbytes, int wave, int lane, bool pick = false) {
    row = wave * RPI + lane / (RB / 16);
#pragma unroll
    for (int i = 0; i < VAR; ++i) {
      const uint32_t c = ((lane % (RB / 16)) ^ Swz<RB>::of(i * 4 * RPI + row)) * 16;
      off[i] = c < (uint32_t)dbytes ? (pick ? 0u : (uint32_t)(row * (int)ldbytes)) + c : OOB;
    }
  }
};
template <int RB, int ROWS> constexpr int dma_count() { return ROWS >= 4 * (1024 / RB) ? ROWS * RB / 4096 : 1; }      // instructions per wave
// The numbers of the rows that a lane's instructions fill, where a tile's rows are any rows of the tensor; fetched a tile ahead.
template <int N> struct RowNumbers { uint32_t n[N]; };
template <int RB, int ROWS>
__device__ __forceinline__ void order_fetch(RowNumbers<dma_count<RB, ROWS>()>& rn, const int* order, int k0, int L, const DmaLane<RB>& dl) {
#pragma unroll
  for (int i = 0; i < dma_count<RB, ROWS>(); ++i) {
    const int k = k0 + i * 4 * DmaLane<RB>::RPI + dl.row;
    rn.n[i] = k < L ? order[k] : 0;
  }
}
template <int RB, int ROWS, int NW, bool PICK = false>
__device__ __forceinline__ void dma_tile(char* smem, uint32_t lds, const void* base, int64_t ldbytes, const DmaLane<RB>& dl, int wave,
                                         const uint32_t (&w)[NW], const RowNumbers<dma_count<RB, ROWS>()>* rn = nullptr) {
  constexpr int RPI = DmaLane<RB>::RPI, N = dma_count<RB, ROWS>();
  static_assert(NW == ROWS / 32, "");
  if (ROWS < 4 * RPI && wave * RPI >= ROWS) return;                  // (narrow rows: two waves fill the tile)
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const i32x4 rs = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32), 0x7fffffff, 0x00020000};      // raw buffer, 2^31 - 1 bytes
  const uint32_t l0 = (uint32_t)(uintptr_t)(lds_void*)smem + lds + wave * 1024;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r0 = i * 4 * RPI;                                      // (the word of row r0 + dl.row: 4 RPI divides 32 or is 32 k)
    uint32_t word = w[r0 / 32];
    int bit = r0 % 32 + dl.row;
    if constexpr (4 * RPI > 32 && ROWS > 32) { if (dl.row >= 32) word = w[r0 / 32 + 1]; bit &= 31; }
    uint32_t off = dl.off[i % DmaLane<RB>::VAR];
    if constexpr (PICK) off = off == OOB ? OOB : off + rn->n[i] * (uint32_t)ldbytes;
    off = (word >> bit) & 1u ? off : OOB;
    // asm: the compiler lets no transposing LDS read start before the DMA it knows of has landed (it cannot tell the buffers
    // apart), i.e. it would wait for the NEXT tile in the middle of this one.  wait_tiles orders the DMA; the asm has no outputs.
    // (m0 is reserved: the compiler keeps nothing in it, and takes no clobber of it.)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds"
                 :: "v"(off), "s"(rs), "s"(l0 + i * 4096), "s"(PICK ? 0 : r0 * (int)ldbytes) : "memory");
  }
}
// This wave's DMA has landed and its LDS reads are done; then all waves'.  The builtin, not asm: the compiler has to know that
// nothing is outstanding, or it waits for everything where a value loaded before the loop is first used in it.  The barrier itself
// touches no memory as far as the optimiser is told: the empty asm on either side keeps LDS reads and writes on theirs.
__device__ __forceinline__ void wait_tiles() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// 64 floats of a row statistic, one a lane: base[lane], or 0 where lane >= n
__device__ __forceinline__ void dma_floats(char* smem, uint32_t lds, const float* base, int n, int lane) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const i32x4 rs = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32), 0x7fffffff, 0x00020000};
  const uint32_t off = lane < n ? lane * 4u : OOB, l0 = (uint32_t)(uintptr_t)(lds_void*)smem + lds;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" :: "v"(off), "s"(rs), "s"(l0) : "memory");
}

// the other half wave's value joined in: lane and lane ^ 32 hold the same row
__device__ __forceinline__ float both_max(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// ---- matrix products ----------------------------------------------------------------------------------------------------------
// Operands are bf16 as they stand (NP = 1), fp32 (NP = 1, v_mfma_f32_32x32x2_f32), or fp32 as three bf16 planes (NP = 3): x = hi + mid + lo
// with hi = bf16(x), mid = bf16(x - hi), lo = bf16(x - hi - mid), 2^-27 of x short at most.  A product of two such numbers is six
// bf16 products (mid lo, lo mid and lo lo are below 2^-26 of it): 6 x 32 cycles of the matrix pipe for 32 x 32 x 16 where the fp32
// instruction takes 512, and the sums are fp32 either way.
// Frag: a lane's own row (32 rows of a wave), the half of its features that its half wave (lh) feeds to the product over d.
template <typename T, int DT> struct Frag;
template <int DT> struct Frag<uint16_t, DT> { bf16x8 v[DT / 16]; };
template <int DT> struct Frag<float, DT> { float4 v[DT / 8]; };
template <typename T, int DT, int NP> struct Rows { Frag<T, DT> p[NP]; };

// 8 values -> their planes.  WHOLE: for all of fp32 (inputs): what a plane would round to infinity is cut to the largest bf16, so
// that finite values stay finite (3.39e38 .. 3.40e38), and an infinity, handed down to the last plane, has products of one sign.  NaN
// goes through the cut into the next plane's remainder.
template <bool WHOLE = false> __device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&p)[3]) {
  constexpr float TOP = 3.3895313892515355e38f;          // bf16 0x7f7f
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = r[2 * e], b = r[2 * e + 1];
      if constexpr (WHOLE) if (k < 2) { a = fminf(fmaxf(a, -TOP), TOP); b = fminf(fmaxf(b, -TOP), TOP); }
      w[e] = cvt_pk_bf16_rne(a, b);
      r[2 * e] -= __uint_as_float(w[e] << 16);
      r[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
    }
    const uint4 u = make_uint4(w[0], w[1], w[2], w[3]);
    p[k] = *reinterpret_cast<const bf16x8*>(&u);
  }
}

// the lane's row of a tensor in memory (planes are made here); E: its element type there
template <typename T, int DT, int NP>
__device__ __forceinline__ void load_rows(Rows<T, DT, NP>& f, const void* base, int64_t at, int D, int lh, bool ok) {
  if constexpr (NP == 1) {
    const T* row = reinterpret_cast<const T*>(base) + at;
    constexpr int E = 16 / sizeof(T);                        // elements per 16-byte piece; lane lh takes the pieces 2 i + lh
#pragma unroll
    for (int i = 0; i < DT / E / 2; ++i) {
      const int d = (2 * i + lh) * E;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (ok && d < D) u = *reinterpret_cast<const uint4*>(row + d);
      f.p[0].v[i] = *reinterpret_cast<const typename std::remove_reference<decltype(f.p[0].v[0])>::type*>(&u);
    }
  } else {
    const float* row = reinterpret_cast<const float*>(base) + at;
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) {
      const int d = (2 * i + lh) * 8;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (ok && d < D) {
        a = *reinterpret_cast<const float4*>(row + d);
        b = *reinterpret_cast<const float4*>(row + d + 4);
      }
      const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      bf16x8 q[3];
      split8<true>(x, q);
      f.p[0].v[i] = q[0]; f.p[1].v[i] = q[1]; f.p[2].v[i] = q[2];
    }
  }
}
// s += a . b over 16 features, planes from the smallest products to the largest.  SWAP: the operands' roles are exchanged against
// another kernel's, which forms the same product: the same order there and here gives the same bits.
template <bool SWAP> __device__ __forceinline__ void mma_planes(f32x16& s, const bf16x8 (&a)[3], const bf16x8 (&b)[3]) {
  constexpr int I[6] = {2, 0, 1, 1, 0, 0}, J[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
  for (int k = 0; k < 6; ++k)
    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[SWAP ? J[k] : I[k]], b[SWAP ? I[k] : J[k]], s, 0, 0, 0);
}
__device__ __forceinline__ void zero16(f32x16& a) {
#pragma unroll
  for (int r = 0; r < 16; ++r) a[r] = 0.f;
}

// s[32 tile rows][32 lane rows] += tile(rows blk * 32 ..) . lane rows      (TS: bytes from plane to plane of the tile)
template <typename T, int DT, int NP, int TS, bool SWAP = false>
__device__ __forceinline__ void mma_rows(f32x16& s, const char* tile, int blk, const Rows<T, DT, NP>& f, int li, int lh) {
  constexpr int RB = stored(DT) * sizeof(T);
  const char* row = tile + (blk * 32 + li) * RB;
  const uint32_t x = (lh ^ Swz<RB>::of(li)) * 16;
  if constexpr (NP == 3) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) {
      bf16x8 a[3], b[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        a[k] = *reinterpret_cast<const bf16x8*>(row + k * TS + (x ^ (i * 32)));
        b[k] = f.p[k].v[i];
      }
      mma_planes<SWAP>(s, a, b);
    }
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) {
      const bf16x8 a = *reinterpret_cast<const bf16x8*>(row + (x ^ (i * 32)));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, f.p[0].v[i], s, 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < DT / 8; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(row + (x ^ (i * 32))), b = f.p[0].v[i];
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, b.x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, b.y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, b.z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, b.w, s, 0, 0, 0);
    }
  }
}

// x_row . y_row of the lane's own row: the diagonal of the rows' product, by the same instructions in the same order as mma_rows
// forms a tile row's -- equal rows give equal bits, so dP - delta is 0, not a rounding, where a query sees one key alone.
template <typename T, int DT, int NP>
__device__ __forceinline__ float rows_dot(const Rows<T, DT, NP>& xs, const Rows<T, DT, NP>& ys, int li, int lh) {
  const Frag<T, DT>&x = xs.p[0], &y = ys.p[0];
  f32x16 s;
  zero16(s);
  if constexpr (NP == 3) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) {
      const bf16x8 a[3] = {x.v[i], xs.p[1].v[i], xs.p[2].v[i]}, b[3] = {y.v[i], ys.p[1].v[i], ys.p[2].v[i]};
      mma_planes<false>(s, a, b);
    }
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v[i], y.v[i], s, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < DT / 8; ++i) {
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[i].x, y.v[i].x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[i].y, y.v[i].y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[i].z, y.v[i].z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[i].w, y.v[i].w, s, 0, 0, 0);
    }
  }
  float d = 0.f;                                         // row li stands in register (li & 3) + 4 (li >> 3) of half wave (li >> 2) & 1
#pragma unroll
  for (int r = 0; r < 16; ++r) d = r == (li & 3) + 4 * (li >> 3) ? s[r] : d;
  return both_sum(lh == ((li >> 2) & 1) ? d : 0.f);
}

__device__ __forceinline__ bf16x8 pack8(const f32x16& a, int s2) {
  uint4 v = make_uint4(cvt_pk_bf16_rne(a[s2 * 8 + 0], a[s2 * 8 + 1]), cvt_pk_bf16_rne(a[s2 * 8 + 2], a[s2 * 8 + 3]),
                       cvt_pk_bf16_rne(a[s2 * 8 + 4], a[s2 * 8 + 5]), cvt_pk_bf16_rne(a[s2 * 8 + 6], a[s2 * 8 + 7]));
  return *reinterpret_cast<bf16x8*>(&v);
}

// acc[dt][32 features][32 lane rows] += tile(rows blk * 32 ..)^T . p      (p: accumulator registers of a 32 x 32 product.  Planes:
// split like the operands.  bf16: rounded to bf16 here, the one rounding between the two products of an fp32-accumulated chain.  It
// is as large as the rounding of the result: out is 0.0023 off its 64-bit value (2-norm), 0.00165 of which are its own.  FINE adds
// p's remainder as a second operand, and only the result's rounding is left; it is taken where the keys' bytes are the bound (few rows,
// forward: 1500 keys 14.0 -> 14.1 us, 65537 keys 108.9 -> 110.0), not where it costs: 4 x 4096 x 4096 x 128 522 -> 705, training 8 x
// 2048 x 1500 x 64 422 -> 458, 48 x 1000 x 133 x 64 70 -> 73, and their gradients would need the same of dS.)
template <typename T, int DT, int NP, int TS, bool FINE = false>
__device__ __forceinline__ void mma_cols(f32x16 (&acc)[DT / 32], const char* tile, int blk, const f32x16& p, int lane) {
  constexpr int RB = stored(DT) * sizeof(T);
  const int li = lane & 31, lh = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int tq = lane & 15, tc = (lane >> 4) & 1, r0 = lh * 4 + (tq >> 2);
    const uint32_t x = ((tc * 2 + ((tq & 3) >> 1)) ^ Swz<RB>::of(r0)) * 16 + (tq & 1) * 8;
    const char* base = tile + (blk * 32 + r0) * RB;
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      bf16x8 pb[3];
      if constexpr (NP == 3) {
        const float v[8] = {p[s2 * 8], p[s2 * 8 + 1], p[s2 * 8 + 2], p[s2 * 8 + 3], p[s2 * 8 + 4], p[s2 * 8 + 5], p[s2 * 8 + 6], p[s2 * 8 + 7]};
        split8<>(v, pb);
      } else {
        pb[0] = pack8(p, s2);
        if constexpr (FINE) {
          const uint4 h = *reinterpret_cast<const uint4*>(&pb[0]);
          const uint32_t w[4] = {h.x, h.y, h.z, h.w};
          f32x16 rest;
#pragma unroll
          for (int e = 0; e < 8; ++e) rest[e] = p[s2 * 8 + e] - __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
          pb[1] = pack8(rest, 0);
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT / 32; ++dt) {
        bf16x8 a[3];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          // rows r0 + 16 s2 and r0 + 16 s2 + 8: the swizzle has a period of 16 rows
          const char* q = base + k * TS + s2 * 16 * RB;
          const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(const_cast<char*>(q + (x ^ (dt * 64)))));
          const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(const_cast<char*>(q + 8 * RB + (x ^ (dt * 64) ^ (Swz<RB>::of(8) * 16)))));
          const uint2 ua = *reinterpret_cast<const uint2*>(&t), ub = *reinterpret_cast<const uint2*>(&b);
          const uint4 u = make_uint4(ua.x, ua.y, ub.x, ub.y);
          a[k] = *reinterpret_cast<const bf16x8*>(&u);
        }
        if constexpr (NP == 3) mma_planes<false>(acc[dt], a, pb);
        else {
          if constexpr (FINE) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], pb[1], acc[dt], 0, 0, 0);
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], pb[0], acc[dt], 0, 0, 0);
        }
      }
    }
  } else {
    const uint32_t x = ((li >> 2) ^ Swz<RB>::of(lh * 4)) * 16 + (li & 3) * 4;
    const char* base = tile + (blk * 32 + lh * 4) * RB;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (r & 3) + 8 * (r >> 2);
#pragma unroll
      for (int dt = 0; dt < DT / 32; ++dt) {
        const float a = *reinterpret_cast<const float*>(base + row * RB + (x ^ (dt * 128) ^ (Swz<RB>::of(row) * 16)));
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[dt], 0, 0, 0);
      }
    }
  }
}

// a lane's row of acc (features dt * 32 + 8 g + 4 lh + 0..3) times c -> memory
template <typename T, int DT>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DT / 32], int D, int lh, float c) {
#pragma unroll
  for (int dt = 0; dt < DT / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + g * 8 + lh * 4;
      if (d >= D) continue;
      const float x = acc[dt][g * 4] * c, y = acc[dt][g * 4 + 1] * c, z = acc[dt][g * 4 + 2] * c, w = acc[dt][g * 4 + 3] * c;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + d) = make_uint2(cvt_pk_bf16_rne(x, y), cvt_pk_bf16_rne(z, w));
      else *reinterpret_cast<float4*>(row + d) = make_float4(x, y, z, w);
    }
}
template <typename T, int DT>
__device__ __forceinline__ void store_zero(T* row, int D, int lh) {
#pragma unroll
  for (int i = 0; i < DT / 8; ++i) {
    const int d = i * 8 + lh * 4;
    if (d < D) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + d) = make_uint2(0, 0);
      else *reinterpret_cast<float4*>(row + d) = make_float4(0, 0, 0, 0);
    }
  }
}

// A wave's 32 rows of acc times the lanes' c -> memory, whole rows at a time: the accumulator holds 4 features of a row per lane, so
// stored directly a wave would touch 32 rows with 8 or 16 bytes each, 4 DT / 32 times over.  `lds`: 32 * DT * sizeof(To) bytes of the
// wave's own (a tile buffer that every wave has finished with).  at(row): where row 0..31 goes, nullptr = not stored.  Lanes with
// keep = false store zeros (whatever their accumulators hold).
template <typename To, int DT, typename At>
__device__ __forceinline__ void store_tile(char* lds, const f32x16 (&acc)[DT / 32], int D, int lane, float c, bool keep, At at) {
  constexpr int RB = stored(DT) * sizeof(To), LPR = RB / 16, RPI = 64 / LPR;       // lanes per row, rows per instruction
  const int li = lane & 31, lh = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < DT / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float x = keep ? acc[dt][g * 4] * c : 0.f, y = keep ? acc[dt][g * 4 + 1] * c : 0.f;
      const float z = keep ? acc[dt][g * 4 + 2] * c : 0.f, w = keep ? acc[dt][g * 4 + 3] * c : 0.f;
      const int byte = (dt * 32 + g * 8 + lh * 4) * sizeof(To);
      char* p = lds + li * RB + (((byte / 16) ^ Swz<RB>::of(li)) * 16 + byte % 16);
      if constexpr (sizeof(To) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16_rne(x, y), cvt_pk_bf16_rne(z, w));
      else *reinterpret_cast<float4*>(p) = make_float4(x, y, z, w);
    }
#pragma unroll
  for (int i = 0; i < 32 / RPI; ++i) {
    const int row = i * RPI + lane / LPR, d = (lane % LPR) * (16 / (int)sizeof(To));
    const uint4 u = *reinterpret_cast<const uint4*>(lds + row * RB + (((lane % LPR) ^ Swz<RB>::of(row)) * 16));
    To* p = at(row);
    if (p && d < D) *reinterpret_cast<uint4*>(p + d) = u;
  }
}

// The seen keys of a tile as bit words, 32 keys each (uniform over the wave).  Without a mask they follow from the length; with
// one, lane i holds the mask bytes of keys i and (tiles of 128) 64 + i, fetched one tile before they are needed.
template <int KT> struct KeyWords {
  uint32_t w[KT / 32];
  __device__ __forceinline__ bool none() const {
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) x |= w[i];
    return x == 0;
  }
};
template <int KT> struct MaskBytes { uint8_t b[(KT + 63) / 64]; };
template <int KT>
__device__ __forceinline__ void mask_fetch(MaskBytes<KT>& m, const uint8_t* mask, int k0, int klen, int lane) {
#pragma unroll
  for (int i = 0; i < (KT + 63) / 64; ++i) {
    const int key = k0 + i * 64 + lane;
    m.b[i] = mask && key < klen ? mask[key] : 0;
  }
}
template <int KT>
__device__ __forceinline__ KeyWords<KT> key_words(const MaskBytes<KT>& m, bool has_mask, int k0, int klen, int lane) {
  KeyWords<KT> r;
  if (!has_mask && k0 + KT <= klen) {
#pragma unroll
    for (int i = 0; i < KT / 32; ++i) r.w[i] = 0xffffffffu;
    return r;
  }
#pragma unroll
  for (int i = 0; i < (KT + 63) / 64; ++i) {
    const uint64_t w = __builtin_amdgcn_ballot_w64(k0 + i * 64 + lane < klen && m.b[i] == 0);
    r.w[2 * i] = (uint32_t)w;
    if (2 * i + 1 < KT / 32) r.w[2 * i + 1] = (uint32_t)(w >> 32);
  }
  return r;
}
// word `blk` of a tile (blk is uniform, not a constant: a chain of selects keeps the words in registers)
template <int KT> __device__ __forceinline__ uint32_t word_at(const KeyWords<KT> k, int blk) {
  uint32_t w = k.w[0];
#pragma unroll
  for (int i = 1; i < KT / 32; ++i) w = blk == i ? k.w[i] : w;
  return w;
}
// Scores start at 0 for a seen key and at -inf for one that is not (its row was filled with zeros, so the product adds 0): the mask
// is the accumulator's first value, read from LDS, and costs nothing after it.  Only tiles that have unseen keys write and read it.
template <int KT>
__device__ __forceinline__ void start_put(float* start, const KeyWords<KT> k, int tid) {
  uint32_t all = k.w[0], w = k.w[0];
#pragma unroll
  for (int i = 1; i < KT / 32; ++i) {
    all &= k.w[i];
    w = (tid >> 5) == i ? k.w[i] : w;
  }
  if (all != 0xffffffffu && tid < KT) start[tid] = (w >> (tid & 31)) & 1u ? 0.f : -INFINITY;
}
// s = tile rows (blk * 32 ..) . f + that start (two copies of the product: a full tile's starts at the constant 0, without a register)
template <typename T, int DT, int NP, int TS>
__device__ __forceinline__ void mma_rows_seen(f32x16& s, const char* tile, int blk, const Rows<T, DT, NP>& f, const float* start, uint32_t w,
                                              int li, int lh) {
  if (w == 0xffffffffu) {
    zero16(s);
    mma_rows<T, DT, NP, TS>(s, tile, blk, f, li, lh);
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(start + g * 8 + lh * 4);
      s[g * 4] = x.x; s[g * 4 + 1] = x.y; s[g * 4 + 2] = x.z; s[g * 4 + 3] = x.w;
    }
    mma_rows<T, DT, NP, TS>(s, tile, blk, f, li, lh);
  }
}

// A block's four waves are RG = 4 / KG groups of 32 rows by KG groups of keys: KG = 1 where rows fill the chip, 4 where there are
// at most 32 of them, 2 between (and where blocks of 128 rows would be too few, or too uneven, to fill it).  A tile holds NB blocks
// of 32 keys for each key group: two where two tiles of K and V fit in 64 KB (two blocks a CU), so that the softmax's bookkeeping is
// shared by 64 keys.
template <typename T, int DT, int KG, int NP> constexpr int key_blocks() { return KG == 1 && stored(DT) * sizeof(T) * NP <= 256 ? 2 : 1; }

// Waves per SIMD to ask registers for: `most` where rows are shared out alone, as far as LDS lets them in; two with key groups.
template <typename T, int DT, int KG, int NP> constexpr int waves_wanted(int most) {
  return stored(DT) * sizeof(T) * NP >= 512 || (KG == 4 && stored(DT) * sizeof(T) >= 256) ? 1 : (KG == 1 ? most : 2);
}
template <typename T, int NP> struct OutOf { typedef T type; };
template <typename T> struct OutOf<T, 3> { typedef float type; };

// a block's share of the key tiles: split s of S takes tiles [s n / S, (s + 1) n / S) of the n that the item has
__device__ __forceinline__ void tile_range(int n, int s, int S, int& t0, int& t1) {
  t0 = (int)((int64_t)n * s / S);
  t1 = (int)((int64_t)n * (s + 1) / S);
}

// 4 features of block row r, summed over the key groups in order ([wave][32 rows of LDO] floats)
template <int KG, int LDO> __device__ __forceinline__ float4 group_sum(const float* so, int r, int d) {
  const float* p = so + ((r / 32) * KG * 32 + r % 32) * LDO + d;
  float4 x = *reinterpret_cast<const float4*>(p);
#pragma unroll
  for (int w = 1; w < KG; ++w) {
    const float4 y = *reinterpret_cast<const float4*>(p + w * 32 * LDO);
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
  }
  return x;
}

// ------------------------------------------------------------------------------------------------------------- forward
template <typename T, int DT, int KG, int NP, bool PICK>
__global__ __launch_bounds__(256, (waves_wanted<T, DT, KG, NP>(NP == 3 ? 3 : stored(DT) * sizeof(T) <= 128 ? 4 : 2))) void xattn_fwd_kernel(XArgs a) {
  typedef typename OutOf<T, NP>::type O;
  constexpr int RB = stored(DT) * sizeof(T), RG = 4 / KG, NB = key_blocks<T, DT, KG, NP>(), KT = 32 * KG * NB;
  constexpr int TS = KT * RB, TILE = NP * TS;            // a plane of a tile, a tile
  constexpr int NBUF = 4 * TILE <= 131072 ? 2 : 1;
  constexpr int LDO = DT + 4;                            // rows of the join start 4 banks apart
  constexpr int JOIN = KG > 1 ? 4 * 32 * LDO * 4 : 0, SMEM = 2 * NBUF * TILE > JOIN ? 2 * NBUF * TILE : JOIN;
  static_assert(KG > 1 || 4 * 32 * stored(DT) * 4 <= SMEM, "");
  __shared__ __attribute__((aligned(1024))) char smem[SMEM + 2 * KT * 4 + (KG > 1 ? 1280 : 0)];
  float* start = reinterpret_cast<float*>(smem + SMEM);          // [buffer][KT], see start_put
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
  const int rg = wave / KG, kg = wave % KG;
  const int v = xcd_block(a.nrt * a.splits * a.G * a.B, a.chunk);
  if (v < 0) return;
  const int rt = v % a.nrt, sp = (v / a.nrt) % a.splits, nth = v / (a.nrt * a.splits), g = nth % a.G, b = item_at(a, nth / a.G, lane), bg = b * a.G + g;
  const int M = a.Lq * a.R;
  const int klen = clamp_len(a.len, b, a.Lk), Mv = clamp_len(a.qlen, b, a.Lq) * a.R;
  const int m0 = rt * 32 * RG, m = m0 + rg * 32 + li;
  const int qi = m / a.R, head = g * a.R + m % a.R;
  const bool live = m < Mv;
  O* orow = reinterpret_cast<O*>(a.out) + b * a.ob + qi * a.ol + head * a.oh;
  const int64_t prow = (int64_t)bg * M + m, prows = (int64_t)a.B * a.G * M;
  float* pml = a.part ? a.part + prows * a.splits * a.D + (sp * prows + prow) * 2 : nullptr;
  int t0, t1;
  tile_range((klen + KT - 1) / KT, sp, a.splits, t0, t1);
  if (m0 >= Mv || t0 >= t1) {                            // no live row, or no key in this share
    if (kg == 0)
      if (m < M) {
        if (a.splits > 1) { if (lh == 0) { pml[0] = -INFINITY; pml[1] = 0.f; } }
        else {
          store_zero<O, DT>(orow, a.D, lh);
          if (a.lse && lh == 0) a.lse[((int64_t)b * a.H + head) * a.Lq + qi] = -INFINITY;
        }
      }
    return;
  }
  const T* kbase = reinterpret_cast<const T*>(a.t0) + b * a.t0b + g * a.t0h;
  const T* vbase = reinterpret_cast<const T*>(a.t1) + b * a.t1b + g * a.t1h;
  const uint8_t* mask = a.mask ? a.mask + b * a.maskb : nullptr;
  const int dbytes = (NP == 3 ? DT : a.D) * (int)sizeof(T);
  const int64_t klb = a.t0l * (int64_t)sizeof(T), vlb = a.t1l * (int64_t)sizeof(T);

  MaskBytes<KT> mb;
  mask_fetch(mb, mask, t0 * KT, klen, lane);
  KeyWords<KT> cur = key_words(mb, mask != nullptr, t0 * KT, klen, lane), nxt = cur;
  DmaLane<RB> kdl, vdl;
  kdl.init(klb, dbytes, wave, lane, PICK);
  vdl.init(vlb, dbytes, wave, lane, PICK);
  const int* order = PICK ? a.order + (int64_t)b * a.Lk : nullptr;
  RowNumbers<dma_count<RB, KT>()> rn;
  if constexpr (PICK) order_fetch<RB, KT>(rn, order, t0 * KT, a.Lk, kdl);
  auto fill = [&](int t, int buf, const KeyWords<KT>& kw) {
    const int64_t first = PICK ? 0 : (int64_t)t * KT;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      dma_tile<RB, KT, KT / 32, PICK>(smem, buf * 2 * TILE + k * TS, kbase + k * a.t0p + first * a.t0l, klb, kdl, wave, kw.w, &rn);
      dma_tile<RB, KT, KT / 32, PICK>(smem, buf * 2 * TILE + TILE + k * TS, vbase + k * a.t1p + first * a.t1l, vlb, vdl, wave, kw.w, &rn);
    }
    start_put(start + buf * KT, kw, tid);
    if constexpr (PICK) order_fetch<RB, KT>(rn, order, (t + 1) * KT, a.Lk, kdl);
  };
  fill(t0, 0, cur);
  Rows<T, DT, NP> qf;
  load_rows(qf, a.q, b * a.qb + qi * a.ql + head * a.qh, a.D, lh, live);
  mask_fetch(mb, mask, (t0 + 1) * KT, klen, lane);

  f32x16 o[DT / 32];
#pragma unroll
  for (int i = 0; i < DT / 32; ++i) zero16(o[i]);
  const float SC = a.scale * LOG2E;                      // scores in the log2 domain: p = exp2(SC s - SC m)
  float mx = -INFINITY, l = 0.f;
  wait_tiles();
  for (int t = t0; t < t1; ++t) {
    const int buf = NBUF == 2 ? (t - t0) & 1 : 0;
    if (t + 1 < t1) {
      nxt = key_words(mb, mask != nullptr, (t + 1) * KT, klen, lane);
      if (NBUF == 2) {
        fill(t + 1, buf ^ 1, nxt);
        mask_fetch(mb, mask, (t + 2) * KT, klen, lane);
      }
    }
    if (!cur.none()) {
      const char* tk = smem + buf * 2 * TILE;
      const char* tv = tk + TILE;
      f32x16 s[NB];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const int blk = kg * NB + kb;
        mma_rows_seen<T, DT, NP, TS>(s[kb], tk, blk, qf, start + buf * KT + blk * 32, word_at(cur, blk), li, lh);
      }
      __builtin_amdgcn_s_setprio(0);
      float mt = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[kb][r]);
      mt = both_max(mt);
      // The maximum moves only when a tile exceeds it by more than 8 in the log2 domain (p <= 256 is harmless; o and l
      // carry the same maximum): the rescaling of o leaves the common path.
      const bool move = mt * SC > mx * SC + 8.f;
      if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float mn = move ? mt : mx;
        const float al = mn == mx ? 1.f : __builtin_amdgcn_exp2f((mx - mn) * SC);
        mx = mn;
        l *= al;
#pragma unroll
        for (int i = 0; i < DT / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= al;
      }
      const float sub = mx == -INFINITY ? 0.f : mx, off = -sub * SC;
      float ls = 0.f;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          // (fp32: (s - max) SC, so that the largest P is 1 to the last bit; bf16 rounds P anyway and takes one instruction)
          s[kb][r] = __builtin_amdgcn_exp2f(sizeof(O) == 2 ? fmaf(s[kb][r], SC, off) : (s[kb][r] - sub) * SC);
          ls += s[kb][r];
        }
      l += ls;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) mma_cols<T, DT, NP, TS, KG == 4>(o, tv, kg * NB + kb, s[kb], lane);
      __builtin_amdgcn_s_setprio(0);
    }
    if (NBUF == 1 && t + 1 < t1) {
      wait_tiles();                                      // every wave has read the tile: it may be overwritten
      fill(t + 1, 0, nxt);
      mask_fetch(mb, mask, (t + 2) * KT, klen, lane);
    }
    wait_tiles();
    cur = nxt;
  }
  l = both_sum(l);                                       // (a lane summed its half of the keys)
  if (!live) {                                           // a row past the queries: as one that sees no key
    mx = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < DT / 32; ++i) zero16(o[i]);
  }
  const float m2 = mx == -INFINITY ? -INFINITY : mx * SC;      // log2 domain
  if constexpr (KG == 1) {
    const int mw = m0 + wave * 32;
    if (a.splits > 1) {
      store_tile<float, DT>(smem + wave * 32 * stored(DT) * 4, o, a.D, lane, 1.f, true, [&](int r) {
        return mw + r < M ? a.part + (sp * prows + (int64_t)bg * M + mw + r) * a.D : nullptr;
      });
      if (lh == 0 && m < M) { pml[0] = m2; pml[1] = l; }
    } else {
      store_tile<O, DT>(smem + wave * 32 * stored(DT) * sizeof(O), o, a.D, lane, l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l), true, [&](int r) {
        return mw + r < M ? reinterpret_cast<O*>(a.out) + b * a.ob + (mw + r) / a.R * a.ol + (g * a.R + (mw + r) % a.R) * a.oh : nullptr;
      });
      if (a.lse && lh == 0 && m < M) a.lse[((int64_t)b * a.H + head) * a.Lq + qi] = l == 0.f ? -INFINITY : (m2 + log2f(l)) * LN2;
    }
  } else {
    // join the key groups of a row group: ml[wave][32] = (max, sum), then o scaled to the common maximum, summed in group order
    float* ml = reinterpret_cast<float*>(smem + SMEM + 2 * KT * 4);
    float* inv = ml + 256;                               // [RG * 32]
    if (lh == 0) { ml[(wave * 32 + li) * 2] = m2; ml[(wave * 32 + li) * 2 + 1] = l; }
    wait_tiles();
    float mm = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < KG; ++w) mm = fmaxf(mm, ml[((rg * KG + w) * 32 + li) * 2]);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < KG; ++w) {
      const float* p = ml + ((rg * KG + w) * 32 + li) * 2;
      lt += p[1] * __builtin_amdgcn_exp2f(p[0] - base);
    }
    const float c = __builtin_amdgcn_exp2f(m2 - base);
    float* so = reinterpret_cast<float*>(smem);          // [wave][32 rows of LDO]
#pragma unroll
    for (int dt = 0; dt < DT / 32; ++dt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<float4*>(so + (wave * 32 + li) * LDO + dt * 32 + gq * 8 + lh * 4) =
            make_float4(o[dt][gq * 4] * c, o[dt][gq * 4 + 1] * c, o[dt][gq * 4 + 2] * c, o[dt][gq * 4 + 3] * c);
    if (kg == 0 && lh == 0) {
      inv[rg * 32 + li] = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
      if (m < M) {
        if (a.splits > 1) { pml[0] = mm; pml[1] = lt; }
        else if (a.lse) a.lse[((int64_t)b * a.H + head) * a.Lq + qi] = lt == 0.f ? -INFINITY : (mm + log2f(lt)) * LN2;
      }
    }
    wait_tiles();
    for (int i = tid; i < RG * 32 * (DT / 4); i += 256) {
      const int r = i / (DT / 4), d = (i % (DT / 4)) * 4, mr = m0 + r;
      if (mr >= M || d >= a.D) continue;
      const float4 x = group_sum<KG, LDO>(so, r, d);
      if (a.splits > 1) {
        *reinterpret_cast<float4*>(a.part + (sp * prows + (int64_t)bg * M + mr) * a.D + d) = x;
      } else {
        const float cl = inv[r];
        T* p = reinterpret_cast<T*>(a.out) + b * a.ob + (mr / a.R) * a.ol + (g * a.R + mr % a.R) * a.oh + d;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16_rne(x.x * cl, x.y * cl), cvt_pk_bf16_rne(x.z * cl, x.w * cl));
        else *reinterpret_cast<float4*>(p) = make_float4(x.x * cl, x.y * cl, x.z * cl, x.w * cl);
      }
    }
  }
}

// Join the splits of a forward launch: a wave per row.  Lane s holds the (max, sum) of split s; the partial rows are read by
// W / 4 lanes each, 256 / W splits at a time (W = 32, 64, 128 >= D), and their sums joined across those lane groups.  An empty
// split has max = -inf, sum = 0, and its partial row is not read (it is not written either).
constexpr int MAX_SPLITS = 64;
template <typename T, int W>
__global__ __launch_bounds__(256) void xattn_join_kernel(XArgs a) {
  const int lane = threadIdx.x & 63;
  const int M = a.Lq * a.R;
  const int64_t rows = (int64_t)a.B * a.G * M, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int bg = (int)(row / M), m = (int)(row % M), g = bg % a.G, b = bg / a.G, qi = m / a.R, head = g * a.R + m % a.R;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < a.splits) ml = *reinterpret_cast<const float2*>(a.part + rows * a.splits * a.D + (lane * rows + row) * 2);
  const float mm = wave_max(ml.x), base = mm == -INFINITY ? 0.f : mm;
  const float c = __builtin_amdgcn_exp2f(ml.x - base);
  const float l = wave_sum(c * ml.y);
  constexpr int LPR = W / 4, GR = 64 / LPR, U = 4;
  const int d = (lane % LPR) * 4, grp = lane / LPR;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < a.splits; s0 += GR * U) {
    float4 p[U];
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int sp = s0 + u * GR + grp;
      w[u] = __shfl(c, sp & 63, 64);
      p[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      const bool full = __shfl(ml.x, sp & 63, 64) != -INFINITY;
      if (sp < a.splits && full && d < a.D) p[u] = *reinterpret_cast<const float4*>(a.part + (sp * rows + row) * a.D + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * GR + grp >= a.splits) w[u] = 0.f;
      x.x = fmaf(w[u], p[u].x, x.x); x.y = fmaf(w[u], p[u].y, x.y); x.z = fmaf(w[u], p[u].z, x.z); x.w = fmaf(w[u], p[u].w, x.w);
    }
  }
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) {
    x.x += __shfl_xor(x.x, o, 64); x.y += __shfl_xor(x.y, o, 64); x.z += __shfl_xor(x.z, o, 64); x.w += __shfl_xor(x.w, o, 64);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (grp == 0 && d < a.D) {
    T* p = reinterpret_cast<T*>(a.out) + b * a.ob + qi * a.ol + head * a.oh + d;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16_rne(x.x * inv, x.y * inv), cvt_pk_bf16_rne(x.z * inv, x.w * inv));
    else *reinterpret_cast<float4*>(p) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  }
  if (a.lse && lane == 0) a.lse[((int64_t)b * a.H + head) * a.Lq + qi] = l == 0.f ? -INFINITY : (mm + log2f(l)) * LN2;
}

// ------------------------------------------------------------------------------------------------------------- dQ (and delta)
// Same walk as the forward; P is rebuilt from lse.  A row without keys has lse = -inf: it takes +inf here, every P is 0.
//
// delta = do . o is off by the rounding of a bf16 o, which weighs where a query sees a few keys (o is as large as a value then, and
// the scores' gradient a difference of few terms: 3 keys gave dq an error of 0.0037, 100 keys 0.0024).  Items of up to FEW seen keys,
// by their length or by their mask, take delta + sum_j P_j (do . v_j - delta) instead: the exact sum.  Their keys are gathered into
// one block of 32 tile rows for that, and every wave and share forms the sum by itself.  (0 stays 0 where one key is seen.)
constexpr int FEW = 32;
// 16 bytes of the mask from key k on; keys at or past klen count as dropped
__device__ __forceinline__ uint4 mask16(const uint8_t* mask, int k, int klen) {
  uint4 u;
  if (__builtin_amdgcn_ballot_w64(k + 16 > klen) == 0) {
    __builtin_memcpy(&u, mask + k, 16);
  } else {
    uint32_t m[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) m[i] = k + i < klen ? mask[k + i] : 1;
    u = make_uint4(m[0] | m[1] << 8 | m[2] << 16 | m[3] << 24, m[4] | m[5] << 8 | m[6] << 16 | m[7] << 24,
                   m[8] | m[9] << 8 | m[10] << 16 | m[11] << 24, m[12] | m[13] << 8 | m[14] << 16 | m[15] << 24);
  }
  return u;
}
// bit 8 j + 7: byte j of x is zero
__device__ __forceinline__ uint32_t zero_byte_bits(uint32_t x) { return ~(((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u; }
// The number of seen keys, or FEW + 1 if they are more; where they are not, list[0 ..] receives their numbers (`put`: by this wave).
// first: mask16 of the lane's first keys, fetched early: most masks are done after those, which costs the backward of 4 x 64 x 4096
// keys half a us.  Then 8192 keys a step (2 x 8 rows, 65537 keys of which a mask leaves 3: 58 us with the sum, 46 without; 512 keys
// a step 256).
__device__ __forceinline__ int few_keys(const uint8_t* mask, const int* order, int klen, int lane, int* list, bool put, const uint4& first) {
  if (!mask) {
    if (klen <= FEW && put && lane < klen) list[lane] = order ? order[lane] : lane;
    return klen <= FEW ? klen : FEW + 1;
  }
  int n = 0;
  auto add = [&](const uint4& u, int k) {
    const uint32_t z[4] = {zero_byte_bits(u.x), zero_byte_bits(u.y), zero_byte_bits(u.z), zero_byte_bits(u.w)};
    const int mine = __builtin_popcount(z[0]) + __builtin_popcount(z[1]) + __builtin_popcount(z[2]) + __builtin_popcount(z[3]);
    if (__builtin_amdgcn_ballot_w64(mine != 0) == 0) return;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const int before = n + upto - mine;
    n += __builtin_amdgcn_readlane(upto, 63);
    if (!put || n > FEW) return;
    int at = before;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      for (uint32_t x = z[i]; x; x &= x - 1) list[at++] = k + 4 * i + __builtin_ctz(x) / 8;
  };
  add(first, lane * 16);
  for (int k0 = 1024; k0 < klen && n <= FEW; k0 += 8192) {
    uint4 u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = mask16(mask, k0 + i * 1024 + lane * 16, klen);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n <= FEW) add(u[i], k0 + i * 1024 + lane * 16);
  }
  return n <= FEW ? n : FEW + 1;
}
template <typename T, int DT, int KG, int NP, bool PICK>
__global__ __launch_bounds__(256, (waves_wanted<T, DT, KG, NP>(NP == 1 && stored(DT) * sizeof(T) <= 128 ? 3 : 2))) void xattn_dq_kernel(XArgs a) {
  typedef typename OutOf<T, NP>::type O;
  constexpr int RB = stored(DT) * sizeof(T), RG = 4 / KG, NB = key_blocks<T, DT, KG, NP>(), KT = 32 * KG * NB;
  constexpr int TS = KT * RB, TILE = NP * TS;
  constexpr int NBUF = 4 * TILE <= 131072 ? 2 : 1;
  constexpr int LDO = DT + 4;
  constexpr int JOIN = KG > 1 ? 4 * 32 * LDO * 4 : 0, SMEM = 2 * NBUF * TILE > JOIN ? 2 * NBUF * TILE : JOIN;
  static_assert(KG > 1 || 4 * 32 * stored(DT) * 4 <= SMEM, "");
  constexpr bool SUMS = NP == 1 && sizeof(T) == 2;       // (fp32: o is as good as the sums)
  static_assert(!SUMS || NBUF == 2, "");                 // (the few keys are gathered into the second buffer)
  __shared__ __attribute__((aligned(1024))) char smem[SMEM + 2 * KT * 4 + (SUMS ? FEW * 4 : 0)];
  float* start = reinterpret_cast<float*>(smem + SMEM);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
  const int rg = wave / KG, kg = wave % KG;
  const int v = xcd_block(a.nrt * a.splits * a.G * a.B, a.chunk);
  if (v < 0) return;
  const int rt = v % a.nrt, sp = (v / a.nrt) % a.splits, nth = v / (a.nrt * a.splits), g = nth % a.G, b = item_at(a, nth / a.G, lane), bg = b * a.G + g;
  const int M = a.Lq * a.R;
  const int klen = clamp_len(a.len, b, a.Lk), Mv = clamp_len(a.qlen, b, a.Lq) * a.R;
  const int m0 = rt * 32 * RG, m = m0 + rg * 32 + li;
  const int qi = m / a.R, head = g * a.R + m % a.R;
  const bool live = m < Mv;
  O* dqrow = reinterpret_cast<O*>(a.dq) + (((int64_t)b * a.Lq + qi) * a.H + head) * a.D;
  const int64_t prow = (int64_t)bg * M + m, prows = (int64_t)a.B * a.G * M;
  const int64_t srow = ((int64_t)b * a.H + head) * a.Lq + qi;
  Rows<T, DT, NP> qf, dof;
  float lse2 = INFINITY;
  load_rows(dof, a.dout, b * a.gb + qi * a.gl + head * a.gh, a.D, lh, live);
  load_rows(qf, a.o, b * a.ob + qi * a.ol + head * a.oh, a.D, lh, live);
  float dl = rows_dot(qf, dof, li, lh);
  if (live) {
    const float x = a.lse[srow];
    lse2 = x == -INFINITY ? INFINITY : x * LOG2E;
  }
  if (sp == 0 && m < M && lh == 0 && kg == 0) {
    a.lse2[srow] = lse2;
    if (!SUMS) a.delta[srow] = dl;
  }
  int t0, t1;
  tile_range((klen + KT - 1) / KT, sp, a.splits, t0, t1);
  if (m0 >= Mv || t0 >= t1) {
    if (m < M && kg == 0) {
      if (a.splits > 1) store_zero<float, DT>(a.part + (sp * prows + prow) * a.D, a.D, lh);
      else store_zero<O, DT>(dqrow, a.D, lh);
    }
    return;
  }
  const T* kbase = reinterpret_cast<const T*>(a.t0) + b * a.t0b + g * a.t0h;
  const T* vbase = reinterpret_cast<const T*>(a.t1) + b * a.t1b + g * a.t1h;
  const uint8_t* mask = a.mask ? a.mask + b * a.maskb : nullptr;
  const int dbytes = (NP == 3 ? DT : a.D) * (int)sizeof(T);
  const int64_t klb = a.t0l * (int64_t)sizeof(T), vlb = a.t1l * (int64_t)sizeof(T);
  const uint4 first = SUMS && mask ? mask16(mask, lane * 16, klen) : make_uint4(0, 0, 0, 0);
  MaskBytes<KT> mb;
  mask_fetch(mb, mask, t0 * KT, klen, lane);
  KeyWords<KT> cur = key_words(mb, mask != nullptr, t0 * KT, klen, lane), nxt = cur;
  DmaLane<RB> kdl, vdl;
  kdl.init(klb, dbytes, wave, lane, PICK);
  vdl.init(vlb, dbytes, wave, lane, PICK);
  const int* order = PICK ? a.order + (int64_t)b * a.Lk : nullptr;
  RowNumbers<dma_count<RB, KT>()> rn;
  if constexpr (PICK) order_fetch<RB, KT>(rn, order, t0 * KT, a.Lk, kdl);
  auto fill = [&](int t, int buf, const KeyWords<KT>& kw) {
    const int64_t first = PICK ? 0 : (int64_t)t * KT;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      dma_tile<RB, KT, KT / 32, PICK>(smem, buf * 2 * TILE + k * TS, kbase + k * a.t0p + first * a.t0l, klb, kdl, wave, kw.w, &rn);
      dma_tile<RB, KT, KT / 32, PICK>(smem, buf * 2 * TILE + TILE + k * TS, vbase + k * a.t1p + first * a.t1l, vlb, vdl, wave, kw.w, &rn);
    }
    start_put(start + buf * KT, kw, tid);
    if constexpr (PICK) order_fetch<RB, KT>(rn, order, (t + 1) * KT, a.Lk, kdl);
  };
  fill(t0, 0, cur);
  load_rows(qf, a.q, b * a.qb + qi * a.ql + head * a.qh, a.D, lh, live);
  mask_fetch(mb, mask, (t0 + 1) * KT, klen, lane);
  f32x16 dq[DT / 32];
#pragma unroll
  for (int i = 0; i < DT / 32; ++i) zero16(dq[i]);
  const float SC = a.scale * LOG2E;
  int* list = reinterpret_cast<int*>(start + 2 * KT);
  const int n = SUMS ? few_keys(mask, order, klen, lane, list, wave == 0, first) : 0;
  wait_tiles();
  if constexpr (SUMS) {
    if (n <= FEW) {                                      // (the same for the whole block)
      char* few = smem + 2 * TILE;
      for (int i = tid; i < 2 * 32 * (RB / 16); i += 256) {
        const int c = i % (RB / 16), r = i / (RB / 16) % 32, x = i / (RB / 16 * 32);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < n && c * 16 < dbytes) u = *reinterpret_cast<const uint4*>((x ? vbase : kbase) + list[r] * (x ? a.t1l : a.t0l) + c * (16 / sizeof(T)));
        *reinterpret_cast<uint4*>(few + x * TILE + r * RB + (c ^ Swz<RB>::of(r)) * 16) = u;
      }
      if (tid < 32) start[KT + tid] = tid < n ? 0.f : -INFINITY;
      wait_tiles();
      f32x16 s, dp;
      zero16(dp);
      mma_rows_seen<T, DT, NP, TS>(s, few, 0, qf, start + KT, n == 32 ? 0xffffffffu : (1u << n) - 1u, li, lh);
      mma_rows<T, DT, NP, TS>(dp, few + TILE, 0, dof, li, lh);
      float c = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) c = fmaf(__builtin_amdgcn_exp2f(fmaf(s[r], SC, -lse2)), dp[r] - dl, c);
      dl += both_sum(c);
      wait_tiles();                                      // every wave has read the buffer: the second tile may come
    }
    if (sp == a.splits - 1 && m < M && lh == 0 && kg == 0) a.delta[srow] = dl;       // (the last share of an item with keys has a tile)
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = NBUF == 2 ? (t - t0) & 1 : 0;
    if (t + 1 < t1) {
      nxt = key_words(mb, mask != nullptr, (t + 1) * KT, klen, lane);
      if (NBUF == 2) {
        fill(t + 1, buf ^ 1, nxt);
        mask_fetch(mb, mask, (t + 2) * KT, klen, lane);
      }
    }
    const char* tk = smem + buf * 2 * TILE;
    const char* tv = tk + TILE;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      const int blk = kg * NB + kb;
      const uint32_t w = word_at(cur, blk);
      if (w == 0) continue;
      f32x16 s, dp;
      zero16(dp);
      __builtin_amdgcn_s_setprio(1);
      mma_rows_seen<T, DT, NP, TS>(s, tk, blk, qf, start + buf * KT + blk * 32, w, li, lh);      // (unseen: P = exp2(-inf) = 0)
      mma_rows<T, DT, NP, TS>(dp, tv, blk, dof, li, lh);
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], SC, -lse2)) * (dp[r] - dl);
      __builtin_amdgcn_s_setprio(1);
      mma_cols<T, DT, NP, TS>(dq, tk, blk, s, lane);
      __builtin_amdgcn_s_setprio(0);
    }
    if (NBUF == 1 && t + 1 < t1) {
      wait_tiles();
      fill(t + 1, 0, nxt);
      mask_fetch(mb, mask, (t + 2) * KT, klen, lane);
    }
    wait_tiles();
    cur = nxt;
  }
  if constexpr (KG == 1) {
    const int mw = m0 + wave * 32;
    if (a.splits > 1)
      store_tile<float, DT>(smem + wave * 32 * stored(DT) * 4, dq, a.D, lane, a.scale, true, [&](int r) {
        return mw + r < M ? a.part + (sp * prows + (int64_t)bg * M + mw + r) * a.D : nullptr;
      });
    else
      store_tile<O, DT>(smem + wave * 32 * stored(DT) * sizeof(O), dq, a.D, lane, a.scale, true, [&](int r) {
        return mw + r < M ? reinterpret_cast<O*>(a.dq) + (((int64_t)b * a.Lq + (mw + r) / a.R) * a.H + g * a.R + (mw + r) % a.R) * a.D : nullptr;
      });
  } else {
    float* so = reinterpret_cast<float*>(smem);          // sums over the key groups
#pragma unroll
    for (int dt = 0; dt < DT / 32; ++dt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<float4*>(so + (wave * 32 + li) * LDO + dt * 32 + gq * 8 + lh * 4) =
            make_float4(dq[dt][gq * 4], dq[dt][gq * 4 + 1], dq[dt][gq * 4 + 2], dq[dt][gq * 4 + 3]);
    wait_tiles();
    for (int i = tid; i < RG * 32 * (DT / 4); i += 256) {
      const int r = i / (DT / 4), d = (i % (DT / 4)) * 4, mr = m0 + r;
      if (mr >= M || d >= a.D) continue;
      float4 x = group_sum<KG, LDO>(so, r, d);
      x.x *= a.scale; x.y *= a.scale; x.z *= a.scale; x.w *= a.scale;
      if (a.splits > 1) *reinterpret_cast<float4*>(a.part + (sp * prows + (int64_t)bg * M + mr) * a.D + d) = x;
      else {
        T* p = reinterpret_cast<T*>(a.dq) + (((int64_t)b * a.Lq + mr / a.R) * a.H + g * a.R + mr % a.R) * a.D + d;
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16_rne(x.x, x.y), cvt_pk_bf16_rne(x.z, x.w));
        else *reinterpret_cast<float4*>(p) = x;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- dK, dV
// acc of the giving waves -> acc of their partners through LDS (all waves of the block call it)
template <int N> __device__ __forceinline__ void add_from(f32x16 (&acc)[N], char* lds, int lane, bool gives) {
  float4* p = reinterpret_cast<float4*>(lds) + lane;
  if (gives) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) p[(i * 4 + g) * 64] = make_float4(acc[i][g * 4], acc[i][g * 4 + 1], acc[i][g * 4 + 2], acc[i][g * 4 + 3]);
  }
  wait_tiles();
  if (!gives) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 x = p[(i * 4 + g) * 64];
        acc[i][g * 4] += x.x; acc[i][g * 4 + 1] += x.y; acc[i][g * 4 + 2] += x.z; acc[i][g * 4 + 3] += x.w;
      }
  }
  wait_tiles();
}

// A block owns 32 KW keys (KW = 4, or 2 where that would be too few blocks), a lane one key: its K and V rows stay in registers.
// The block walks tiles of 64 query rows (32 of planes), head after head of the group; with KW = 2 two waves share the keys and each takes half of
// a tile's rows.  S = Q K^T here, so the registers are 16 queries and their lse / delta come from LDS.  What an unseen key computes
// stays in its own lane; zeros are stored for it.
// Registers: two blocks of rows in flight where a lane's K, V, dK and dV leave room for them.  With the waves asked for here the compiler
// keeps 1 register of <64, 4 waves of keys>, 8 of <128, 4> and 25 of <128, 2> (bf16) in scratch; asking for a wave less frees them, and is
// slower: backward 8 x 2048 x 1500 x 16 heads of 64 366 -> 374 us, 48 x 1000 x 133 x 4 x 64 62 -> 73, 4 x 2048 x 2048 x 16 / 4 x 128
// 533 -> 550, 16 x 500 x 200 x 8 x 128 57 -> 67.
template <typename T, int DT, int NP> constexpr int DKV_UNROLL = stored(DT) * sizeof(T) * NP >= 256 ? 1 : 2;
template <typename T, int DT, int KW, int NP>
__global__ __launch_bounds__(256, (stored(DT) * sizeof(T) * NP >= 512 ? 1 : stored(DT) * sizeof(T) * NP >= 256 ? 2 : 3)) void xattn_dkv_kernel(XArgs a) {
  typedef typename OutOf<T, NP>::type O;
  constexpr int RB = stored(DT) * sizeof(T), RT = NP == 3 ? 32 : 64, TS = RT * RB, TILE = NP * TS, RW = 4 / KW, NBLK = RT / 32 / RW;
  constexpr int SHARE = 32 * stored(DT) * 4;             // LDS of a wave for its results, once the tiles are done with
  static_assert(NBLK >= 1 && 4 * SHARE <= 4 * TILE, "");
  constexpr int STAT = 4 * TILE;                         // [buf][lse2 | delta][64]
  __shared__ __attribute__((aligned(1024))) char smem[STAT + 2 * 512];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 31, lh = lane >> 5;
  const int kwv = wave / RW, rwv = wave % RW;
  const int v = xcd_block(a.nrt * a.splits * a.G * a.B, a.chunk);
  if (v < 0) return;
  const int kt = v % a.nrt, sp = (v / a.nrt) % a.splits, nth = v / (a.nrt * a.splits), g = nth % a.G, b = item_at(a, nth / a.G, lane);
  const int klen = clamp_len(a.len, b, a.Lk), qv = clamp_len(a.qlen, b, a.Lq);
  const int key = kt * 32 * KW + kwv * 32 + li;
  const bool seen = key < klen && !(a.mask && a.mask[b * a.maskb + key]);
  const bool some = __builtin_amdgcn_ballot_w64(seen) != 0;
  // the block's p-th key is key number order[p] of the item, its row of k, v and of the gradients
  const int* order = a.order ? a.order + (int64_t)b * a.Lk : nullptr;
  const int knum = order && key < a.Lk ? order[key] : key;
  const int64_t krow = ((int64_t)b * a.Lk + knum) * a.G + g, krows = (int64_t)a.B * a.Lk * a.G;
  const int nt = (qv + RT - 1) / RT, total = nt * a.R;
  int t0, t1;
  tile_range(total, sp, a.splits, t0, t1);
  if (kt * 32 * KW >= klen || t0 >= t1) {
    if (key < a.Lk && rwv == 0) {
      if (a.splits > 1) {
        store_zero<float, DT>(a.part + (sp * 2 * krows + krow) * a.D, a.D, lh);
        store_zero<float, DT>(a.part + ((sp * 2 + 1) * krows + krow) * a.D, a.D, lh);
      } else {
        store_zero<O, DT>(reinterpret_cast<O*>(a.dk) + krow * a.D, a.D, lh);
        store_zero<O, DT>(reinterpret_cast<O*>(a.dv) + krow * a.D, a.D, lh);
      }
    }
    return;
  }
  const int dbytes = (NP == 3 ? DT : a.D) * (int)sizeof(T);
  const int64_t qlb = a.t0l * (int64_t)sizeof(T), glb = a.t1l * (int64_t)sizeof(T);
  DmaLane<RB> qdl, gdl;
  qdl.init(qlb, dbytes, wave, lane);
  gdl.init(glb, dbytes, wave, lane);
  auto fill = [&](int t, int buf) {
    const int r = t / nt, q0 = (t - r * nt) * RT, head = g * a.R + r, left = qv - q0;
    uint32_t w[RT / 32];
#pragma unroll
    for (int i = 0; i < RT / 32; ++i) w[i] = left >= 32 * (i + 1) ? 0xffffffffu : (left <= 32 * i ? 0u : (1u << (left - 32 * i)) - 1u);
    const T* qp = reinterpret_cast<const T*>(a.t0) + b * a.t0b + (int64_t)q0 * a.t0l + head * a.t0h;
    const T* gp = reinterpret_cast<const T*>(a.t1) + b * a.t1b + (int64_t)q0 * a.t1l + head * a.t1h;
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      dma_tile<RB, RT>(smem, buf * 2 * TILE + k * TS, qp + k * a.t0p, qlb, qdl, wave, w);
      dma_tile<RB, RT>(smem, buf * 2 * TILE + TILE + k * TS, gp + k * a.t1p, glb, gdl, wave, w);
    }
    if (wave < 2) {                                      // (rows past the queries are zeros throughout: they add 0, whatever P is)
      const float* st = (wave == 0 ? a.lse2 : a.delta) + ((int64_t)b * a.H + head) * a.Lq + q0;
      dma_floats(smem, STAT + buf * 512 + wave * 256, st, left < RT ? left : RT, lane);
    }
  };
  fill(t0, 0);
  Rows<T, DT, NP> kf, vf;
  load_rows(kf, a.k, b * a.kb + (int64_t)knum * a.kl + g * a.kh, a.D, lh, seen);
  load_rows(vf, a.v, b * a.vb + (int64_t)knum * a.vl + g * a.vh, a.D, lh, seen);
  f32x16 dk[DT / 32], dv[DT / 32];
#pragma unroll
  for (int i = 0; i < DT / 32; ++i) { zero16(dk[i]); zero16(dv[i]); }
  const float SC = a.scale * LOG2E;
  wait_tiles();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    if (t + 1 < t1) fill(t + 1, buf ^ 1);
    const char* tq = smem + buf * 2 * TILE;
    const char* tg = tq + TILE;
    const float* st = reinterpret_cast<const float*>(smem + STAT + buf * 512);
    if (some)                                            // (a wave whose keys are all unseen only helps to load)
#pragma unroll DKV_UNROLL<T, DT, NP>
    for (int hb = 0; hb < NBLK; ++hb) {
      const int blk = rwv * NBLK + hb;
      f32x16 s, dp;
      zero16(s);
      zero16(dp);
      __builtin_amdgcn_s_setprio(1);
      mma_rows<T, DT, NP, TS, true>(s, tq, blk, kf, li, lh);
      mma_rows<T, DT, NP, TS, true>(dp, tg, blk, vf, li, lh);
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const float4 L = *reinterpret_cast<const float4*>(st + blk * 32 + gq * 8 + lh * 4);
        const float4 E = *reinterpret_cast<const float4*>(st + 64 + blk * 32 + gq * 8 + lh * 4);
        const float ls[4] = {L.x, L.y, L.z, L.w}, de[4] = {E.x, E.y, E.z, E.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = gq * 4 + e;
          s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], SC, -ls[e]));
          dp[r] = s[r] * (dp[r] - de[e]);
        }
      }
      __builtin_amdgcn_s_setprio(1);
      mma_cols<T, DT, NP, TS>(dv, tg, blk, s, lane);
      mma_cols<T, DT, NP, TS>(dk, tq, blk, dp, lane);
      __builtin_amdgcn_s_setprio(0);
    }
    wait_tiles();
  }
  if constexpr (RW == 2) {                               // the second half of the rows joins the first
    add_from(dk, smem + kwv * SHARE, lane, rwv == 1);
    add_from(dv, smem + kwv * SHARE, lane, rwv == 1);
    if (rwv == 1) return;
  }
  const int kw = kt * 32 * KW + kwv * 32;
  auto row_of = [&](int r) { return ((int64_t)b * a.Lk + (order ? order[kw + r] : kw + r)) * a.G + g; };
  if (a.splits > 1) {
    float* pk = a.part + sp * 2 * krows * a.D;
    float* pv = pk + krows * a.D;
    auto at = [&](float* base) { return [=](int r) { return kw + r < a.Lk ? base + row_of(r) * a.D : nullptr; }; };
    store_tile<float, DT>(smem + wave * SHARE, dk, a.D, lane, a.scale, seen, at(pk));
    store_tile<float, DT>(smem + wave * SHARE, dv, a.D, lane, 1.f, seen, at(pv));
  } else {
    auto at = [&](void* base) {
      return [=](int r) { return kw + r < a.Lk ? reinterpret_cast<O*>(base) + row_of(r) * a.D : nullptr; };
    };
    store_tile<O, DT>(smem + wave * SHARE, dk, a.D, lane, a.scale, seen, at(a.dk));
    store_tile<O, DT>(smem + wave * SHARE, dv, a.D, lane, 1.f, seen, at(a.dv));
  }
}

// Sum the splits of a gradient in order.  dq partials are in (item, key head, q, r) row order, dk / dv partials in output order.
template <typename T, bool DQ>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XArgs a) {
  const int d4 = a.D / 4, M = a.Lq * a.R;
  const int64_t rows = DQ ? (int64_t)a.B * a.G * M : 2 * (int64_t)a.B * a.Lk * a.G;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * d4) return;
  const int64_t row = i / d4;
  const int d = (int)(i % d4) * 4;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float4 y = *reinterpret_cast<const float4*>(a.part + (s * rows + row) * a.D + d);
    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
  }
  T* p;
  if (DQ) {
    const int bg = (int)(row / M), m = (int)(row % M), g = bg % a.G, b = bg / a.G;
    p = reinterpret_cast<T*>(a.dq) + (((int64_t)b * a.Lq + m / a.R) * a.H + g * a.R + m % a.R) * a.D + d;
  } else {
    const int64_t half = rows / 2;
    p = (row < half ? reinterpret_cast<T*>(a.dk) + row * a.D : reinterpret_cast<T*>(a.dv) + (row - half) * a.D) + d;
  }
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16_rne(x.x, x.y), cvt_pk_bf16_rne(x.z, x.w));
  else *reinterpret_cast<float4*>(p) = x;
}

// fp32 [B, L, Hn, D] -> bf16 planes [3][B][Hn][L][W], features D .. W - 1 zero; rows at or past len[b] are left out (no tile reads
// them).  Up to four tensors a launch (grid z); 10 bytes of memory traffic an element.
struct SplitArgs {
  const float* src[4];
  uint16_t* dst[4];
  const int64_t* len[4];
  const int* order[4];                                   // rows are taken in this order ([B, L]), or as they stand
  int64_t sb[4], sl[4], sh[4];
  int L[4], Hn[4];
  int B, D, W;
};
__global__ __launch_bounds__(256) void xattn_split_kernel(SplitArgs a) {
  const int z = blockIdx.z, L = a.L[z], Hn = a.Hn[z], ppr = a.W / 8;         // 8-feature pieces per row
  const int64_t plane = (int64_t)a.B * Hn * L * a.W;
  for (int bh = blockIdx.y; bh < a.B * Hn; bh += gridDim.y) {
    const int b = bh / Hn, h = bh - b * Hn, n = clamp_len(a.len[z], b, L);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)n * ppr; i += (int64_t)gridDim.x * 256) {
      const int64_t l = i / ppr;
      const int d = (int)(i - l * ppr) * 8;
      float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
      if (d < a.D) {
        const int64_t from = a.order[z] ? a.order[z][(int64_t)b * L + l] : l;
        const float* p = a.src[z] + b * a.sb[z] + from * a.sl[z] + h * a.sh[z] + d;
        u = *reinterpret_cast<const float4*>(p);
        v = *reinterpret_cast<const float4*>(p + 4);
      }
      const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
      bf16x8 q[3];
      split8<true>(x, q);
      uint16_t* o = a.dst[z] + ((int64_t)bh * L + l) * a.W + d;
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(o + k * plane) = q[k];
    }
  }
}

// The keys of an item in a new order: those that are seen first, in their own order, then the others.  order [B, Lk], count [B].
// The other kernels then walk the first count[b] keys, without a mask: keys that it drops cost nothing instead of a whole product
// (8 x 2048 x 1500 x 16 heads, training, one key in four dropped: 541 -> 461 us).  A block orders 2048 keys; those before it, it counts.
__device__ __forceinline__ int zero_bytes(uint32_t x) { return __builtin_popcount(zero_byte_bits(x)); }
__global__ __launch_bounds__(256) void xattn_order_kernel(const uint8_t* mask, int64_t maskb, const int64_t* len, int Lk, int* order, int64_t* count) {
  __shared__ int red[8];
  const int chunks = (Lk + 2047) / 2048, b = blockIdx.x / chunks, k0 = blockIdx.x % chunks * 2048, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = clamp_len(len, b, Lk);
  mask += b * maskb;
  order += (int64_t)b * Lk;
  // seen keys in front of the block: single bytes up to a 16-byte border, then pieces
  const int end = min(k0, n), head = min(end, (int)(-(intptr_t)mask & 15)), pieces = (end - head) / 16;
  int before = 0;
  if (tid < head) before += mask[tid] == 0;
  for (int i = tid; i < pieces; i += 256) {
    const uint4 u = *reinterpret_cast<const uint4*>(mask + head + i * 16);
    before += zero_bytes(u.x) + zero_bytes(u.y) + zero_bytes(u.z) + zero_bytes(u.w);
  }
  if (head + pieces * 16 + tid < end) before += mask[head + pieces * 16 + tid] == 0;
  // a thread's eight keys, and the seen ones among those of the lower lanes
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = k0 + tid * 8 + i;
    seen |= k < n && mask[k] == 0 ? 1u << i : 0u;
  }
  const int mine = __builtin_popcount(seen);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o, 64);
  if (lane == 63) { red[wave] = upto; red[4 + wave] = before; }
  __syncthreads();
  int at = red[4] + red[5] + red[6] + red[7] + upto - mine;
  for (int w = 0; w < wave; ++w) at += red[w];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int k = k0 + tid * 8 + i;
    if (k < Lk) {
      const bool s = (seen >> i) & 1u;
      order[s ? at : Lk - 1 - (k - at)] = k;             // k - at unseen keys stand before an unseen one
      at += s ? 1 : 0;
    }
  }
  if (k0 + 2048 >= Lk && tid == 255) count[b] = at;
}

// How many shares of a long axis (n tiles) give the launch about `want` blocks, each with at least `least` tiles.
int split_count(int64_t blocks, int64_t n, int64_t want, int64_t least) {
  int64_t s = (want + blocks - 1) / blocks;
  const int64_t most = n / least;
  if (s > most) s = most;
  if (s > MAX_SPLITS) s = MAX_SPLITS;
  return s < 1 ? 1 : (int)s;
}
// The same for blocks of 64 and 128 rows, whose shares write (and the join reads) whole tiles of partial results: the count with the
// least expected time, in us -- tile_us a tile of the share, more where blocks wait for a CU (LDS holds one block) or share it (two
// blocks take 1.4 times one's time together), 4 for the launch of the join and 0.8 a MB of partial results.  Measured at 1 / 2 / 4 / 8 shares: 29 x 8 heads of 128, 54 rows x
// 451 keys 17 / 26 / 32 / 47 us, 16 x 8 heads of 64, 60 x 2000 28 / 25 / 23 / 25, 4 x 8 x 64, 60 x 4000 48 / 31 / 21 / 17, 2 x 4 x
// 128, 1000 x 4000 62 / 43 / 35 / 45, fp32 3 x 4 x 64, 400 x 2000 106 / 67 / 46 / 40.
int share_count(int64_t blocks, int64_t n, int at_once, double tile_us, double part_mb) {
  static const int counts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
  int best = 1;
  double least = 1e30;
  for (const int s : counts) {
    if (s > n) break;
    const double load = (double)blocks * s / (at_once == 256 ? 256 : 366), t = (double)((n + s - 1) / s) * tile_us * (load > 1 ? load : 1) + (s > 1 ? 4 + 0.8 * part_mb * s : 0);
    if (t < least) { least = t; best = s; }
  }
  return best;
}
struct Plan { int planes, width, kg, nrt, fwd, dq, kw, nkt, dkv; bool order; };
// Sizes alone decide.  512 blocks are two per CU, and shares are cut to reach that (2 x 65537 keys of one token: 256 blocks, one per CU,
// 110 us, 512 113, 1024 118).  48 x 1000 x 133 bf16 training with shares for 512 / 1024 / 2048 blocks: 74 / 79 /
// 81 us (every share writes its part once more); two key groups from 512 blocks of 128 rows down: 8 x 500 x 700 49 us, from 1024: the
// fp32 forward at 608 blocks 137 -> 155 us (each row of blocks reads all keys).
// fp32 goes through planes where their making (10 bytes of traffic a value, a launch) pays, the fp32 instruction / planes: forward 15 x
// 8 heads of 128, 378 keys, 70 rows 54 / 66 us, 130 rows 71 / 79, 260 rows 104 / 98; 8 x 4 heads of 64, 2000 keys, 200 rows 48.5 / 48.9,
// 400 rows 109 / 70; backward, with the same planes for two kernels more, 15 x 8 x 378 x 128, 70 rows 151 / 142, 8 x 4 x 2000 x 64, 100
// rows 83 / 77; but 30 x 8 heads of 64, 60 keys, 100 rows (9e7 rows x keys x width) 35 / 45, 2 x 4 x 300 x 64, 400 rows (6e7) 50 / 57.
constexpr double PLANES_FROM = 1 << 27;
// A mask's keys are put in order from here on (rows x keys x width of an LDS row, six times that with planes): the ordering is a launch of 3 us.
// One key in four dropped, without / with it, at 1.4e9 (8 x 8 heads x 500 x 700 x 64) 16.5 / 19.1 us, at 4.3e9 (8 x 8 x 1024 x 1024 x
// 64) 28.5 / 28.1 and 107 / 102 (training), at 5.9e9 (4 x 8 x 1024 x 1400 x 128) 37 / 36, at 5.5e9 in planes 171 / 162.  (The rows
// that a mask leaves out are zeros in the tiles otherwise: they cost the product, but little power.)
constexpr double ORDER_FROM = 4294967296.;
Plan make_plan(int B, int Lq, int Lk, int H, int G, int D, int bf16, bool bwd) {
  Plan p;
  const int64_t M = (int64_t)Lq * (H / G), BG = (int64_t)B * G;
  p.width = D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128;
  p.planes = !bf16 && M > (bwd ? 64 : 192) && (double)BG * M * Lk * p.width >= PLANES_FROM ? 3 : 1;
  const int row = stored(p.width) * (bf16 || p.planes == 3 ? 2 : 4) * p.planes;
  p.kg = p.planes == 3 ? 1 : M <= 32 ? 4 : M <= 64 || !bf16 || BG * ((M + 127) / 128) < 512 ? 2 : 1;
  const int rows = 128 / p.kg;
  p.nrt = (int)((M + rows - 1) / rows);
  const int KT = 32 * p.kg * (p.kg == 1 && row <= 256 ? 2 : 1);
  const int64_t kt = (Lk + KT - 1) / KT;
  const int want = row >= 512 || (p.kg == 4 && row >= 256) ? 256 : 512;        // (LDS holds one block of these per CU)
  // (a token over under eight tiles of up to 32 KB is one share: the join is a launch more, 4 us of the host's time.  700 keys of 64 bf16
  // features, shared out / not: 32 x 4 heads 14 / 10 us a call, 10.1 / 8.9 in a graph; 8 x 4 heads 13.5 / 10.9, 9.6 / 10.5)
  if (p.kg == 4) {
    p.fwd = row <= 128 && kt < 8 ? 1 : split_count(BG * p.nrt, kt, want, 2);
    p.dq = split_count(BG * p.nrt, kt, want, 4);
  } else {
    // a tile's two products (the gradient's three) at a CU's share of the matrix rate, 4.5 or 0.6 TFLOP/s, and what is not overlapped
    const double us = 4e-6 * rows * KT * p.width * (p.planes == 3 ? 6 : 1) / (bf16 || p.planes == 3 ? 4.5 : 0.6), mb = 4e-6 * BG * M * D;
    p.fwd = share_count(BG * p.nrt, kt, want, 0.4 + 1.15 * us, mb);
    p.dq = share_count(BG * p.nrt, kt, want, 0.4 + 1.7 * us, mb);
  }
  p.kw = p.planes == 1 && BG * ((Lk + 127) / 128) < 512 ? 2 : 4;
  p.nkt = (Lk + 32 * p.kw - 1) / (32 * p.kw);
  p.order = M > 64 && (bf16 || p.planes == 3) && (double)BG * M * Lk * stored(p.width) * (p.planes == 3 ? 6 : 1) >= ORDER_FROM;
  const int RT = p.planes == 3 ? 32 : 64;
  p.dkv = split_count(BG * p.nkt, (int64_t)((Lq + RT - 1) / RT) * (H / G), row >= 512 ? 256 : 512, 128 / RT);
  return p;
}
int64_t order_bytes(const Plan& p, int B, int Lk) { return p.order ? ((int64_t)4 * B * Lk + 15) / 16 * 16 + ((int64_t)8 * B + 15) / 16 * 16 : 0; }
int64_t plane_bytes(const Plan& p, int B, int L, int Hn) { return p.planes == 3 ? (int64_t)6 * B * L * Hn * p.width : 0; }

// Runs of logical blocks per XCD (see xcd_block): as long as the blocks of one (item, key head), but never fewer than 64 runs
// -- eight per XCD, so that ragged items even out.
dim3 grid_for(XArgs& a) {
  const int64_t per = (int64_t)a.nrt * a.splits, total = per * a.G * a.B;
  int64_t c = total / 64;
  if (c > per) c = per;
  if (c < 1) c = 1;
  a.chunk = (int)c;
  return dim3((unsigned)((total + 8 * c - 1) / (8 * c) * 8 * c));
}

template <typename T, int DT>
void launch_fwd(XArgs& a, const Plan& p, hipStream_t st) {
  const dim3 g = grid_for(a);
  if constexpr (sizeof(T) == 2) {
    if (p.planes == 3) { hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 1, 3, false>), g, dim3(256), 0, st, a); return; }       // (planes are made in order)
    if (p.kg == 1) {
      if (a.order) hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 1, 1, true>), g, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 1, 1, false>), g, dim3(256), 0, st, a);
      return;
    }
    if (a.order) { hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 2, 1, true>), g, dim3(256), 0, st, a); return; }
  }
  if (p.kg == 4) hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 4, 1, false>), g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((xattn_fwd_kernel<T, DT, 2, 1, false>), g, dim3(256), 0, st, a);
}
template <typename T, int DT>
void launch_dq(XArgs& a, const Plan& p, hipStream_t st) {
  const dim3 g = grid_for(a);
  if constexpr (sizeof(T) == 2) {
    if (p.planes == 3) { hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 1, 3, false>), g, dim3(256), 0, st, a); return; }
    if (p.kg == 1) {
      if (a.order) hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 1, 1, true>), g, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 1, 1, false>), g, dim3(256), 0, st, a);
      return;
    }
    if (a.order) { hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 2, 1, true>), g, dim3(256), 0, st, a); return; }
  }
  if (p.kg == 4) hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 4, 1, false>), g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((xattn_dq_kernel<T, DT, 2, 1, false>), g, dim3(256), 0, st, a);
}
template <typename T, int DT>
void launch_dkv(XArgs& a, const Plan& p, hipStream_t st) {
  const dim3 g = grid_for(a);
  if (p.planes == 3) {
    if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((xattn_dkv_kernel<T, DT, 4, 3>), g, dim3(256), 0, st, a);
  } else if (p.kw == 4) hipLaunchKernelGGL((xattn_dkv_kernel<T, DT, 4, 1>), g, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((xattn_dkv_kernel<T, DT, 2, 1>), g, dim3(256), 0, st, a);
}
#define BY_WIDTH(T, CALL)              \
  do {                                 \
    if (a.D <= 32) { CALL(T, 32); }    \
    else if (a.D <= 64) { CALL(T, 64); } \
    else if (a.D <= 96) { CALL(T, 96); } \
    else { CALL(T, 128); }             \
  } while (0)

int check(const styler_xattn_t* x, bool bwd) {
  if (!x || !x->q || !x->k || !x->v || !x->out) return STYLER_EINVAL;
  if (x->B < 1 || x->Lq < 1 || x->Lk < 1 || x->H < 1 || x->G < 1 || x->H % x->G || x->D < 8 || x->D > 128 || x->D % 8) return STYLER_EINVAL;
  if (!(x->scale > 0.f) || x->scale > 3e38f) return STYLER_EINVAL;
  if ((int64_t)x->Lq * (x->H / x->G) > (1 << 30) || (int64_t)x->Lk > (1 << 30)) return STYLER_EINVAL;
  const int es = x->bf16 ? 2 : 4, e16 = 16 / es;
  const int64_t st[] = {x->qb, x->ql, x->qh, x->kb, x->kl, x->kh, x->vb, x->vl, x->vh, x->ob, x->ol, x->oh, x->gb, x->gl, x->gh};
  for (int i = 0; i < (bwd ? 15 : 12); ++i)
    if (st[i] < 0 || st[i] % e16) return STYLER_EALIGN;
  // a tile's rows (128 at most) are addressed with 32-bit byte offsets from the tile's base
  const int64_t rows[] = {x->ql, x->kl, x->vl, bwd ? x->gl : 0};
  for (int64_t r : rows) if (r * es >= (1 << 23)) return STYLER_EINVAL;
  const void* p[] = {x->q, x->k, x->v, x->out, bwd ? x->dout : nullptr, bwd ? x->dq : nullptr, bwd ? x->dk : nullptr, bwd ? x->dv : nullptr};
  for (const void* q : p) if ((uintptr_t)q & 15) return STYLER_EALIGN;
  if (bwd && (!x->dout || !x->dq || !x->dk || !x->dv || !x->lse)) return STYLER_EINVAL;
  const Plan pl = make_plan(x->B, x->Lq, x->Lk, x->H, x->G, x->D, x->bf16, bwd);
  const int64_t bg = (int64_t)x->B * x->G;
  // a launch has fewer than 2^32 threads, the padding of the runs (grid_for: one eighth at most) among them
  if (bg * pl.nrt * (pl.fwd > pl.dq ? pl.fwd : pl.dq) > 0xe00000 || (bwd && bg * pl.nkt * pl.dkv > 0xe00000)) return STYLER_EINVAL;
  return 0;
}
XArgs args(const styler_xattn_t* x) {
  XArgs a = {};
  a.q = x->q; a.k = x->k; a.v = x->v; a.o = x->out; a.out = x->out; a.dout = x->dout; a.dq = x->dq; a.dk = x->dk; a.dv = x->dv;
  a.lse = x->lse; a.len = x->len; a.qlen = x->q_len; a.mask = x->mask; a.maskb = x->maskb;
  a.qb = x->qb; a.ql = x->ql; a.qh = x->qh; a.kb = x->kb; a.kl = x->kl; a.kh = x->kh; a.vb = x->vb; a.vl = x->vl; a.vh = x->vh;
  a.ob = x->ob; a.ol = x->ol; a.oh = x->oh; a.gb = x->gb; a.gl = x->gl; a.gh = x->gh;
  a.sort = (x->len || x->q_len) && x->B > 1 && x->B <= 16 && (int64_t)x->Lq * x->Lk >= 1 << 18;
  a.B = x->B; a.Lq = x->Lq; a.Lk = x->Lk; a.H = x->H; a.G = x->G; a.R = x->H / x->G; a.D = x->D; a.scale = x->scale;
  return a;
}

}  // namespace

extern "C" int64_t styler_cross_attention_workspace_bytes(int B, int Lq, int Lk, int H, int G, int D, int bf16, int masked, int bwd) {
  if (B < 1 || Lq < 1 || Lk < 1 || G < 1 || H < G || H % G || D < 8 || D > 128) return 0;
  const Plan p = make_plan(B, Lq, Lk, H, G, D, bf16, bwd != 0);
  const int64_t qrows = (int64_t)B * H * Lq, krows = (int64_t)B * G * Lk;
  const int64_t kv = 2 * plane_bytes(p, B, Lk, G) + (masked ? order_bytes(p, B, Lk) : 0);
  if (!bwd) return (p.fwd > 1 ? (4 * p.fwd * qrows * (D + 2) + 15) / 16 * 16 : 0) + kv;
  int64_t part = p.dq > 1 ? p.dq * qrows * D : 0;
  const int64_t pkv = p.dkv > 1 ? 2 * p.dkv * krows * D : 0;
  if (pkv > part) part = pkv;                            // the two gradients' launches follow each other: one buffer
  return (4 * (part + (qrows + 3) / 4 * 8) + 15) / 16 * 16 + kv + 2 * plane_bytes(p, B, Lq, H);
}

namespace {
// the tensors' planes, one after the other at `at`
// the seen keys first, if that pays: order and count at `at` (order_bytes), and the rest of the call sees a batch of lengths without a mask
void put_in_order(XArgs& a, const Plan& p, char* at, hipStream_t st) {
  if (!a.mask || !p.order || a.Lk * a.kl * 4 >= (int64_t)1 << 31 || a.Lk * a.vl * 4 >= (int64_t)1 << 31) return;      // (32-bit offsets)
  int* order = (int*)at;
  int64_t* count = (int64_t*)(at + ((int64_t)4 * a.B * a.Lk + 15) / 16 * 16);
  hipLaunchKernelGGL(xattn_order_kernel, dim3((a.Lk + 2047) / 2048 * a.B), dim3(256), 0, st, a.mask, a.maskb, a.len, a.Lk, order, count);
  a.order = order;
  a.len = count;
  a.mask = nullptr;
}
struct SplitJob { const void* src; int64_t sb, sl, sh; int L, Hn; const int64_t* len; const int* order; };
void launch_split(const SplitJob* job, int n, uint16_t* at, const XArgs& a, const Plan& p, hipStream_t st) {
  SplitArgs s = {};
  s.B = a.B; s.D = a.D; s.W = p.width;
  int most = 0, heads = 0;
  for (int i = 0; i < n; ++i) {
    s.src[i] = (const float*)job[i].src; s.dst[i] = at; s.len[i] = job[i].len; s.order[i] = job[i].order;
    s.sb[i] = job[i].sb; s.sl[i] = job[i].sl; s.sh[i] = job[i].sh; s.L[i] = job[i].L; s.Hn[i] = job[i].Hn;
    at += (int64_t)3 * a.B * job[i].L * job[i].Hn * p.width;
    if (job[i].L > most) most = job[i].L;
    if (job[i].Hn > heads) heads = job[i].Hn;
  }
  const int64_t x = ((int64_t)most * (p.width / 8) + 255) / 256, y = (int64_t)a.B * heads;
  hipLaunchKernelGGL(xattn_split_kernel, dim3((unsigned)(x < 1024 ? x : 1024), (unsigned)(y < 65535 ? y : 65535), n), dim3(256), 0, st, s);
}
// tiles come from the tensors themselves, or from their planes
void tiles_from(XArgs& a, const void* x0, int64_t b0, int64_t l0, int64_t h0, const void* x1, int64_t b1, int64_t l1, int64_t h1) {
  a.t0 = x0; a.t0b = b0; a.t0l = l0; a.t0h = h0; a.t0p = 0;
  a.t1 = x1; a.t1b = b1; a.t1l = l1; a.t1h = h1; a.t1p = 0;
}
void tiles_from_planes(XArgs& a, const uint16_t* x0, int L, int Hn, int W) {
  const int64_t plane = (int64_t)a.B * Hn * L * W;
  tiles_from(a, x0, (int64_t)Hn * L * W, W, (int64_t)L * W, x0 + 3 * plane, (int64_t)Hn * L * W, W, (int64_t)L * W);
  a.t0p = a.t1p = plane;
}
}  // namespace

extern "C" int styler_cross_attention(const styler_xattn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check(x, false)) return rc;
  const int64_t need = styler_cross_attention_workspace_bytes(x->B, x->Lq, x->Lk, x->H, x->G, x->D, x->bf16, x->mask != nullptr, 0);
  if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return STYLER_EINVAL;
  const Plan p = make_plan(x->B, x->Lq, x->Lk, x->H, x->G, x->D, x->bf16, false);
  hipStream_t st = (hipStream_t)stream;
  XArgs a = args(x);
  a.nrt = p.nrt; a.splits = p.fwd; a.part = p.fwd > 1 ? (float*)workspace : nullptr;
  char* end = (char*)workspace + need;                   // from the end: the order, the planes
  if (x->mask) put_in_order(a, p, end -= order_bytes(p, x->B, x->Lk), st);
  if (p.planes == 3) {
    uint16_t* planes = (uint16_t*)(end - 2 * plane_bytes(p, x->B, x->Lk, x->G));
    const SplitJob job[2] = {{x->k, x->kb, x->kl, x->kh, x->Lk, x->G, a.len, a.order}, {x->v, x->vb, x->vl, x->vh, x->Lk, x->G, a.len, a.order}};
    launch_split(job, 2, planes, a, p, st);
    tiles_from_planes(a, planes, x->Lk, x->G, p.width);
  } else {
    tiles_from(a, x->k, x->kb, x->kl, x->kh, x->v, x->vb, x->vl, x->vh);
  }
#define FWD(T, W) launch_fwd<T, W>(a, p, st)
  if (x->bf16 || p.planes == 3) BY_WIDTH(uint16_t, FWD); else BY_WIDTH(float, FWD);
#undef FWD
  if (p.fwd > 1) {
    const unsigned blocks = (unsigned)(((int64_t)x->B * x->H * x->Lq + 3) / 4);
#define JOIN(T, W) hipLaunchKernelGGL((xattn_join_kernel<T, stored(W)>), dim3(blocks), dim3(256), 0, st, a)
    if (x->bf16) BY_WIDTH(uint16_t, JOIN); else BY_WIDTH(float, JOIN);
#undef JOIN
  }
  return launch_status();
}

extern "C" int styler_cross_attention_bwd(const styler_xattn_t* x, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check(x, true)) return rc;
  const int64_t need = styler_cross_attention_workspace_bytes(x->B, x->Lq, x->Lk, x->H, x->G, x->D, x->bf16, x->mask != nullptr, 1);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return STYLER_EINVAL;
  const Plan p = make_plan(x->B, x->Lq, x->Lk, x->H, x->G, x->D, x->bf16, true);
  hipStream_t st = (hipStream_t)stream;
  XArgs a = args(x);
  const int64_t qrows = (int64_t)x->B * x->H * x->Lq, krows = (int64_t)x->B * x->G * x->Lk;
  a.delta = (float*)workspace;
  a.lse2 = a.delta + (qrows + 3) / 4 * 4;
  a.part = a.lse2 + (qrows + 3) / 4 * 4;
  const int64_t kvb = 2 * plane_bytes(p, x->B, x->Lk, x->G), qb = 2 * plane_bytes(p, x->B, x->Lq, x->H);
  char* end = (char*)workspace + need;
  if (x->mask) put_in_order(a, p, end -= order_bytes(p, x->B, x->Lk), st);
  uint16_t* planes = (uint16_t*)(end - kvb - qb);        // k, v, q, dout
  if (p.planes == 3) {
    const SplitJob job[4] = {{x->k, x->kb, x->kl, x->kh, x->Lk, x->G, a.len, a.order}, {x->v, x->vb, x->vl, x->vh, x->Lk, x->G, a.len, a.order},
                             {x->q, x->qb, x->ql, x->qh, x->Lq, x->H, x->q_len, nullptr},
                             {x->dout, x->gb, x->gl, x->gh, x->Lq, x->H, x->q_len, nullptr}};
    launch_split(job, 4, planes, a, p, st);
    tiles_from_planes(a, planes, x->Lk, x->G, p.width);
  } else {
    tiles_from(a, x->k, x->kb, x->kl, x->kh, x->v, x->vb, x->vl, x->vh);
  }
  a.nrt = p.nrt; a.splits = p.dq;
#define DQ(T, W) launch_dq<T, W>(a, p, st)
  if (x->bf16 || p.planes == 3) BY_WIDTH(uint16_t, DQ); else BY_WIDTH(float, DQ);
#undef DQ
  if (p.dq > 1) {
    const unsigned blocks = (unsigned)((qrows * (x->D / 4) + 255) / 256);
    if (x->bf16) hipLaunchKernelGGL((xattn_sum_kernel<uint16_t, true>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((xattn_sum_kernel<float, true>), dim3(blocks), dim3(256), 0, st, a);
  }
  if (p.planes == 3) tiles_from_planes(a, planes + kvb / 2, x->Lq, x->H, p.width);
  else tiles_from(a, x->q, x->qb, x->ql, x->qh, x->dout, x->gb, x->gl, x->gh);
  a.nrt = p.nkt; a.splits = p.dkv;
#define DKV(T, W) launch_dkv<T, W>(a, p, st)
  if (x->bf16 || p.planes == 3) BY_WIDTH(uint16_t, DKV); else BY_WIDTH(float, DKV);
#undef DKV
  if (p.dkv > 1) {
    const unsigned blocks = (unsigned)((2 * krows * (x->D / 4) + 255) / 256);
    if (x->bf16) hipLaunchKernelGGL((xattn_sum_kernel<uint16_t, false>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((xattn_sum_kernel<float, false>), dim3(blocks), dim3(256), 0, st, a);
  }
  return launch_status();
}
