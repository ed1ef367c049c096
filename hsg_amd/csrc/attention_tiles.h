// attention_tiles.h -- the kernels of attention.hip, templates over the element type (float, bf16 as hsgk_bf16,
// _Float16) and the padded head width DP (32, 64, 128; float also 96).
//
// Mathematics, per (batch item, key head): rows q_c of the queries that use this key head (column c = query position *
// shared heads + head inside the group), keys k_j, values v_j,
//   s_jc = k_j . q_c,  p_jc = exp2(s_jc * c2 - lse_c),  c2 = scale * log2(e),  lse_c = log2 sum_j exp2(s_jc c2)
//   o_c = sum_j p_jc v_j
//   delta_c = do_c . o_c,  dp_jc = v_j . do_c,  ds_jc = p_jc (dp_jc - delta_c)
//   dq_c = scale sum_j ds_jc k_j,  dk_j = scale sum_c ds_jc q_c,  dv_j = sum_c p_jc do_c
// No score is ever stored: the backward pass recomputes s and p from q, k and lse.
//
// One scheme serves the three kernels.  A wave owns 32 COLUMNS (queries in the forward and dq kernels, keys in the
// dk / dv kernel) whose vectors stay in registers as the B operand of v_mfma_f32_32x32x{2,16}; the other side's rows
// stream through LDS in tiles.  The product comes out with the column in the lane (lane & 31) and the rows in the
// registers, so row statistics, the running maximum and the rescaling are per-lane scalars, and the probabilities are,
// without any exchange between lanes, the B operand of the second product: its contraction runs over the rows in the
// order in which the registers hold them (row (r & 3) + 8 (r >> 2) + 4 (lane >> 5)), and its A operand -- the streamed
// tile, transposed -- is fetched in that same order (ds_read_b64_tr_b16 for 16-bit types, plain 4-byte reads for float).
#pragma once
#include "common.h"

namespace hsgk {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4v = __attribute__((ext_vector_type(4))) float;
using h16x8v = __attribute__((ext_vector_type(8))) _Float16;
using b16x8v = __attribute__((ext_vector_type(8))) __bf16;
using b16x2v = __attribute__((ext_vector_type(2))) __bf16;
using h16x2v = __attribute__((ext_vector_type(2))) _Float16;
using f32x2v = __attribute__((ext_vector_type(2))) float;
typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 tr_h16x4;

struct AttnArgs {
  const void *q, *k, *v, *g, *o;         // g: the gradient of the output; o: the output, contiguous [B,L,H,D]
  int64_t qs[3], ks[3], vs[3], gs[3];    // strides (batch item, row, head) in elements
  const uint8_t *pad;                    // [B,S], nonzero: not a key (null: all are)
  int64_t pad_b;
  int B, L, S, H, G, HG, D, C;           // HG = H / G, C = L * HG columns per key head
  int DL;                                // D rounded up to 16-byte pieces: what the rows of q, k, v and g hold, aligned
  int causal, ovec;                      // ovec: 16-byte pieces of the rows of o are aligned
  float scale, c2;
  void *out;                             // o, or dq, or dk (contiguous)
  void *out2;                            // dv
  float *lse, *delta;                    // [B,G,C]
  int have_delta;                        // whose delta is there before dq: 0 nobody's, 1 everyone's, 2 see attn_dq_kernel
  float *part, *part2, *ml;              // split work: partial sums [splits][B*G][columns][DP], (m, l) [splits][B*G][C][2]
  int splits;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int KS = 8;           // contraction steps of one 16-byte operand pair of lanes
  static constexpr int MMA = 4;          // matrix instructions that take them
};
template <> struct Elem<__bf16> { static constexpr int KS = 16, MMA = 1; };
template <> struct Elem<_Float16> { static constexpr int KS = 16, MMA = 1; };

// The order of READS LDS reads and MMAS matrix instructions of the code before this line: AHEAD reads first, then in turn,
// so that an operand is on its way while the matrix unit works on earlier ones (the compiler alone keeps two in flight; dk
// and dv at width 128, one wave a SIMD: 830 us without, 777 with it; the other kernels gain nothing and lose nothing).
template <int READS, int MMAS, int AHEAD> __device__ __forceinline__ void read_ahead() {
  constexpr int A = AHEAD < READS ? AHEAD : READS, PER = MMAS / READS;
  __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
  for (int i = 0; i < READS - A; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, PER, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, MMAS - (READS - A) * PER, 0);
}

__device__ __forceinline__ void mma(f32x16 &acc, const uint4 &a, const uint4 &b, float) {
  const f32x4v x = __builtin_bit_cast(f32x4v, a), y = __builtin_bit_cast(f32x4v, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16 &acc, const uint4 &a, const uint4 &b, __bf16) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8v, a), __builtin_bit_cast(b16x8v, b), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16 &acc, const uint4 &a, const uint4 &b, _Float16) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8v, a), __builtin_bit_cast(h16x8v, b), acc, 0, 0, 0);
}

// two values rounded to nearest even and packed
__device__ __forceinline__ uint32_t pack2(float x, float y, __bf16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{x, y}, b16x2v));
}
__device__ __forceinline__ uint32_t pack2(float x, float y, _Float16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2v{x, y}, h16x2v));
}

// the B operand of contraction step kk over a block of 32 rows whose values sit in x[16]
template <typename T> __device__ __forceinline__ uint4 row_frag(const float (&x)[16], int kk) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(uint4, f32x4v{x[4 * kk], x[4 * kk + 1], x[4 * kk + 2], x[4 * kk + 3]});
  } else {
    const int r = 8 * kk;
    return uint4{pack2(x[r], x[r + 1], T()), pack2(x[r + 2], x[r + 3], T()), pack2(x[r + 4], x[r + 5], T()),
                 pack2(x[r + 6], x[r + 7], T())};
  }
}

template <typename T> __device__ __forceinline__ float dot_piece(const uint4 &a, const uint4 &b) {
  constexpr int E = 16 / sizeof(T);
  T x[E], y[E];
  __builtin_memcpy(x, &a, 16);
  __builtin_memcpy(y, &b, 16);
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) s = fmaf((float)x[i], (float)y[i], s);
  return s;
}

// A tile of streamed rows in LDS, in 16-byte pieces.  Two kinds of reads have to find their data on different banks: 16
// lanes that take one piece of 16 consecutive rows, and lanes that take 64 bytes of 4 consecutive rows for the transpose
// (16-bit types; float: 128 bytes of one row).  Piece x of row r lies at x ^ swap(r), which serves both.
template <typename T, int DP> struct Tile {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int E = 16 / (int)sizeof(T);          // elements of a piece
  static constexpr int PPR = DP / E;                     // pieces per row
  static constexpr int KK = DP / Elem<T>::KS;            // contraction steps over the head width
  static constexpr int RK = 32 / Elem<T>::KS;            // ... over a block of 32 rows
  static constexpr int DB = DP / 32;
  using Columns = uint4[KK];                             // a lane's share of a column vector, as B operands
  __device__ __forceinline__ static int swap(int r) {    // (depends on r & 15)
    if constexpr (!kHalf) return DP == 32 ? (r >> 1) & 7 : r & 7;
    else if constexpr (DP == 32) return (r >> 2) & 3;
    else if constexpr (DP == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  __device__ __forceinline__ static int piece(int r, int x) { return r * DP + (x ^ swap(r)) * E; }   // element offset
};

// a lane's offsets into a tile: A operands by rows (32 consecutive rows x contraction step over the head width) and by
// columns (32 head elements x contraction step over 32 rows)
template <typename T, int DP> struct Lanes {
  using Ti = Tile<T, DP>;
  int row[Ti::KK], col[Ti::kHalf ? Ti::DB : 2][Ti::kHalf ? 2 : 4];
  __device__ __forceinline__ explicit Lanes(int lane) {
    const int h = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < Ti::KK; ++kk) row[kk] = Ti::piece(lane & 31, 2 * kk + h);
    if constexpr (Ti::kHalf) {
      // 16 lanes hand in the addresses of a 4-row x 16-column patch in 8-byte pieces, lane i of them gets column i
      const int r = 4 * h + ((lane & 15) >> 2);
#pragma unroll
      for (int db = 0; db < Ti::DB; ++db)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          col[db][u] = Ti::piece(r + 8 * u, 4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 4 * (lane & 1);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) col[u][i] = Ti::piece(8 * u + 4 * h + i, (lane & 31) >> 2) + (lane & 3) - 8 * u * DP;
    }
  }
  __device__ __forceinline__ uint4 rows(const T *tile, int row0, int kk) const {
    return *reinterpret_cast<const uint4 *>(tile + row0 * DP + row[kk]);
  }
  __device__ __forceinline__ uint4 cols(const T *tile, int row0, int db, int kk) const {
    if constexpr (Ti::kHalf) {
      const T *p = tile + (row0 + 16 * kk) * DP;
      const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr_h16x4 *)(p + col[db][0]));
      const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr_h16x4 *)(p + col[db][1]));
      const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
      return uint4{a.x, a.y, b.x, b.y};
    } else {
      const float *p = reinterpret_cast<const float *>(tile) + (row0 + 8 * kk) * DP + 32 * db;
      const int *c = col[kk & 1];
      return __builtin_bit_cast(uint4, f32x4v{p[c[0]], p[c[1]], p[c[2]], p[c[3]]});
    }
  }
};

// keeps a rarely taken branch a branch: the compiler would compute both sides of every element
__device__ __forceinline__ void rare() { asm volatile("; rare"); }

// Streamed rows go from memory straight into LDS, 16 bytes a lane (a wave fills 1 KB in lane order, so a lane fetches the
// piece that belongs into its place); no register holds them on the way.  Written as an instruction because the compiler
// would wait for it at the next LDS read, whichever buffer that reads; the loop waits itself (stream()).  m0, which holds the
// place, is the compiler's and is put back (it cannot be named as clobbered).
__device__ __forceinline__ void load_to_lds(const void *from, uint32_t lds_byte) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "s"(lds_byte), "v"(from) : "memory");
}
// (the builtin, not an instruction of ours: the compiler then knows that its own loads from before the loop have arrived and
//  does not wait for them -- and so for the tile under way -- at their first use inside it)
__device__ __forceinline__ void wait_for_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)(p);
}

template <typename T, int DP, int TR> struct Rows {
  using Ti = Tile<T, DP>;
  static constexpr int N = TR * Ti::PPR / 256;
  static_assert(TR * Ti::PPR % 256 == 0, "a tile is a whole number of pieces a thread");
  const T *p[N];
  __device__ __forceinline__ static int row_of(int n) { return ((int)threadIdx.x + 256 * n) / Ti::PPR; }
  __device__ __forceinline__ static int piece_of(int n) {
    return (((int)threadIdx.x + 256 * n) % Ti::PPR) ^ Ti::swap(row_of(n) & 15);
  }
  // a row at or past `end` is fetched as row end - 1: its scores are hidden, and what it holds enters other sums already
  template <typename At> __device__ __forceinline__ void place(At at, int row0, int end) {
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] = at(min(row0 + row_of(n), end - 1)) + piece_of(n) * Ti::E;
  }
  __device__ __forceinline__ void advance(int64_t by) {
#pragma unroll
    for (int n = 0; n < N; ++n) p[n] += by;
  }
  // D: elements of a row rounded up to pieces; the places behind it were zeroed once
  __device__ __forceinline__ void issue(const T *tile, int D) const {
    const uint32_t base = lds_address(tile) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (piece_of(n) * Ti::E < D) load_to_lds(p[n], base + n * 4096);
  }
  // bit n of gone: piece n belongs to a row that nobody sees; it may hold anything and becomes zero
  __device__ __forceinline__ static void clear(T *tile, uint32_t gone) {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if ((gone >> n) & 1) *reinterpret_cast<uint4 *>(tile + ((int)threadIdx.x + 256 * n) * Ti::E) = uint4{0, 0, 0, 0};
  }
};

// 16 bytes of a row from element e0 on, zeros past D
template <typename T> __device__ __forceinline__ uint4 load_piece(const T *row, int e0, int D, bool vec) {
  constexpr int E = 16 / sizeof(T);
  if (vec) return e0 < D ? *reinterpret_cast<const uint4 *>(row + e0) : uint4{0, 0, 0, 0};
  T x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = e0 + i < D ? row[e0 + i] : (T)0.0f;
  uint4 r;
  __builtin_memcpy(&r, x, 16);
  return r;
}

// column vectors of the lane, kept as B operands (D: rounded up to pieces)
template <typename T, int DP>
__device__ __forceinline__ void load_columns(typename Tile<T, DP>::Columns &x, const T *row, int D, int lane) {
#pragma unroll
  for (int kk = 0; kk < Tile<T, DP>::KK; ++kk) {
    const int e0 = kk * Elem<T>::KS + (lane >> 5) * (Elem<T>::KS / 2);
    x[kk] = row && e0 < D ? *reinterpret_cast<const uint4 *>(row + e0) : uint4{0, 0, 0, 0};
  }
}

// maximum and sum over the two lanes that hold a column
__device__ __forceinline__ float both_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

__device__ __forceinline__ void col_of(const AttnArgs &a, int c, int &i, int &hh) {
  if (a.HG == 1) { i = c; hh = 0; } else { i = (int)((unsigned)c / (unsigned)a.HG); hh = c - i * a.HG; }
}

template <typename T> __device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4 *>(p) = float4{a, b, c, d};
  else
    *reinterpret_cast<uint2 *>(p) = uint2{pack2(a, b, T()), pack2(c, d, T())};
}

// one column's result, held as O^T blocks: element 32 db + 8 q + 4 h + i sits in acc[db][4 q + i]
template <typename T, int DB>
__device__ __forceinline__ void store_column(T *row, const f32x16 (&acc)[DB], float f, int D, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = 32 * db + 8 * q + 4 * h;
      const float x[4] = {acc[db][4 * q] * f, acc[db][4 * q + 1] * f, acc[db][4 * q + 2] * f, acc[db][4 * q + 3] * f};
      if ((D & 3) == 0) {
        if (e < D) store4<T>(row + e, x[0], x[1], x[2], x[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e + i < D) row[e + i] = (T)x[i];
      }
    }
}

// power-of-two scale of the columns of ds in float16, whose range ds leaves quickly (it is a probability times a
// gradient): the lane's factor falls whenever a value would pass 2^15, the sums so far follow it exactly
template <typename T, int DB> struct ColumnScale {
  float f = 1.0f;
  __device__ __forceinline__ void start() {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) f = 0x1p100f;
  }
  __device__ __forceinline__ void apply(float (&ds)[16], f32x16 (&acc)[DB]) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
      float top = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
      top = both_max(top);
      if (__any(top * f > 32768.0f)) {
        if (top * f > 32768.0f) {
          int e = 0;
          (void)frexpf(top, &e);
          e = top < __builtin_inff() ? e : 0;
          const float g = ldexpf(1.0f, 13 - e);
          const float d = g / f;
          f = g;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[db][r] *= d;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= f;
    }
  }
};

template <typename T> constexpr float prob_shift() {         // log2 of the factor the probabilities carry into float16
  return sizeof(T) == 2 && !__is_same(T, __bf16) ? 15.0f : 0.0f;
}
// the forward pass scales what it has summed so far only when a maximum has grown by 2^kAttnLazy, so that probabilities may
// reach that meanwhile (a maximum of many columns grows in almost every tile otherwise: 16 heads x 8192 x 8192 causal, width
// 128, bfloat16, 320 us; 301 this way)
constexpr float kAttnLazy = 8.0f;
template <typename T> constexpr float fwd_shift() { return prob_shift<T>() == 0.0f ? 0.0f : prob_shift<T>() - kAttnLazy; }

// A workgroup of four waves with 32 columns each (KW = 1), or with the same 32 columns, each wave on a quarter of every
// tile's rows, their results joined at the end (KW = 4: few columns).
// (Measured and not kept: 64 columns a wave, so that an A operand read from LDS serves two matrix instructions.  bfloat16,
// us for 32, 64 and 2 x 64 columns with halved rows: forward of 16 heads x 8192 x 8192 causal, width 128, 435, 680, 901;
// 96 heads x 785 x 785, width 64, 37, 46, 71.  One wave less a SIMD costs more than the LDS traffic.  Nor two waves for the
// same 32 columns: 34 -> 47 and, 24 heads x 2305 x 2305, 60 -> 87.)
template <typename T, int DP, int KW> struct Shape {
  static constexpr int COLS = 128 / KW;                                            // columns of a workgroup
  static constexpr int TR = KW == 4 ? 128 : sizeof(T) == 4 && DP >= 96 ? 32 : 64;  // streamed rows per tile
  static constexpr int NS = TR / KW / 32;                                          // 32-row blocks of a wave per tile
  static constexpr int TILE = TR * DP * (int)sizeof(T);                            // bytes of one staged tile
  static constexpr int NBUF = 4 * TILE <= 128 * 1024 ? 2 : 1;
  static constexpr int JOIN = KW > 1 ? 4 * 32 * (DP + 1) * 4 : 0;
  static constexpr int LDS = 2 * NBUF * TILE > JOIN ? 2 * NBUF * TILE : JOIN;
  static constexpr bool UNROLL = sizeof(T) == 2;                                   // (float32: bound by its matrix instructions)
  static constexpr int AHEAD = sizeof(T) == 4 ? 4 : 8;                                            // see read_ahead
  // waves of a SIMD that the registers have to leave room for (no more than the LDS does)
  static constexpr int W0 = LDS > 80 * 1024 ? 1 : LDS > 52 * 1024 ? 2 : 3;
  static constexpr int WF = DP == 32 ? W0 : W0 < 2 || (sizeof(T) == 4 && DP >= 96) ? 1 : 2;
  static constexpr int WB = DP >= 96 ? 1 : WF;
};

// partial results of the waves, for the join (the caller synchronises before and after)
template <int DP>
__device__ __forceinline__ void join_put(float *lds, const f32x16 (&acc)[DP / 32], float f, int w, int lane) {
  float *p = lds + (w * 32 + (lane & 31)) * (DP + 1) + 4 * (lane >> 5);
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) p[32 * db + 8 * (r >> 2) + (r & 3)] = acc[db][r] * f;
}
// element d of column col: the sum over the waves that share it, in wave order
template <int DP, int KW> __device__ __forceinline__ float join_get(const float *lds, int col, int d) {
  const float *p = lds + ((col >> 5) * KW * 32 + (col & 31)) * (DP + 1) + d;
  float s = p[0];
#pragma unroll
  for (int k = 1; k < KW; ++k) s += p[k * 32 * (DP + 1)];
  return s;
}

// the tiles of [lo, hi), the first of which is on its way (issue(lo, 0)): the next one is while one is computed on.
// land(buf): what a thread still does to its own share of the tile that has arrived, before the others see it.
template <int TR, int NBUF, bool UNROLL, typename Issue, typename Land, typename Compute>
__device__ __forceinline__ void stream(int lo, int hi, Issue issue, Land land, Compute compute) {
  auto step = [&](int t0, int buf) {
    const bool more = t0 + TR < hi;
    wait_for_lds();
    land(buf);
    __syncthreads();                          // the tile is whole, and nobody reads the other buffer any more
    if (NBUF == 2 && more) issue(t0 + TR, buf ^ 1);
    compute(t0, buf);
    if (NBUF == 1 && more) {
      __syncthreads();
      issue(t0 + TR, 0);
    }
  };
  if (UNROLL && NBUF == 2) {                  // over the buffers, whose addresses are constants then: 4 - 8 % of the forward pass
    for (int t0 = lo; t0 < hi; t0 += 2 * TR) {
      step(t0, 0);
      if (t0 + TR < hi) step(t0 + TR, 1);
    }
  } else {
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += TR) {
      step(t0, buf);
      if (NBUF == 2) buf ^= 1;
    }
  }
  wait_for_lds();                             // (the first tile of an empty range)
}

// zeros where the tiles' rows end before DP
template <int BYTES> __device__ __forceinline__ void clear_tiles(unsigned char *lds, bool narrow) {
  if (!narrow) return;
  for (int t = (int)threadIdx.x * 16; t < BYTES; t += 256 * 16) *reinterpret_cast<uint4 *>(lds + t) = uint4{0, 0, 0, 0};
  __syncthreads();
}

// Which part, column block and (batch item, key head) a workgroup takes.  Workgroup ids are dealt round-robin over the 8
// XCDs, each with an L2 of its own: workgroups that stream the same rows belong on one XCD, and every XCD should get heads of
// every batch item, whose lengths differ.  Without causality a head stays on one XCD, eight heads side by side.  With it the
// blocks differ in work, so the longest of all heads come first and the heads take turns (with 8 heads or a divisor or
// multiple of 8 a head still stays on its XCDs).  Parts of split rows are
// counted from the end that every block sees, so the first parts are whole, and neighbours in the order differ little: within
// an XCD workgroups are placed in order, and one that has to wait holds up the rest (dk and dv of 16 heads on 4, 8192 x 8192,
// width 128: 1.54 times as long with the two parts of a block next to each other).
struct Place {
  int sp, cb, bg;
};
__device__ __forceinline__ Place place_of(const AttnArgs &a, int blocks, bool descending) {
  Place p;
  unsigned id = blockIdx.x;
  if (a.causal) {
    const unsigned heads = (unsigned)(a.B * a.G);
    p.bg = (int)(id % heads);
    id /= heads;
    p.sp = (int)(id / (unsigned)blocks);
    p.cb = (int)(id % (unsigned)blocks);
    if (descending) p.cb = blocks - 1 - p.cb;
  } else {
    const unsigned per = (unsigned)(blocks * a.splits), eights = (unsigned)(a.B * a.G) & ~7u;
    if (id < eights * per) {
      p.bg = (int)((id >> 3) / per * 8 + (id & 7));
      id = (id >> 3) % per;
    } else {
      id -= eights * per;
      p.bg = (int)(eights + id / per);
      id %= per;
    }
    p.sp = (int)(id % (unsigned)a.splits);
    p.cb = (int)(id / (unsigned)a.splits);
  }
  return p;
}

// the keys [lo, hi) of a workgroup with columns c0 .. c0 + cols - 1: its split, what its last query sees; first_limit: the
// last key that its first query sees
__device__ __forceinline__ void key_range(const AttnArgs &a, int sp, int tr, int c0, int cols, int &lo, int &hi, int &first_limit) {
  lo = 0; hi = a.S; first_limit = a.S;
  if (a.splits > 1) {
    const int chunk = ((a.S + a.splits - 1) / a.splits + tr - 1) / tr * tr;
    lo = (int)min((int64_t)sp * chunk, (int64_t)a.S);
    hi = min(lo + chunk, a.S);
  }
  if (a.causal) {
    int il, ih;
    col_of(a, min(c0 + cols, a.C) - 1, il, ih);
    hi = min(hi, il + a.S - a.L + 1);
    col_of(a, c0, il, ih);
    first_limit = il + a.S - a.L;
  }
}

// last + 1 visible key of [lo, hi) (workgroup-uniform; lo when there is none)
__device__ inline int visible_end(const uint8_t *pad, int lo, int hi, int *red) {
  int last = lo;
  for (int j = lo + (int)threadIdx.x; j < hi; j += 256)
    if (!pad[j]) last = j + 1;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const int l = __shfl_xor(last, off);
    last = l > last ? l : last;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = last;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) last = red[w] > last ? red[w] : last;
  return __builtin_amdgcn_readfirstlane(last);
}

// keys and values of one (batch item, key head) on their way into LDS, with the flags of the keys that nobody sees
template <typename T, int DP, int TR> struct KeyRows {
  Rows<T, DP, TR> k, v;
  const T *kb, *vb;
  static constexpr int W = (TR + 63) / 64;
  static_assert(W <= 2, "a tile's flags are two words");
  int flag[W] = {}, left = 0;                           // of the tile on its way: row 64 i + lane is padded; rows up to the end
  uint64_t gone[W] = {};                                // of the tile that has landed: the rows that nobody sees
  __device__ __forceinline__ void issue(const AttnArgs &a, const uint8_t *pad, int lo, int t0, int hi, const T *tk, const T *tv) {
    if (t0 == lo || t0 + TR > hi) {
      k.place([&](int j) { return kb + (int64_t)j * a.ks[1]; }, t0, hi);
      v.place([&](int j) { return vb + (int64_t)j * a.vs[1]; }, t0, hi);
    } else {
      k.advance((int64_t)TR * a.ks[1]);
      v.advance((int64_t)TR * a.vs[1]);
    }
    k.issue(tk, a.DL);
    v.issue(tv, a.DL);
    left = hi - t0;
    if (pad) {                                          // (looked at only when the tile has landed: waiting here cost 40 %)
#pragma unroll
      for (int i = 0; i < W; ++i) flag[i] = pad[min(t0 + 64 * i + (int)(threadIdx.x & 63), hi - 1)];
    }
  }
  __device__ __forceinline__ void land(bool pad, T *tk, T *tv) {
    const int lane = (int)(threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < W; ++i) gone[i] = __ballot(64 * i + lane < TR && (64 * i + lane >= left || flag[i]));
    if (pad && any()) {                                 // (behind the end comes row end - 1, which may be padded)
      uint32_t bits = 0;
#pragma unroll
      for (int n = 0; n < Rows<T, DP, TR>::N; ++n) {
        const int row = Rows<T, DP, TR>::row_of(n);
        bits |= (uint32_t)((word(row >> 6) >> (row & 63)) & 1) << n;
      }
      Rows<T, DP, TR>::clear(tk, bits);
      Rows<T, DP, TR>::clear(tv, bits);
    }
  }
  __device__ __forceinline__ uint64_t word(int i) const { return W == 1 || i == 0 ? gone[0] : gone[W - 1]; }
  __device__ __forceinline__ bool any() const { return gone[0] || gone[W - 1]; }
  // bit (r & 3) + 8 (r >> 2): the lane's row r of the 32 rows from r0 on
  __device__ __forceinline__ uint32_t bits_of(int r0, int h) const { return (uint32_t)(word(r0 >> 6) >> ((r0 & 63) + 4 * h)); }
};
// ---------------------------------------------------------------------------------------------------------------------
// forward: columns = queries, keys and values stream.  Long sequences are bound by the matrix and the vector unit in turn (a
// wave multiplies or takes exponentials, and few waves share a SIMD: 1.3 and 1.6 on average in the next two), medians of ten: 24
// heads x 2305 x 2305, width 64, bfloat16, 57 us, 570 TFLOP/s; 16 heads x 8192 x 8192 causal, width 128, 295 us, 930 TFLOP/s (a
// large matrix product 1130).  float32 adds matrix instructions of a seventh of the rate.  Few queries are bound by the keys and
// values: one token of 16 heads on 4, 2 x 32768 keys, width 128, 25 + 5 us, 5.2 TB/s (a large copy 5.2).
template <typename T, int DP, int KW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Shape<T, DP, KW>::WF)))
void attn_fwd_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, KW>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ float stat[2][4][32];
  __shared__ int red[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const Place at = place_of(a, (a.C + Sh::COLS - 1) / Sh::COLS, true);
  const int b = at.bg / a.G, gh = at.bg - b * a.G;
  const int c0 = at.cb * Sh::COLS, c = c0 + 32 * (w / KW) + (lane & 31);
  const uint8_t *pad = a.pad ? a.pad + (int64_t)b * a.pad_b : nullptr;
  int lo, hi, first_limit;
  key_range(a, at.sp, TR, c0, Sh::COLS, lo, hi, first_limit);
  auto tile = [&](int buf, int which) { return reinterpret_cast<T *>(lds + (2 * buf + which) * Sh::TILE); };
  clear_tiles<2 * Sh::NBUF * Sh::TILE>(lds, a.DL < DP);
  KeyRows<T, DP, TR> st;
  st.kb = static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)gh * a.ks[2];
  st.vb = static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)gh * a.vs[2];
  auto issue = [&](int t0, int buf) { st.issue(a, pad, lo, t0, hi, tile(buf, 0), tile(buf, 1)); };
  if (lo < hi) issue(lo, 0);

  const Lanes<T, DP> ln(lane);
  typename Ti::Columns q;
  int i, hh;
  col_of(a, c < a.C ? c : 0, i, hh);
  load_columns<T, DP>(q, c < a.C ? static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] +
                                       (int64_t)(gh * a.HG + hh) * a.qs[2]
                                 : nullptr, a.DL, lane);
  const int lim = a.causal ? i + a.S - a.L : a.S;                     // the last key that the column sees
  if (pad && lo < hi) hi = visible_end(pad, lo, hi, red);

  f32x16 acc[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) acc[db] = f32x16{0.0f};
  float m = -__builtin_inff(), l = 0.0f;                              // maximum of the scores, this half's sum
  constexpr int X = NS < 2 ? NS : 2;                                  // row blocks at a time
  auto block = [&](int t0, int buf, int r0) {
    const T *tk = tile(buf, 0), *tv = tile(buf, 1);
    float s[X][16];
#pragma unroll
    for (int x = 0; x < X; ++x) {
      f32x16 y = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) mma(y, ln.rows(tk, r0 + 32 * x, kk), q[kk], T());
#pragma unroll
      for (int r = 0; r < 16; ++r) s[x][r] = y[r];
    }
    read_ahead<X * Ti::KK, X * Ti::KK * Elem<T>::MMA, Sh::AHEAD>();
    uint4 fv[Ti::DB];
#pragma unroll
    for (int db = 0; db < Ti::DB; ++db) fv[db] = ln.cols(tv, r0, db, 0);
    if (st.any() || t0 + TR - 1 > first_limit) {
      rare();
#pragma unroll
      for (int x = 0; x < X; ++x) {
        const uint32_t bits = st.bits_of(r0 + 32 * x, h);
        const int row = t0 + r0 + 32 * x + 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int off = (r & 3) + 8 * (r >> 2);
          if (((bits >> off) & 1) || row + off > lim) s[x][r] = -__builtin_inff();
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[x][r]);
    top = both_max(top);
    const float mn = fmaxf(m, top);
    if (__any((mn - m) * a.c2 > kAttnLazy)) {                         // (a column whose maximum stays: factor 1)
      // (the difference of the two references as they are rounded below: of scores around 3000 whose parts are joined here,
      //  exp2((m - mn) c2) would weigh one against the other by 1.5e-4 too much or too little)
      const float f = !(mn > m) ? 1.0f : m == -__builtin_inff() ? 0.0f : exp2f((fwd_shift<T>() - mn * a.c2) - (fwd_shift<T>() - m * a.c2));
      l *= f;
#pragma unroll
      for (int db = 0; db < Ti::DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= f;
      m = mn;
    }
    const float base = m == -__builtin_inff() ? 0.0f : fwd_shift<T>() - m * a.c2;
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[x][r] = __builtin_amdgcn_exp2f(fmaf(s[x][r], a.c2, base));
        l += s[x][r];
      }
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 p = row_frag<T>(s[x], kk);
        const int next = x * Ti::RK + kk + 1;
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) {
          mma(acc[db], fv[db], p, T());
          if (next < X * Ti::RK) fv[db] = ln.cols(tv, r0 + 32 * (next / Ti::RK), db, next % Ti::RK);
        }
      }
  };
  auto compute = [&](int t0, int buf) {
#pragma unroll 1
    for (int x = 0; x < NS; x += X) block(t0, buf, 32 * (NS * (w % KW) + x));
  };
  stream<TR, Sh::NBUF, Sh::UNROLL>(lo, hi, issue, [&](int buf) { st.land(pad, tile(buf, 0), tile(buf, 1)); }, compute);

  l = both_sum(l);
  const float mt = l == 0.0f ? -__builtin_inff() : m * a.c2 - fwd_shift<T>();      // log2 of the factor taken out of l and acc
  auto out_row = [&](int ci, int ch) { return static_cast<T *>(a.out) + (((int64_t)b * a.L + ci) * a.H + gh * a.HG + ch) * a.D; };
  const int64_t first = (int64_t)at.bg * a.C, part = (int64_t)at.sp * a.B * a.G * a.C;
  if constexpr (KW > 1) {
    float *jo = reinterpret_cast<float *>(lds);
    __syncthreads();
    if (h == 0) { stat[0][w][lane] = mt; stat[1][w][lane] = l; }
    __syncthreads();
    auto top = [&](int w0, int col) {                                 // over the waves that share the column
      float x = stat[0][w0][col];
#pragma unroll
      for (int k = 1; k < KW; ++k) x = fmaxf(x, stat[0][w0 + k][col]);
      return x;
    };
    const float M = top(w / KW * KW, lane & 31);
    join_put<DP>(jo, acc, exp2f(mt - (M == -__builtin_inff() ? 0.0f : M)), w, lane);
    __syncthreads();
    for (int t = threadIdx.x; t < Sh::COLS * DP; t += 256) {
      const int col = t / DP, d = t % DP, cc = c0 + col, w0 = (col >> 5) * KW;
      if (cc >= a.C) continue;
      float MM = top(w0, col & 31), L = 0.0f;
      const bool none = MM == -__builtin_inff();
      if (none) MM = 0.0f;
#pragma unroll
      for (int k = 0; k < KW; ++k) L += stat[1][w0 + k][col & 31] * exp2f(stat[0][w0 + k][col & 31] - MM);
      const float o = join_get<DP, KW>(jo, col, d);
      if (a.splits > 1) {
        a.part[(part + first + cc) * DP + d] = o;
        if (d == 0) { a.ml[2 * (part + first + cc)] = none ? -__builtin_inff() : MM; a.ml[2 * (part + first + cc) + 1] = L; }
      } else {
        int ci, ch;
        col_of(a, cc, ci, ch);
        if (d < a.D) out_row(ci, ch)[d] = (T)(L == 0.0f ? 0.0f : o / L);
        if (d == 0 && a.lse) a.lse[first + cc] = L == 0.0f ? __builtin_inff() : MM + log2f(L);
      }
    }
  } else if (c < a.C) {
    if (a.splits > 1) {
      store_column<float, Ti::DB>(a.part + (part + first + c) * DP, acc, 1.0f, DP, lane);
      if (h == 0) { a.ml[2 * (part + first + c)] = mt; a.ml[2 * (part + first + c) + 1] = l; }
    } else {
      store_column<T, Ti::DB>(out_row(i, hh), acc, l == 0.0f ? 0.0f : 1.0f / l, a.D, lane);
      if (h == 0 && a.lse) a.lse[first + c] = l == 0.0f ? __builtin_inff() : mt + log2f(l);
    }
  }
}

// joins the splits of the forward kernel: a workgroup per column; its threads are DP head elements x shares of the parts
constexpr int kAttnMaxSplits = 256;
template <typename T, int DP> __global__ __launch_bounds__(256) void attn_fwd_join_kernel(const AttnArgs a) {
  constexpr int Y = 256 / DP;
  __shared__ float red[Y][DP], wt[kAttnMaxSplits], rm[4], rl[4];
  const int64_t at = blockIdx.x, n = (int64_t)a.B * a.G * a.C;
  const int t = threadIdx.x, d = t % DP, y = t / DP;
  float mt = -__builtin_inff(), l = 0.0f;
  if (t < a.splits) { mt = a.ml[2 * (t * n + at)]; l = a.ml[2 * (t * n + at) + 1]; }
  float M = mt;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
  if ((t & 63) == 0) rm[t >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
  if (M == -__builtin_inff()) M = 0.0f;
  const float f = exp2f(mt - M);
  wt[t] = f;
  l *= f;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off);
  if ((t & 63) == 0) rl[t >> 6] = l;
  __syncthreads();
  const float L = (rl[0] + rl[1]) + (rl[2] + rl[3]);
  float o = 0.0f;
#pragma unroll 8
  for (int s = y; s < a.splits; s += Y) o = fmaf(a.part[(s * n + at) * DP + d], wt[s], o);
  if (y < Y) red[y][d] = o;                                           // (256 is no multiple of 96)
  __syncthreads();
  if (y) return;
  for (int x = 1; x < Y; ++x) o += red[x][d];
  const int bg = (int)(at / a.C), c = (int)(at % a.C), b = bg / a.G, gh = bg % a.G;
  int i, hh;
  col_of(a, c, i, hh);
  if (d < a.D) static_cast<T *>(a.out)[(((int64_t)b * a.L + i) * a.H + gh * a.HG + hh) * a.D + d] = (T)(L == 0.0f ? 0.0f : o / L);
  if (d == 0 && a.lse) a.lse[at] = L == 0.0f ? __builtin_inff() : M + log2f(L);
}

// ... the same for few parts of many columns: a thread per four head elements (20480 columns of width 64 in 2 parts: 5 us, 21
// with a workgroup per column)
constexpr int kAttnFewSplits = 8;
template <typename T, int DP> __global__ __launch_bounds__(256) void attn_fwd_join_few_kernel(const AttnArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.B * a.G * a.C, at = t / (DP / 4);
  const int d = (int)(t % (DP / 4)) * 4;
  if (at >= n || d >= a.D) return;
  float M = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.ml[2 * (s * n + at)]);
  if (M == -__builtin_inff()) M = 0.0f;
  float L = 0.0f;
  f32x4v o = f32x4v{0.0f};
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2f(a.ml[2 * (s * n + at)] - M);
    L = fmaf(a.ml[2 * (s * n + at) + 1], f, L);
    o += *reinterpret_cast<const f32x4v *>(a.part + (s * n + at) * DP + d) * f;
  }
  const int bg = (int)(at / a.C), c = (int)(at % a.C), b = bg / a.G, gh = bg % a.G;
  int i, hh;
  col_of(a, c, i, hh);
  T *to = static_cast<T *>(a.out) + (((int64_t)b * a.L + i) * a.H + gh * a.HG + hh) * a.D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (d + e < a.D) to[e] = (T)(L == 0.0f ? 0.0f : o[e] / L);
  if (d == 0 && a.lse) a.lse[at] = L == 0.0f ? __builtin_inff() : M + log2f(L);
}

// ---------------------------------------------------------------------------------------------------------------------
// dq, or with SUM delta alone: columns = queries, keys and values stream; three products, bound like the forward pass (the
// two shapes there: 75 us, 650 TFLOP/s, and 413 us, 1000 TFLOP/s)
//
// delta = do . o carries the rounding of a 16-bit o: as much as one of do . v, while what is left of dp - delta over few
// keys is no more (relative error of dq against 64 bits, where rounding the exact dq gives 1: 2.3 for 2 keys, 1.55 for 16,
// 1.46 for 128, more where values have a common part).  It enters dq times the mean key, which narrow heads follow closely
// (width 24, 451 keys: 1.49).  Queries that see at most exact_keys() keys therefore get delta = sum p dp, summed in float32
// by a launch of its own, whose two products they can afford (1.43 then; 96 heads x 197 x 197, width 64, bfloat16: 11 us
// beside 12 + 14 + 15 for forward, dq, dk and dv; 40 heads x 451 x 451, width 24, float16: 9 us beside 12 + 12 + 13).
constexpr int exact_keys(int padded_width) { return padded_width == 32 ? 4096 : 256; }

template <typename T, int DP, int KW, bool SUM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Shape<T, DP, KW>::WF)))
void attn_dq_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, KW>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ int red[4];
  __shared__ float dsum[SUM && KW > 1 ? 4 : 1][32];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const Place at = place_of(a, (a.C + Sh::COLS - 1) / Sh::COLS, true);
  const int b = at.bg / a.G, gh = at.bg - b * a.G;
  const int c0 = at.cb * Sh::COLS, c = c0 + 32 * (w / KW) + (lane & 31);
  const bool mine = c < a.C;
  const uint8_t *pad = a.pad ? a.pad + (int64_t)b * a.pad_b : nullptr;
  int lo, hi, first_limit;
  key_range(a, at.sp, TR, c0, Sh::COLS, lo, hi, first_limit);
  int last, last_h;                                                   // 2: whose last query sees few keys, whatever the split
  col_of(a, min(c0 + Sh::COLS, a.C) - 1, last, last_h);
  const bool there = a.have_delta == 1 || (a.have_delta == 2 && last + a.S - a.L < exact_keys(DP));
  if (SUM && !there) return;
  auto tile = [&](int buf, int which) { return reinterpret_cast<T *>(lds + (2 * buf + which) * Sh::TILE); };
  clear_tiles<2 * Sh::NBUF * Sh::TILE>(lds, a.DL < DP);
  KeyRows<T, DP, TR> st;
  st.kb = static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)gh * a.ks[2];
  st.vb = static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)gh * a.vs[2];
  auto issue = [&](int t0, int buf) { st.issue(a, pad, lo, t0, hi, tile(buf, 0), tile(buf, 1)); };
  if (lo < hi) issue(lo, 0);

  const Lanes<T, DP> ln(lane);
  typename Ti::Columns q, g;
  int i, hh;
  col_of(a, mine ? c : 0, i, hh);
  const int head = gh * a.HG + hh;
  load_columns<T, DP>(q, mine ? static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)head * a.qs[2]
                              : nullptr, a.DL, lane);
  load_columns<T, DP>(g, mine ? static_cast<const T *>(a.g) + (int64_t)b * a.gs[0] + (int64_t)i * a.gs[1] + (int64_t)head * a.gs[2]
                              : nullptr, a.DL, lane);
  const int64_t row_at = (((int64_t)b * a.L + i) * a.H + head) * a.D, col_at = (int64_t)at.bg * a.C + c;
  const int lim = a.causal ? i + a.S - a.L : a.S;
  const float lse = mine ? a.lse[col_at] : __builtin_inff();
  if (pad && lo < hi) hi = visible_end(pad, lo, hi, red);
  const bool exact = SUM && hi - lo <= exact_keys(DP);
  float delta = 0.0f;
  if (!SUM && there) {
    if (mine) delta = a.delta[col_at];
  } else if (!exact) {
    if (mine) {
      const T *orow = static_cast<const T *>(a.o) + row_at;
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk)
        delta += dot_piece<T>(g[kk], load_piece<T>(orow, kk * Elem<T>::KS + h * (Elem<T>::KS / 2), a.D, a.ovec));
    }
    delta = both_sum(delta);
    if (mine && h == 0 && at.sp == 0 && w % KW == 0) a.delta[col_at] = delta;
    if (SUM) {
      wait_for_lds();                                                 // (the first tile is on its way)
      return;
    }
  }
  float sum = 0.0f;

  f32x16 acc[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) acc[db] = f32x16{0.0f};
  ColumnScale<T, Ti::DB> cs;
  cs.start();
  auto compute = [&](int t0, int buf) {
    const T *tk = tile(buf, 0), *tv = tile(buf, 1);
    const bool some_hidden = st.any() || t0 + TR - 1 > first_limit;
#pragma unroll 1
    for (int n = 0; n < NS; ++n) {
      const int r0 = 32 * (NS * (w % KW) + n);
      f32x16 x = f32x16{0.0f}, y = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) {
        mma(x, ln.rows(tk, r0, kk), q[kk], T());
        mma(y, ln.rows(tv, r0, kk), g[kk], T());
      }
      read_ahead<2 * Ti::KK, 2 * Ti::KK * Elem<T>::MMA, Sh::AHEAD>();
      uint4 fk[Ti::DB];
#pragma unroll
      for (int db = 0; db < Ti::DB; ++db) fk[db] = ln.cols(tk, r0, db, 0);
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c2, -lse)) * (y[r] - delta);
      if (some_hidden) {
        rare();
        const uint32_t bits = st.bits_of(r0, h);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int row = 8 * r4 + 4 * h;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (((bits >> (8 * r4 + e)) & 1) || t0 + r0 + row + e > lim) ds[4 * r4 + e] = 0.0f;
        }
      }
      if constexpr (SUM) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += ds[r];
        continue;
      }
      cs.apply(ds, acc);
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 p = row_frag<T>(ds, kk);
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) {
          mma(acc[db], fk[db], p, T());
          if (kk + 1 < Ti::RK) fk[db] = ln.cols(tk, r0, db, kk + 1);
        }
      }
    }
  };
  stream<TR, Sh::NBUF, Sh::UNROLL>(lo, hi, issue, [&](int buf) { st.land(pad, tile(buf, 0), tile(buf, 1)); }, compute);
  if constexpr (SUM) {
    delta = both_sum(sum);
    if constexpr (KW > 1) {
      if (h == 0) dsum[w][lane] = delta;
      __syncthreads();
      delta = (dsum[0][lane & 31] + dsum[1][lane & 31]) + (dsum[2][lane & 31] + dsum[3][lane & 31]);
    }
    if (mine && h == 0 && w % KW == 0) a.delta[col_at] = delta;
    return;
  }

  const float f = a.scale / cs.f;
  const int64_t part = (int64_t)at.sp * a.B * a.G * a.C;
  if constexpr (KW > 1) {
    float *jo = reinterpret_cast<float *>(lds);
    __syncthreads();
    join_put<DP>(jo, acc, f, w, lane);
    __syncthreads();
    for (int t = threadIdx.x; t < Sh::COLS * DP; t += 256) {
      const int col = t / DP, d = t % DP, cc = c0 + col;
      if (cc >= a.C || d >= a.D) continue;
      const float o = join_get<DP, KW>(jo, col, d);
      int ci, ch;
      col_of(a, cc, ci, ch);
      if (a.splits > 1) a.part[(part + (int64_t)at.bg * a.C + cc) * DP + d] = o;
      else static_cast<T *>(a.out)[(((int64_t)b * a.L + ci) * a.H + gh * a.HG + ch) * a.D + d] = (T)o;
    }
  } else if (mine) {
    if (a.splits > 1) store_column<float, Ti::DB>(a.part + (part + col_at) * DP, acc, f, DP, lane);
    else store_column<T, Ti::DB>(static_cast<T *>(a.out) + row_at, acc, f, a.D, lane);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// dk and dv: columns = keys, the queries that use this key head and their output gradients stream; the heads of a group are
// rows of the same stream, so shared heads are summed here, in a fixed order and without atomics.  Four products; the two
// shapes above: 89 us, 730 TFLOP/s, and 784 us, 700 TFLOP/s (at width 128 the sums of dk and dv leave registers for one wave
// a SIMD, which waits for its own exponentials).  Shared columns at width 128 do not fit the registers: float32 spills 173 of
// 512 (16 heads x 256 x 256: 40 us beside 22 for forward and 27 for dq), the 16-bit types 17 and 20 (16 us beside 14 and 11).
template <typename T, int DP, int KW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Shape<T, DP, KW>::WB)))
void attn_dkv_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, KW>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ __attribute__((aligned(16))) float slse[Sh::NBUF][TR], sdel[Sh::NBUF][TR];
  __shared__ __attribute__((aligned(16))) int slim[Sh::NBUF][TR];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const Place at = place_of(a, (a.S + Sh::COLS - 1) / Sh::COLS, false);          // (the first keys are seen by the most queries)
  const int b = at.bg / a.G, gh = at.bg - b * a.G;
  const int j0 = at.cb * Sh::COLS, j = j0 + 32 * (w / KW) + (lane & 31);
  const bool mine = j < a.S, seen = mine && !(a.pad && a.pad[(int64_t)b * a.pad_b + j]);
  // columns (queries) of this workgroup
  int lo = 0, hi = a.C;
  if (a.splits > 1) {
    const int chunk = ((a.C + a.splits - 1) / a.splits + TR - 1) / TR * TR;
    hi = (int)max(a.C - (int64_t)at.sp * chunk, (int64_t)0);
    lo = max(hi - chunk, 0);
  }
  if (a.causal) {                                                     // the first query that sees key j0
    const int64_t i0 = (int64_t)j0 - (a.S - a.L);
    if (i0 > 0) lo = (int)max((int64_t)lo, min(i0 * a.HG, (int64_t)a.C));
  }
  auto tile = [&](int buf, int which) { return reinterpret_cast<T *>(lds + (2 * buf + which) * Sh::TILE); };
  clear_tiles<2 * Sh::NBUF * Sh::TILE>(lds, a.DL < DP);
  Rows<T, DP, TR> sq, sg;
  float rl = 0.0f, rd = 0.0f;
  int rlim = 0;
  const bool even = TR % a.HG == 0;                                   // a tile is a whole number of query positions
  const T *qb = static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)gh * a.HG * a.qs[2];
  const T *gb = static_cast<const T *>(a.g) + (int64_t)b * a.gs[0] + (int64_t)gh * a.HG * a.gs[2];
  const float *lb = a.lse + (int64_t)at.bg * a.C, *db_ = a.delta + (int64_t)at.bg * a.C;
  auto issue = [&](int t0, int buf) {
    if (t0 == lo || t0 + TR > hi || !even) {
      sq.place([&](int c) { int i, hh; col_of(a, c, i, hh); return qb + (int64_t)i * a.qs[1] + (int64_t)hh * a.qs[2]; }, t0, hi);
      sg.place([&](int c) { int i, hh; col_of(a, c, i, hh); return gb + (int64_t)i * a.gs[1] + (int64_t)hh * a.gs[2]; }, t0, hi);
    } else {
      const int64_t by = TR / a.HG;
      sq.advance(by * a.qs[1]);
      sg.advance(by * a.gs[1]);
    }
    sq.issue(tile(buf, 0), a.DL);
    sg.issue(tile(buf, 1), a.DL);
    if ((int)threadIdx.x < TR) {
      const int c = t0 + (int)threadIdx.x;
      rl = c < hi ? lb[c] : __builtin_inff();
      rd = c < hi ? db_[c] : 0.0f;
      int i, hh;
      col_of(a, c, i, hh);
      rlim = a.causal ? i + a.S - a.L : a.S;
    }
  };
  if (lo < hi) issue(lo, 0);
  const Lanes<T, DP> ln(lane);
  typename Ti::Columns k, v;
  load_columns<T, DP>(k, seen ? static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)j * a.ks[1] + (int64_t)gh * a.ks[2]
                              : nullptr, a.DL, lane);
  load_columns<T, DP>(v, seen ? static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)j * a.vs[1] + (int64_t)gh * a.vs[2]
                              : nullptr, a.DL, lane);
  if (a.pad && !__builtin_amdgcn_readfirstlane(__syncthreads_or(seen))) hi = lo;   // all of its keys are padding

  f32x16 ak[Ti::DB], av[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) { ak[db] = f32x16{0.0f}; av[db] = f32x16{0.0f}; }
  ColumnScale<T, Ti::DB> cs;
  cs.start();
  auto compute = [&](int t0, int buf) {
    const T *tq = tile(buf, 0), *tg = tile(buf, 1);
    int il = 0, ih;
    if (a.causal) col_of(a, t0, il, ih);                              // (the tile's first query)
    const bool some_hidden = a.causal && j0 + Sh::COLS - 1 > il + a.S - a.L;
#pragma unroll 1
    for (int n = 0; n < NS; ++n) {
      const int r0 = 32 * (NS * (w % KW) + n);
      f32x16 x = f32x16{0.0f}, y = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) {
        mma(x, ln.rows(tq, r0, kk), k[kk], T());
        mma(y, ln.rows(tg, r0, kk), v[kk], T());
      }
      read_ahead<2 * Ti::KK, 2 * Ti::KK * Elem<T>::MMA, Sh::AHEAD>();
      uint4 fg[Ti::DB], fq[Ti::DB];
#pragma unroll
      for (int db = 0; db < Ti::DB; ++db) { fg[db] = ln.cols(tg, r0, db, 0); fq[db] = ln.cols(tq, r0, db, 0); }
      float p[16], ds[16];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int row = r0 + 8 * r4 + 4 * h;
        const float4 ls = *reinterpret_cast<const float4 *>(&slse[buf][row]);
        const float4 de = *reinterpret_cast<const float4 *>(&sdel[buf][row]);
        const float lx[4] = {ls.x, ls.y, ls.z, ls.w}, dx[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * r4 + e] = __builtin_amdgcn_exp2f(fmaf(x[4 * r4 + e], a.c2, -lx[e]));
          ds[4 * r4 + e] = y[4 * r4 + e] - dx[e];
        }
      }
      if (some_hidden) {
        rare();
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int4 lm = *reinterpret_cast<const int4 *>(&slim[buf][r0 + 8 * r4 + 4 * h]);
          const int mx[4] = {lm.x, lm.y, lm.z, lm.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j > mx[e]) { p[4 * r4 + e] = 0.0f; ds[4 * r4 + e] = 0.0f; }
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        ds[r] *= p[r];
        if (prob_shift<T>() != 0.0f) p[r] *= 32768.0f;                // (the probability in a float16 product carries 2^15)
      }
      cs.apply(ds, ak);
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 pf = row_frag<T>(p, kk), df = row_frag<T>(ds, kk);
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) {
          mma(av[db], fg[db], pf, T());
          mma(ak[db], fq[db], df, T());
          if (kk + 1 < Ti::RK) { fg[db] = ln.cols(tg, r0, db, kk + 1); fq[db] = ln.cols(tq, r0, db, kk + 1); }
        }
      }
    }
  };
  stream<TR, Sh::NBUF, Sh::UNROLL>(
      lo, hi, issue,
      [&](int buf) {
        if ((int)threadIdx.x < TR) { slse[buf][threadIdx.x] = rl; sdel[buf][threadIdx.x] = rd; slim[buf][threadIdx.x] = rlim; }
      },
      compute);

  // (a padded key's lane has computed with zeros for its key and value: its sums are dropped)
  const float fk = a.scale / cs.f, fv = exp2f(-prob_shift<T>());
  if (!seen) {
#pragma unroll
    for (int db = 0; db < Ti::DB; ++db) { ak[db] = f32x16{0.0f}; av[db] = f32x16{0.0f}; }
  }
  const int64_t part = ((int64_t)at.sp * a.B * a.G + at.bg) * a.S;
  if constexpr (KW > 1) {
    float *jo = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      join_put<DP>(jo, which ? av : ak, which ? fv : fk, w, lane);
      __syncthreads();
      for (int t = threadIdx.x; t < Sh::COLS * DP; t += 256) {
        const int col = t / DP, d = t % DP, jj = j0 + col;
        if (jj >= a.S || d >= a.D) continue;
        const float o = join_get<DP, KW>(jo, col, d);
        if (a.splits > 1) (which ? a.part2 : a.part)[(part + jj) * DP + d] = o;
        else static_cast<T *>(which ? a.out2 : a.out)[(((int64_t)b * a.S + jj) * a.G + gh) * a.D + d] = (T)o;
      }
    }
  } else if (mine) {
    if (a.splits > 1) {
      store_column<float, Ti::DB>(a.part + (part + j) * DP, ak, fk, DP, lane);
      store_column<float, Ti::DB>(a.part2 + (part + j) * DP, av, fv, DP, lane);
    } else {
      const int64_t row = (((int64_t)b * a.S + j) * a.G + gh) * a.D;
      store_column<T, Ti::DB>(static_cast<T *>(a.out) + row, ak, fk, a.D, lane);
      store_column<T, Ti::DB>(static_cast<T *>(a.out2) + row, av, fv, a.D, lane);
    }
  }
}

// sums the splits' partial gradients, in order: columns `n` per (batch item, key head); rows of `out` are
// [B, n / per, heads, D] with `per` columns (shared heads) next to each other
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float *part, int splits, int B, int G, int n, int per, int D,
                                                       T *out) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)B * G * n;
  const int64_t at = t / (DP / 4);
  const int d = (int)(t % (DP / 4)) * 4;
  if (at >= rows || d >= D) return;
  f32x4v s = f32x4v{0.0f};
  for (int x = 0; x < splits; ++x) s += *reinterpret_cast<const f32x4v *>(part + (x * rows + at) * DP + d);
  const int bg = (int)(at / n), c = (int)(at % n), b = bg / G, gh = bg % G;
  T *to = out + ((((int64_t)b * (n / per) + c / per) * G + gh) * per + c % per) * D + d;
  if (D % 4 == 0) {
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)s[e];
    __builtin_memcpy(__builtin_assume_aligned(to, 4 * sizeof(T)), y, sizeof(y));
  } else {
    for (int e = 0; e < 4 && d + e < D; ++e) to[e] = (T)s[e];
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------
enum AttnPass { kAttnFwd, kAttnDelta, kAttnDq, kAttnDkv };
// columns of a workgroup: 32 that its waves share, or 128
enum AttnShape { kAttnShared, kAttnWide };

template <typename T, int DP, int KW, bool DKV> void attn_launch(AttnPass pass, const AttnArgs &a, hipStream_t s) {
  const int cols = DKV ? a.S : a.C, per = Shape<T, DP, KW>::COLS;
  const unsigned grid = (unsigned)((int64_t)a.B * a.G * ((cols + per - 1) / per) * a.splits);
  if constexpr (DKV) {
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP, KW>), dim3(grid), dim3(256), 0, s, a);
  } else if (pass == kAttnFwd) {
    hipLaunchKernelGGL((attn_fwd_kernel<T, DP, KW>), dim3(grid), dim3(256), 0, s, a);
  } else if (pass == kAttnDq) {
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, KW, false>), dim3(grid), dim3(256), 0, s, a);
  } else if constexpr (sizeof(T) == 2) {
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, KW, true>), dim3(grid), dim3(256), 0, s, a);
  }
}

template <typename T, int DP, bool DKV> int attn_run(AttnPass pass, const AttnArgs &a, AttnShape shape, hipStream_t s) {
  if (shape == kAttnWide) attn_launch<T, DP, 1, DKV>(pass, a, s);
  else attn_launch<T, DP, 4, DKV>(pass, a, s);
  HSGK_LAUNCH_CHECK();
  if (a.splits > 1) {
    const int n = DKV ? a.S : a.C, per = DKV ? 1 : a.HG;
    const int64_t rows = (int64_t)a.B * a.G * n;
    const unsigned grid = (unsigned)((rows * (DP / 4) + 255) / 256);
    if (pass == kAttnFwd && a.splits <= kAttnFewSplits)
      hipLaunchKernelGGL((attn_fwd_join_few_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a);
    else if (pass == kAttnFwd)
      hipLaunchKernelGGL((attn_fwd_join_kernel<T, DP>), dim3((unsigned)rows), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a.part, a.splits, a.B, a.G, n, per, a.D,
                         static_cast<T *>(a.out));
    if (DKV)
      hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a.part2, a.splits, a.B, a.G, n, per, a.D,
                         static_cast<T *>(a.out2));
    HSGK_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T, bool DKV> int attn_type(AttnPass pass, const AttnArgs &a, AttnShape shape, hipStream_t s) {
  if (a.D <= 32) return attn_run<T, 32, DKV>(pass, a, shape, s);
  if (a.D <= 64) return attn_run<T, 64, DKV>(pass, a, shape, s);
  if constexpr (sizeof(T) == 4) {
    if (a.D <= 96) return attn_run<T, 96, DKV>(pass, a, shape, s);
  }
  return attn_run<T, 128, DKV>(pass, a, shape, s);
}

// one translation unit a type and side, so that they build next to each other
#define HSGK_ATTN(name) int name(AttnPass pass, const AttnArgs &a, AttnShape shape, hipStream_t s)
HSGK_ATTN(attn_f32);
HSGK_ATTN(attn_bf16);
HSGK_ATTN(attn_f16);
HSGK_ATTN(attn_dkv_f32);
HSGK_ATTN(attn_dkv_bf16);
HSGK_ATTN(attn_dkv_f16);

}  // namespace hsgk
