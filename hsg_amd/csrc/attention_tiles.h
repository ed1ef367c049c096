// attention_tiles.h -- the kernels of attention.hip, templates over the element type (float, bf16 as hsgk_bf16,
// _Float16) and the padded head width DP (32, 64, 128).
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
  int causal, qvec, kvec, vvec, gvec, ovec;   // *vec: 16-byte pieces of that tensor's rows are aligned
  float scale, c2;
  void *out;                             // o, or dq, or dk (contiguous)
  void *out2;                            // dv
  float *lse, *delta;                    // [B,G,C]
  float *part, *part2, *ml;              // split work: partial sums [splits][B*G][columns][DP], (m, l) [splits][B*G][C][2]
  int splits;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int KS = 8;           // contraction steps of one 16-byte operand pair of lanes
};
template <> struct Elem<__bf16> { static constexpr int KS = 16; };
template <> struct Elem<_Float16> { static constexpr int KS = 16; };

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

// 16 bytes of a row from element e0 on, zeros past D
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *row, int e0, int D, bool vec) {
  constexpr int E = 16 / sizeof(T);
  if (vec) {                                  // D is a multiple of E: the piece is all inside or all outside
    return e0 < D ? *reinterpret_cast<const uint4 *>(row + e0) : uint4{0, 0, 0, 0};
  }
  T x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = e0 + i < D ? row[e0 + i] : (T)0.0f;
  uint4 r;
  __builtin_memcpy(&r, x, 16);
  return r;
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

// workgroup ids are dealt round-robin over the 8 XCDs: consecutive logical ids (the column blocks that stream the same
// rows) go to ONE XCD and its L2
__device__ __forceinline__ unsigned xcd_order(unsigned id, unsigned n) {
  const unsigned x = id & 7, per = n >> 3, rem = n & 7;
  return x * per + (x < rem ? x : rem) + (id >> 3);
}

template <typename T, int DP> struct Tile {
  static constexpr int E = 16 / (int)sizeof(T);          // elements of a 16-byte piece
  static constexpr int RS = DP + E;                      // LDS row stride: pieces of consecutive rows on different banks
  static constexpr int KK = DP / Elem<T>::KS;            // contraction steps over the head width
  static constexpr int RK = 32 / Elem<T>::KS;            // ... over a block of 32 rows
  static constexpr int DB = DP / 32;
  static constexpr int PPR = DP / E;                     // pieces per row
  using Columns = uint4[KK];                             // a lane's share of its column vector, as B operands
};

// A operand: 32 consecutive tile rows x contraction step kk over the head width
template <typename T, int DP>
__device__ __forceinline__ uint4 frag_rows(const T *tile, int row0, int kk, int lane) {
  return *reinterpret_cast<const uint4 *>(tile + (row0 + (lane & 31)) * Tile<T, DP>::RS + kk * Elem<T>::KS +
                                          (lane >> 5) * (Elem<T>::KS / 2));
}

// A operand of the transposed tile: head elements 32 db .. + 31 x contraction step kk over rows row0 .. row0 + 31
template <typename T, int DP>
__device__ __forceinline__ uint4 frag_cols(const T *tile, int row0, int db, int kk, int lane) {
  constexpr int RS = Tile<T, DP>::RS;
  if constexpr (sizeof(T) == 4) {
    const float *p = reinterpret_cast<const float *>(tile) + (row0 + 8 * kk + 4 * (lane >> 5)) * RS + 32 * db + (lane & 31);
    return __builtin_bit_cast(uint4, f32x4v{p[0], p[RS], p[2 * RS], p[3 * RS]});
  } else {
    // 16 lanes hand in the addresses of a 4-row x 16-column patch in 8-byte pieces, lane i of them gets column i
    const T *p = tile + (row0 + 16 * kk + 4 * (lane >> 5) + ((lane & 15) >> 2)) * RS + 32 * db + 16 * ((lane >> 4) & 1) +
                 4 * (lane & 3);
    const auto lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr_h16x4 *)(p));
    const auto hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr_h16x4 *)(p + 8 * RS));
    const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
    return uint4{a.x, a.y, b.x, b.y};
  }
}

// streamed rows: registers <- global, LDS <- registers
template <typename T, int DP, int TR> struct Stage {
  static constexpr int N = (TR * Tile<T, DP>::PPR + 255) / 256;
  uint4 r[N];
  template <typename Row>
  __device__ __forceinline__ void fetch(Row row_of, int row0, int D, bool vec) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int id = (int)threadIdx.x + 256 * n;
      const int row = id / Tile<T, DP>::PPR, e0 = (id % Tile<T, DP>::PPR) * Tile<T, DP>::E;
      r[n] = uint4{0, 0, 0, 0};
      if (row < TR) {
        const T *p = row_of(row0 + row);
        if (p) r[n] = load_piece<T>(p, e0, D, vec);
      }
    }
  }
  __device__ __forceinline__ void store(T *tile) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int id = (int)threadIdx.x + 256 * n;
      const int row = id / Tile<T, DP>::PPR, e0 = (id % Tile<T, DP>::PPR) * Tile<T, DP>::E;
      if (row < TR) *reinterpret_cast<uint4 *>(tile + row * Tile<T, DP>::RS + e0) = r[n];
    }
  }
};

// column vectors of the lane, kept as B operands
template <typename T, int DP>
__device__ __forceinline__ void load_columns(typename Tile<T, DP>::Columns &x, const T *row, int D, bool vec, int lane) {
#pragma unroll
  for (int kk = 0; kk < Tile<T, DP>::KK; ++kk)
    x[kk] = row ? load_piece<T>(row, kk * Elem<T>::KS + (lane >> 5) * (Elem<T>::KS / 2), D, vec) : uint4{0, 0, 0, 0};
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

__device__ __forceinline__ void col_of(const AttnArgs &a, int c, int &i, int &hh) {
  if (a.HG == 1) { i = c; hh = 0; } else { i = (int)((unsigned)c / (unsigned)a.HG); hh = c - i * a.HG; }
}

// first and last + 1 visible key of [lo, hi) (workgroup-uniform); hi <= lo when there is none
__device__ inline void visible_range(const uint8_t *pad, int &lo, int &hi, int *red) {
  int first = hi, last = lo;
  for (int j = lo + (int)threadIdx.x; j < hi; j += 256)
    if (!pad[j]) { first = j < first ? j : first; last = j + 1; }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const int f = __shfl_xor(first, off), l = __shfl_xor(last, off);
    first = f < first ? f : first;
    last = l > last ? l : last;
  }
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = first; red[4 + (threadIdx.x >> 6)] = last; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    first = red[w] < first ? red[w] : first;
    last = red[4 + w] > last ? red[4 + w] : last;
  }
  __syncthreads();
  lo = first;
  hi = last;
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
  template <int NS>
  __device__ __forceinline__ void apply(float (&ds)[NS][16], f32x16 (&acc)[DB]) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
      float top = 0.0f;
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[n][r]));
      top = fmaxf(top, other_half(top));
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
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[n][r] *= f;
    }
  }
};

template <typename T> constexpr float prob_shift() {         // log2 of the factor the probabilities carry into float16
  return sizeof(T) == 2 && !__is_same(T, __bf16) ? 15.0f : 0.0f;
}

template <typename T, int DP, bool WK> struct Shape {
  static constexpr int TR = WK ? 128 : (sizeof(T) == 4 && DP == 128 ? 32 : 64);   // streamed rows per tile
  static constexpr int NS = WK ? TR / 128 : TR / 32;                               // 32-row blocks of a wave per tile
  static constexpr int COLS = WK ? 32 : 128;                                       // columns of a workgroup
  static constexpr int TILE = TR * Tile<T, DP>::RS * (int)sizeof(T);               // bytes of one staged tile
  static constexpr int NBUF = 4 * TILE <= 80 * 1024 ? 2 : 1;
  static constexpr int JOIN = WK ? 4 * 32 * (DP + 1) * 4 : 0;
  static constexpr int LDS = 2 * NBUF * TILE > JOIN ? 2 * NBUF * TILE : JOIN;
};

// the four waves' partial results of the same 32 columns: acc * f summed over the waves in wave order
// (the caller has synchronised: the tiles are no longer read)
template <int DP>
__device__ __forceinline__ void join_put(float *lds, const f32x16 (&acc)[DP / 32], float f, int w, int lane) {
  float *p = lds + (w * 32 + (lane & 31)) * (DP + 1) + 4 * (lane >> 5);
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) p[32 * db + 8 * (r >> 2) + (r & 3)] = acc[db][r] * f;
}
template <int DP> __device__ __forceinline__ float join_get(const float *lds, int col, int d) {
  const float *p = lds + col * (DP + 1) + d;
  return ((p[0] + p[32 * (DP + 1)]) + p[2 * 32 * (DP + 1)]) + p[3 * 32 * (DP + 1)];
}

// ---------------------------------------------------------------------------------------------------------------------
// forward.  WK = false: four waves, 128 columns, every wave walks all keys; WK = true: 32 columns, each wave takes a
// quarter of every tile's keys and the four results are joined (few columns)
template <typename T, int DP, bool WK> __global__ __launch_bounds__(256) void attn_fwd_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, WK>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ __attribute__((aligned(16))) int hid[Sh::NBUF][TR];
  __shared__ float stat[2][4][32];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int ncb = (a.C + Sh::COLS - 1) / Sh::COLS;
  unsigned id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = (int)(id % (unsigned)a.splits);
  id /= (unsigned)a.splits;
  int cb = (int)(id % (unsigned)ncb);
  const int bg = (int)(id / (unsigned)ncb), b = bg / a.G, gh = bg - b * a.G;
  if (a.causal) cb = ncb - 1 - cb;                                    // the longest first
  const int c0 = cb * Sh::COLS, c = c0 + (WK ? 0 : 32 * w) + (lane & 31);
  const bool mine = c < a.C;
  int i, hh;
  col_of(a, mine ? c : 0, i, hh);
  const T *kb = static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)gh * a.ks[2];
  const T *vb = static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)gh * a.vs[2];
  const uint8_t *pad = a.pad ? a.pad + (int64_t)b * a.pad_b : nullptr;
  uint4 q[Ti::KK];
  load_columns<T, DP>(q, mine ? static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] +
                                    (int64_t)(gh * a.HG + hh) * a.qs[2]
                              : nullptr, a.D, a.qvec, lane);
  // keys of this workgroup
  int lo = 0, hi = a.S, first_limit = a.S;
  if (a.splits > 1) {
    const int chunk = ((a.S + a.splits - 1) / a.splits + TR - 1) / TR * TR;
    lo = (int)min((int64_t)sp * chunk, (int64_t)a.S);
    hi = min(lo + chunk, a.S);
  }
  const int lim = a.causal ? i + a.S - a.L : a.S;                     // the last key that the column sees
  if (a.causal) {
    int il, ih;
    col_of(a, min(c0 + Sh::COLS, a.C) - 1, il, ih);
    hi = min(hi, il + a.S - a.L + 1);
    col_of(a, c0, il, ih);
    first_limit = il + a.S - a.L;
  }
  if (pad && lo < hi) visible_range(pad, lo, hi, reinterpret_cast<int *>(&stat[0][0][0]));

  f32x16 acc[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) acc[db] = f32x16{0.0f};
  float m = -__builtin_inff(), l = 0.0f;                              // maximum of the scores, this half's sum
  Stage<T, DP, TR> sk, sv;
  int hidden = 0;
  auto fetch = [&](int t0) {
    // (a row behind the last key is not read; a padded one is read and replaced by zeros, whatever it holds)
    sk.fetch([&](int j) -> const T * { return j < hi && !(pad && pad[j]) ? kb + (int64_t)j * a.ks[1] : nullptr; }, t0, a.D, a.kvec);
    sv.fetch([&](int j) -> const T * { return j < hi && !(pad && pad[j]) ? vb + (int64_t)j * a.vs[1] : nullptr; }, t0, a.D, a.vvec);
    if ((int)threadIdx.x < TR) hidden = t0 + (int)threadIdx.x >= hi || (pad && pad[t0 + (int)threadIdx.x]);
  };
  auto put = [&](int buf) {
    sk.store(reinterpret_cast<T *>(lds + (2 * buf) * Sh::TILE));
    sv.store(reinterpret_cast<T *>(lds + (2 * buf + 1) * Sh::TILE));
    if ((int)threadIdx.x < TR) hid[buf][threadIdx.x] = hidden;
  };
  auto compute = [&](int t0, int buf) {
    const T *tk = reinterpret_cast<const T *>(lds + (2 * buf) * Sh::TILE);
    const T *tv = reinterpret_cast<const T *>(lds + (2 * buf + 1) * Sh::TILE);
    const int r0 = WK ? 32 * NS * w : 0;
    float s[NS][16];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x16 x = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) mma(x, frag_rows<T, DP>(tk, r0 + 32 * n, kk, lane), q[kk], T());
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = x[r];
    }
    if (pad || t0 + TR > hi || t0 + TR - 1 > first_limit) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int row = r0 + 32 * n + 8 * r4 + 4 * h;
          const int4 hd = *reinterpret_cast<const int4 *>(&hid[buf][row]);
          const int hx[4] = {hd.x, hd.y, hd.z, hd.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hx[e] || t0 + row + e > lim) s[n][4 * r4 + e] = -__builtin_inff();
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
    top = fmaxf(top, other_half(top));
    const float mn = fmaxf(m, top);
    if (__any(mn > m)) {                                              // (rows whose maximum stays: factor 1)
      const float f = mn > m ? exp2f((m - mn) * a.c2) : 1.0f;
      l *= f;
#pragma unroll
      for (int db = 0; db < Ti::DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= f;
      m = mn;
    }
    const float base = m == -__builtin_inff() ? 0.0f : prob_shift<T>() - m * a.c2;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], a.c2, base));
        l += s[n][r];
      }
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 p = row_frag<T>(s[n], kk);
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) mma(acc[db], frag_cols<T, DP>(tv, r0 + 32 * n, db, kk, lane), p, T());
      }
  };

  if (lo < hi) {
    fetch(lo);
    if (Sh::NBUF == 2) put(0);
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += TR) {
      const bool more = t0 + TR < hi;
      if (Sh::NBUF == 2) {
        if (more) fetch(t0 + TR);
        __syncthreads();
        compute(t0, buf);
        if (more) put(buf ^ 1);
        buf ^= 1;
      } else {
        __syncthreads();
        put(0);
        __syncthreads();
        if (more) fetch(t0 + TR);
        compute(t0, 0);
      }
    }
  }
  l += other_half(l);
  const int64_t at = (int64_t)bg * a.C + c;
  const int64_t prow = (int64_t)sp * a.B * a.G * a.C + at;
  T *orow = static_cast<T *>(a.out) + (((int64_t)b * a.L + i) * a.H + gh * a.HG + hh) * a.D;
  float mt = m * a.c2 - prob_shift<T>();                              // log2 of the factor taken out of l and acc
  if (l == 0.0f) mt = -__builtin_inff();
  if constexpr (WK) {
    __syncthreads();
    if (h == 0) { stat[0][w][lane] = mt; stat[1][w][lane] = l; }
    __syncthreads();
    const int cl = lane & 31;
    float M = fmaxf(fmaxf(stat[0][0][cl], stat[0][1][cl]), fmaxf(stat[0][2][cl], stat[0][3][cl]));
    if (M == -__builtin_inff()) M = 0.0f;
    join_put<DP>(reinterpret_cast<float *>(lds), acc, exp2f(mt - M), w, lane);
    __syncthreads();
    for (int t = threadIdx.x; t < 32 * DP; t += 256) {
      const int col = t / DP, d = t % DP, cc = c0 + col;
      if (cc >= a.C) continue;
      float MM = fmaxf(fmaxf(stat[0][0][col], stat[0][1][col]), fmaxf(stat[0][2][col], stat[0][3][col]));
      const bool none = MM == -__builtin_inff();
      if (none) MM = 0.0f;
      float L = 0.0f;
#pragma unroll
      for (int x = 0; x < 4; ++x) L += stat[1][x][col] * exp2f(stat[0][x][col] - MM);
      const float o = join_get<DP>(reinterpret_cast<const float *>(lds), col, d);
      const int64_t ac = (int64_t)bg * a.C + cc, pc = (int64_t)sp * a.B * a.G * a.C + ac;
      if (a.splits > 1) {
        a.part[pc * DP + d] = o;
        if (d == 0) { a.ml[2 * pc] = none ? -__builtin_inff() : MM; a.ml[2 * pc + 1] = L; }
      } else {
        int ci, ch;
        col_of(a, cc, ci, ch);
        if (d < a.D)
          static_cast<T *>(a.out)[(((int64_t)b * a.L + ci) * a.H + gh * a.HG + ch) * a.D + d] = (T)(L == 0.0f ? 0.0f : o / L);
        if (d == 0 && a.lse) a.lse[ac] = L == 0.0f ? __builtin_inff() : MM + log2f(L);
      }
    }
  } else if (mine) {
    if (a.splits > 1) {
      store_column<float, Ti::DB>(a.part + prow * DP, acc, 1.0f, DP, lane);
      if (h == 0) { a.ml[2 * prow] = mt; a.ml[2 * prow + 1] = l; }
    } else {
      store_column<T, Ti::DB>(orow, acc, l == 0.0f ? 0.0f : 1.0f / l, a.D, lane);
      if (h == 0 && a.lse) a.lse[at] = l == 0.0f ? __builtin_inff() : mt + log2f(l);
    }
  }
}

// joins the splits of the forward kernel: one thread per column and head element, splits in order
template <typename T, int DP> __global__ __launch_bounds__(256) void attn_fwd_join_kernel(const AttnArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.B * a.G * a.C;
  const int64_t at = t / DP;
  const int d = (int)(t % DP);
  if (at >= n) return;
  float M = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, a.ml[2 * (s * n + at)]);
  if (M == -__builtin_inff()) M = 0.0f;
  float L = 0.0f, o = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2f(a.ml[2 * (s * n + at)] - M);
    L = fmaf(a.ml[2 * (s * n + at) + 1], f, L);
    o = fmaf(a.part[(s * n + at) * DP + d], f, o);
  }
  const int bg = (int)(at / a.C), c = (int)(at % a.C), b = bg / a.G, gh = bg % a.G;
  int i, hh;
  col_of(a, c, i, hh);
  if (d < a.D) static_cast<T *>(a.out)[(((int64_t)b * a.L + i) * a.H + gh * a.HG + hh) * a.D + d] = (T)(L == 0.0f ? 0.0f : o / L);
  if (d == 0 && a.lse) a.lse[at] = L == 0.0f ? __builtin_inff() : M + log2f(L);
}

// ---------------------------------------------------------------------------------------------------------------------
// dq (and delta): columns = queries, keys and values stream
template <typename T, int DP, bool WK> __global__ __launch_bounds__(256) void attn_dq_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, WK>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ __attribute__((aligned(16))) int hid[Sh::NBUF][TR];
  __shared__ int red[8];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int ncb = (a.C + Sh::COLS - 1) / Sh::COLS;
  unsigned id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = (int)(id % (unsigned)a.splits);
  id /= (unsigned)a.splits;
  int cb = (int)(id % (unsigned)ncb);
  const int bg = (int)(id / (unsigned)ncb), b = bg / a.G, gh = bg - b * a.G;
  if (a.causal) cb = ncb - 1 - cb;
  const int c0 = cb * Sh::COLS, c = c0 + (WK ? 0 : 32 * w) + (lane & 31);
  const bool mine = c < a.C;
  int i, hh;
  col_of(a, mine ? c : 0, i, hh);
  const int head = gh * a.HG + hh;
  const T *kb = static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)gh * a.ks[2];
  const T *vb = static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)gh * a.vs[2];
  const uint8_t *pad = a.pad ? a.pad + (int64_t)b * a.pad_b : nullptr;
  uint4 q[Ti::KK], g[Ti::KK];
  load_columns<T, DP>(q, mine ? static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)head * a.qs[2]
                              : nullptr, a.D, a.qvec, lane);
  load_columns<T, DP>(g, mine ? static_cast<const T *>(a.g) + (int64_t)b * a.gs[0] + (int64_t)i * a.gs[1] + (int64_t)head * a.gs[2]
                              : nullptr, a.D, a.gvec, lane);
  const int64_t at = (int64_t)bg * a.C + c;
  const int64_t row_at = (((int64_t)b * a.L + i) * a.H + head) * a.D;
  float delta = 0.0f;
  if (mine) {
    const T *orow = static_cast<const T *>(a.o) + row_at;
#pragma unroll
    for (int kk = 0; kk < Ti::KK; ++kk)
      delta += dot_piece<T>(g[kk], load_piece<T>(orow, kk * Elem<T>::KS + h * (Elem<T>::KS / 2), a.D, a.ovec));
  }
  delta += other_half(delta);
  if (mine && h == 0 && sp == 0 && (!WK || w == 0)) a.delta[at] = delta;
  const float lse = mine ? a.lse[at] : __builtin_inff();

  int lo = 0, hi = a.S, first_limit = a.S;
  if (a.splits > 1) {
    const int chunk = ((a.S + a.splits - 1) / a.splits + TR - 1) / TR * TR;
    lo = (int)min((int64_t)sp * chunk, (int64_t)a.S);
    hi = min(lo + chunk, a.S);
  }
  const int lim = a.causal ? i + a.S - a.L : a.S;
  if (a.causal) {
    int il, ih;
    col_of(a, min(c0 + Sh::COLS, a.C) - 1, il, ih);
    hi = min(hi, il + a.S - a.L + 1);
    col_of(a, c0, il, ih);
    first_limit = il + a.S - a.L;
  }
  if (pad && lo < hi) visible_range(pad, lo, hi, red);

  f32x16 acc[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) acc[db] = f32x16{0.0f};
  ColumnScale<T, Ti::DB> cs;
  cs.start();
  Stage<T, DP, TR> sk, sv;
  int hidden = 0;
  auto fetch = [&](int t0) {
    sk.fetch([&](int j) -> const T * { return j < hi && !(pad && pad[j]) ? kb + (int64_t)j * a.ks[1] : nullptr; }, t0, a.D, a.kvec);
    sv.fetch([&](int j) -> const T * { return j < hi && !(pad && pad[j]) ? vb + (int64_t)j * a.vs[1] : nullptr; }, t0, a.D, a.vvec);
    if ((int)threadIdx.x < TR) hidden = t0 + (int)threadIdx.x >= hi || (pad && pad[t0 + (int)threadIdx.x]);
  };
  auto put = [&](int buf) {
    sk.store(reinterpret_cast<T *>(lds + (2 * buf) * Sh::TILE));
    sv.store(reinterpret_cast<T *>(lds + (2 * buf + 1) * Sh::TILE));
    if ((int)threadIdx.x < TR) hid[buf][threadIdx.x] = hidden;
  };
  auto compute = [&](int t0, int buf) {
    const T *tk = reinterpret_cast<const T *>(lds + (2 * buf) * Sh::TILE);
    const T *tv = reinterpret_cast<const T *>(lds + (2 * buf + 1) * Sh::TILE);
    const int r0 = WK ? 32 * NS * w : 0;
    const bool some_hidden = pad || t0 + TR > hi || t0 + TR - 1 > first_limit;
    float ds[NS][16];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x16 x = f32x16{0.0f}, y = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) {
        mma(x, frag_rows<T, DP>(tk, r0 + 32 * n, kk, lane), q[kk], T());
        mma(y, frag_rows<T, DP>(tv, r0 + 32 * n, kk, lane), g[kk], T());
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[n][r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c2, -lse)) * (y[r] - delta);
      if (some_hidden) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int row = r0 + 32 * n + 8 * r4 + 4 * h;
          const int4 hd = *reinterpret_cast<const int4 *>(&hid[buf][row]);
          const int hx[4] = {hd.x, hd.y, hd.z, hd.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hx[e] || t0 + row + e > lim) ds[n][4 * r4 + e] = 0.0f;
        }
      }
    }
    cs.apply(ds, acc);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 p = row_frag<T>(ds[n], kk);
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) mma(acc[db], frag_cols<T, DP>(tk, r0 + 32 * n, db, kk, lane), p, T());
      }
  };
  if (lo < hi) {
    fetch(lo);
    if (Sh::NBUF == 2) put(0);
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += TR) {
      const bool more = t0 + TR < hi;
      if (Sh::NBUF == 2) {
        if (more) fetch(t0 + TR);
        __syncthreads();
        compute(t0, buf);
        if (more) put(buf ^ 1);
        buf ^= 1;
      } else {
        __syncthreads();
        put(0);
        __syncthreads();
        if (more) fetch(t0 + TR);
        compute(t0, 0);
      }
    }
  }
  const float f = a.scale / cs.f;
  if constexpr (WK) {
    __syncthreads();
    join_put<DP>(reinterpret_cast<float *>(lds), acc, f, w, lane);
    __syncthreads();
    for (int t = threadIdx.x; t < 32 * DP; t += 256) {
      const int col = t / DP, d = t % DP, cc = c0 + col;
      if (cc >= a.C || d >= a.D) continue;
      const float o = join_get<DP>(reinterpret_cast<const float *>(lds), col, d);
      int ci, ch;
      col_of(a, cc, ci, ch);
      if (a.splits > 1)
        a.part[((int64_t)sp * a.B * a.G * a.C + (int64_t)bg * a.C + cc) * DP + d] = o;
      else
        static_cast<T *>(a.out)[(((int64_t)b * a.L + ci) * a.H + gh * a.HG + ch) * a.D + d] = (T)o;
    }
  } else if (mine) {
    if (a.splits > 1)
      store_column<float, Ti::DB>(a.part + ((int64_t)sp * a.B * a.G * a.C + at) * DP, acc, f, DP, lane);
    else
      store_column<T, Ti::DB>(static_cast<T *>(a.out) + row_at, acc, f, a.D, lane);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// dk and dv: columns = keys, the queries that use this key head and their output gradients stream; the heads of a
// group are rows of the same stream, so shared heads are summed here, in a fixed order and without atomics
template <typename T, int DP, bool WK> __global__ __launch_bounds__(256) void attn_dkv_kernel(const AttnArgs a) {
  using Sh = Shape<T, DP, WK>;
  using Ti = Tile<T, DP>;
  constexpr int TR = Sh::TR, NS = Sh::NS;
  __shared__ __attribute__((aligned(16))) unsigned char lds[Sh::LDS];
  __shared__ __attribute__((aligned(16))) float slse[Sh::NBUF][TR], sdel[Sh::NBUF][TR];
  __shared__ __attribute__((aligned(16))) int slim[Sh::NBUF][TR];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int nkb = (a.S + Sh::COLS - 1) / Sh::COLS;
  unsigned id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = (int)(id % (unsigned)a.splits);
  id /= (unsigned)a.splits;
  const int kblk = (int)(id % (unsigned)nkb), bg = (int)(id / (unsigned)nkb), b = bg / a.G, gh = bg - b * a.G;
  const int j0 = kblk * Sh::COLS, j = j0 + (WK ? 0 : 32 * w) + (lane & 31);
  const bool mine = j < a.S, seen = mine && !(a.pad && a.pad[(int64_t)b * a.pad_b + j]);
  const T *qb = static_cast<const T *>(a.q) + (int64_t)b * a.qs[0] + (int64_t)gh * a.HG * a.qs[2];
  const T *gb = static_cast<const T *>(a.g) + (int64_t)b * a.gs[0] + (int64_t)gh * a.HG * a.gs[2];
  const float *lb = a.lse + (int64_t)bg * a.C, *db_ = a.delta + (int64_t)bg * a.C;
  uint4 k[Ti::KK], v[Ti::KK];
  load_columns<T, DP>(k, seen ? static_cast<const T *>(a.k) + (int64_t)b * a.ks[0] + (int64_t)j * a.ks[1] + (int64_t)gh * a.ks[2]
                              : nullptr, a.D, a.kvec, lane);
  load_columns<T, DP>(v, seen ? static_cast<const T *>(a.v) + (int64_t)b * a.vs[0] + (int64_t)j * a.vs[1] + (int64_t)gh * a.vs[2]
                              : nullptr, a.D, a.vvec, lane);
  // columns (queries) of this workgroup; a workgroup whose keys are all padding has none
  int lo = 0, hi = a.C;
  if (a.splits > 1) {
    const int chunk = ((a.C + a.splits - 1) / a.splits + TR - 1) / TR * TR;
    lo = (int)min((int64_t)sp * chunk, (int64_t)a.C);
    hi = min(lo + chunk, a.C);
  }
  if (a.causal) {                                                     // the first query that sees key j0
    const int64_t i0 = (int64_t)j0 - (a.S - a.L);
    if (i0 > 0) lo = (int)max((int64_t)lo, min(i0 * a.HG, (int64_t)a.C) / TR * TR);
  }
  if (!__syncthreads_or(seen)) hi = lo;

  f32x16 ak[Ti::DB], av[Ti::DB];
#pragma unroll
  for (int db = 0; db < Ti::DB; ++db) { ak[db] = f32x16{0.0f}; av[db] = f32x16{0.0f}; }
  ColumnScale<T, Ti::DB> cs;
  cs.start();
  Stage<T, DP, TR> sq, sg;
  float rl = 0.0f, rd = 0.0f;
  int rlim = 0;
  auto fetch = [&](int t0) {
    sq.fetch([&](int c) -> const T * {
      if (c >= hi) return nullptr;
      int i, hh;
      col_of(a, c, i, hh);
      return qb + (int64_t)i * a.qs[1] + (int64_t)hh * a.qs[2];
    }, t0, a.D, a.qvec);
    sg.fetch([&](int c) -> const T * {
      if (c >= hi) return nullptr;
      int i, hh;
      col_of(a, c, i, hh);
      return gb + (int64_t)i * a.gs[1] + (int64_t)hh * a.gs[2];
    }, t0, a.D, a.gvec);
    if ((int)threadIdx.x < TR) {
      const int c = t0 + (int)threadIdx.x;
      rl = c < hi ? lb[c] : __builtin_inff();
      rd = c < hi ? db_[c] : 0.0f;
      int i, hh;
      col_of(a, c, i, hh);
      rlim = a.causal ? i + a.S - a.L : a.S;
    }
  };
  auto put = [&](int buf) {
    sq.store(reinterpret_cast<T *>(lds + (2 * buf) * Sh::TILE));
    sg.store(reinterpret_cast<T *>(lds + (2 * buf + 1) * Sh::TILE));
    if ((int)threadIdx.x < TR) { slse[buf][threadIdx.x] = rl; sdel[buf][threadIdx.x] = rd; slim[buf][threadIdx.x] = rlim; }
  };
  auto compute = [&](int t0, int buf) {
    const T *tq = reinterpret_cast<const T *>(lds + (2 * buf) * Sh::TILE);
    const T *tg = reinterpret_cast<const T *>(lds + (2 * buf + 1) * Sh::TILE);
    const int r0 = WK ? 32 * NS * w : 0;
    int il = 0, ih;
    if (a.causal) col_of(a, t0, il, ih);
    const bool some_hidden = a.causal && j0 + Sh::COLS - 1 > il + a.S - a.L;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      f32x16 x = f32x16{0.0f}, y = f32x16{0.0f};
#pragma unroll
      for (int kk = 0; kk < Ti::KK; ++kk) {
        mma(x, frag_rows<T, DP>(tq, r0 + 32 * n, kk, lane), k[kk], T());
        mma(y, frag_rows<T, DP>(tg, r0 + 32 * n, kk, lane), v[kk], T());
      }
      float p[16], ds[1][16];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int row = r0 + 32 * n + 8 * r4 + 4 * h;
        const float4 ls = *reinterpret_cast<const float4 *>(&slse[buf][row]);
        const float4 de = *reinterpret_cast<const float4 *>(&sdel[buf][row]);
        const float lx[4] = {ls.x, ls.y, ls.z, ls.w}, dx[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * r4 + e;
          p[r] = __builtin_amdgcn_exp2f(fmaf(x[r], a.c2, -lx[e]));
          ds[0][r] = y[r] - dx[e];
        }
        if (some_hidden) {
          const int4 lm = *reinterpret_cast<const int4 *>(&slim[buf][row]);
          const int mx[4] = {lm.x, lm.y, lm.z, lm.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j > mx[e]) { p[4 * r4 + e] = 0.0f; ds[0][4 * r4 + e] = 0.0f; }
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[0][r] *= p[r];
      if constexpr (prob_shift<T>() != 0.0f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= 32768.0f;
      }
      cs.apply(ds, ak);
#pragma unroll
      for (int kk = 0; kk < Ti::RK; ++kk) {
        const uint4 pf = row_frag<T>(p, kk), df = row_frag<T>(ds[0], kk);
#pragma unroll
        for (int db = 0; db < Ti::DB; ++db) {
          mma(av[db], frag_cols<T, DP>(tg, r0 + 32 * n, db, kk, lane), pf, T());
          mma(ak[db], frag_cols<T, DP>(tq, r0 + 32 * n, db, kk, lane), df, T());
        }
      }
    }
  };
  if (lo < hi) {
    fetch(lo);
    if (Sh::NBUF == 2) put(0);
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += TR) {
      const bool more = t0 + TR < hi;
      if (Sh::NBUF == 2) {
        if (more) fetch(t0 + TR);
        __syncthreads();
        compute(t0, buf);
        if (more) put(buf ^ 1);
        buf ^= 1;
      } else {
        __syncthreads();
        put(0);
        __syncthreads();
        if (more) fetch(t0 + TR);
        compute(t0, 0);
      }
    }
  }
  // (a padded key's lane has computed with zeros for its key and value: its sums are dropped)
  const float fk = seen ? a.scale / cs.f : 0.0f, fv = seen ? exp2f(-prob_shift<T>()) : 0.0f;
  if (!seen) {
#pragma unroll
    for (int db = 0; db < Ti::DB; ++db) { ak[db] = f32x16{0.0f}; av[db] = f32x16{0.0f}; }
  }
  if constexpr (WK) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      join_put<DP>(reinterpret_cast<float *>(lds), which ? av : ak, which ? fv : fk, w, lane);
      __syncthreads();
      for (int t = threadIdx.x; t < 32 * DP; t += 256) {
        const int col = t / DP, d = t % DP, jj = j0 + col;
        if (jj >= a.S || d >= a.D) continue;
        const float o = join_get<DP>(reinterpret_cast<const float *>(lds), col, d);
        if (a.splits > 1)
          (which ? a.part2 : a.part)[(((int64_t)sp * a.B * a.G + bg) * a.S + jj) * DP + d] = o;
        else
          static_cast<T *>(which ? a.out2 : a.out)[(((int64_t)b * a.S + jj) * a.G + gh) * a.D + d] = (T)o;
      }
    }
  } else if (mine) {
    if (a.splits > 1) {
      const int64_t row = (((int64_t)sp * a.B * a.G + bg) * a.S + j) * DP;
      store_column<float, Ti::DB>(a.part + row, ak, fk, DP, lane);
      store_column<float, Ti::DB>(a.part2 + row, av, fv, DP, lane);
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
  const int64_t at = t / DP;
  const int d = (int)(t % DP);
  if (at >= rows || d >= D) return;
  float s = 0.0f;
  for (int x = 0; x < splits; ++x) s += part[(x * rows + at) * DP + d];
  const int bg = (int)(at / n), c = (int)(at % n), b = bg / G, gh = bg % G;
  out[((((int64_t)b * (n / per) + c / per) * G + gh) * per + c % per) * D + d] = (T)s;
}

// ---- launches ---------------------------------------------------------------------------------------------------------
enum AttnPass { kAttnFwd, kAttnDq, kAttnDkv };

template <typename T, int DP, bool WK> void attn_launch(AttnPass pass, const AttnArgs &a, hipStream_t s) {
  const int cols = pass == kAttnDkv ? a.S : a.C, per = Shape<T, DP, WK>::COLS;
  const unsigned grid = (unsigned)((int64_t)a.B * a.G * ((cols + per - 1) / per) * a.splits);
  if (pass == kAttnFwd)
    hipLaunchKernelGGL((attn_fwd_kernel<T, DP, WK>), dim3(grid), dim3(256), 0, s, a);
  else if (pass == kAttnDq)
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, WK>), dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP, WK>), dim3(grid), dim3(256), 0, s, a);
}

template <typename T, int DP> int attn_run(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) {
  if (wk) attn_launch<T, DP, true>(pass, a, s);
  else attn_launch<T, DP, false>(pass, a, s);
  HSGK_LAUNCH_CHECK();
  if (a.splits > 1) {
    const int n = pass == kAttnDkv ? a.S : a.C;
    const unsigned grid = (unsigned)(((int64_t)a.B * a.G * n * DP + 255) / 256);
    if (pass == kAttnFwd) {
      hipLaunchKernelGGL((attn_fwd_join_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a);
    } else {
      const int per = pass == kAttnDkv ? 1 : a.HG;
      hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a.part, a.splits, a.B, a.G, n, per, a.D,
                         static_cast<T *>(a.out));
      if (pass == kAttnDkv)
        hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3(grid), dim3(256), 0, s, a.part2, a.splits, a.B, a.G, n, per, a.D,
                           static_cast<T *>(a.out2));
    }
    HSGK_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T> int attn_type(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) {
  if (a.D <= 32) return attn_run<T, 32>(pass, a, wk, s);
  if (a.D <= 64) return attn_run<T, 64>(pass, a, wk, s);
  return attn_run<T, 128>(pass, a, wk, s);
}

int attn_f32(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s);
int attn_bf16(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s);
int attn_f16(AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s);

}  // namespace hsgk
