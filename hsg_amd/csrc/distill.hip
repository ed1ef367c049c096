// distill.hip -- distillation of a softmax over V classes (prototypes) from a teacher's k best of them.
//
// Per row: p = softmax over the k entries of t / T (an entry outside [0, V) or with t = -inf does not count),
//   q = softmax over all V of z / T,   loss = T^2 sum_j p_j (log p_j - log q_{idx_j})   (no entry: 0)
//   dz_v = g T (q_v - sum_{j: idx_j = v} p_j)                                            (no entry: 0)
// Both passes are bound by memory: the forward reads the row once and leaves (maximum, sum) for the backward, which reads
// the row and writes the gradient once.  Rows that fit go through LDS (a wave each), longer ones through registers with a
// running maximum and sum (a workgroup each).  TB/s of what has to move, where a 1 GiB copy reaches 5.2 (forward, backward):
// 50176 x 4096 bfloat16, k = 32: 4.4, 5.4; 4099 (rows start anywhere): 3.9, 4.9; 37632 x 2048 float32, k = 20: 4.6, 5.7;
// 12544 x 16384 bfloat16: 5.2, 5.7; 1031 x 100003 float16, k = 64: 3.4 (four workgroups a CU), 5.2.
#include <math.h>

#include "common.h"

namespace hsgk {

constexpr int kDistillMax = HSGK_DISTILL_MAX_K;

struct DistillArgs {
  const void *z;
  int64_t n, V, stride;
  const float *t;
  const int64_t *idx;
  int k;
  float T, c2;               // c2 = log2(e) / T
  float *loss, *stats;       // stats [n][2]
  const float *g;
  void *dz;
};

// threads of one row: a wave (four rows a workgroup) or the whole workgroup
template <int P> __device__ __forceinline__ void row_sync() {
  if constexpr (P == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

template <int P> __device__ __forceinline__ float row_max(float x, float *red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
  if constexpr (P > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < P / 64; ++w) x = fmaxf(x, red[w]);
    __syncthreads();
  }
  return x;
}
template <int P> __device__ __forceinline__ float row_sum(float x, float *red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
  if constexpr (P > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < P / 64; ++w) x += red[w];
    __syncthreads();
  }
  return x;
}

template <typename T> struct Piece {
  static constexpr int E = 16 / (int)sizeof(T);
};

// a row cut into 16-byte pieces at aligned addresses: `head` elements before the first, `full` pieces, the rest from
// element `rest` on.  Piece 0 lies `skip` pieces behind a 128-byte line's start; the threads are counted from there, so that
// what a wave moves at once begins and ends with a line.
template <typename T> struct Cut {
  int head, full, rest, skip;
  __device__ __forceinline__ Cut(const T *row, int V) {
    constexpr int E = Piece<T>::E;
    head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    if (head > V) head = V;
    full = (V - head) / E;
    rest = head + full * E;
    skip = (int)(reinterpret_cast<uintptr_t>(row + head) >> 4) & 7;
  }
};

typedef unsigned u32x4nt __attribute__((ext_vector_type(4)));

// Whether a row is read past the caches: forward and backward both read the logits, so the forward leaves them in the
// 256 MB cache where they fit; larger ones would only push each other out.  (forward + backward, us: 308 MB past 45 + 106,
// through 68 + 116; 206 MB past 43 + 100, through 43 + 73.)
template <bool NT> __device__ __forceinline__ uint4 load16(const uint4 *p) {
  return NT ? __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4nt *>(p))) : *p;
}

// exp2 of (x - base) / T.  The difference comes first: it is exact for 16-bit logits and small where it matters, while
// x c2 - base c2 would carry the rounding of base c2, which what all logits of a row have in common makes large (float16, an
// offset of 1000, T = 0.5: log L off by up to 8e-5) and which the lowest value of bfloat16 takes past float32's range.
__device__ __forceinline__ float power(float x, float base, float c2) { return __builtin_amdgcn_exp2f((x - base) * c2); }

template <typename T> __device__ __forceinline__ void widen(const uint4 &u, float (&x)[Piece<T>::E]) {
  T y[Piece<T>::E];
  __builtin_memcpy(y, &u, 16);
#pragma unroll
  for (int i = 0; i < Piece<T>::E; ++i) x[i] = (float)y[i];
}

// the teacher's entries of a row, P apart in the threads of the row: value, index (-1: does not count), the student's
// logit there.  load() only sends for them; the row itself is on its way before gather() looks at an index.
template <int P> struct Teacher {
  static constexpr int N = kDistillMax / P;
  float t[N], z[N];
  int64_t at[N];
  int v[N];
  float top, mass;
  __device__ __forceinline__ void load(const DistillArgs &a, int64_t row, int th) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int j = th + n * P;
      at[n] = -1;
      t[n] = -__builtin_inff();
      if (j < a.k) {
        at[n] = a.idx[row * a.k + j];
        t[n] = a.t[row * a.k + j];
      }
    }
  }
  template <typename T> __device__ __forceinline__ void gather(const DistillArgs &a, const T *zrow) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = at[n] >= 0 && at[n] < a.V && !(t[n] == -__builtin_inff()) ? (int)at[n] : -1;
      z[n] = v[n] >= 0 ? (float)zrow[v[n]] : 0.0f;
    }
  }
  // maximum and mass; whether any entry counts.  A NaN among them reaches the mass.
  __device__ __forceinline__ bool sum(const DistillArgs &a, float *red) {
    float m = -__builtin_inff(), s = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (v[n] >= 0) m = fmaxf(m, t[n] != t[n] ? __builtin_inff() : t[n]);
    top = row_max<P>(m, red);
#pragma unroll
    for (int n = 0; n < N; ++n) s += weight(a, n);
    mass = row_sum<P>(s, red);
    return top > -__builtin_inff();
  }
  __device__ __forceinline__ float weight(const DistillArgs &a, int n) const {
    return v[n] >= 0 ? __builtin_amdgcn_exp2f((t[n] - top) * a.c2) : 0.0f;
  }
  // this thread's share of sum_j p_j (log p_j - log q_j)
  __device__ __forceinline__ float loss(const DistillArgs &a, float base, float L) const {
    const float lm = logf(mass), lL = logf(L);
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (v[n] < 0) continue;
      const float p = weight(a, n) / mass;
      if (p != 0.0f) s += p * (((t[n] - top) / a.T - lm) - ((z[n] - base) / a.T - lL));
    }
    return s;
  }
};

template <typename T> __device__ __forceinline__ void put_piece(T *o, const T (&y)[Piece<T>::E], bool vec) {
  if (vec) {
    uint4 q;
    __builtin_memcpy(&q, y, 16);
    // (past the caches: the gradient is as large as the logits, which the next pass wants there; 16 - 27 % of the
    //  next forward's time at 206 and 308 MB)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4nt, q), reinterpret_cast<u32x4nt *>(o));
  } else {
#pragma unroll
    for (int e = 0; e < Piece<T>::E; ++e) o[e] = y[e];
  }
}

// the row is written: its k places are written again, each different one by the first entry that names it
template <typename T, int P, typename Grad>
__device__ __forceinline__ void put_entries(const DistillArgs &a, const Teacher<P> &te, int t, float *ws, int *vs, float w, T *dz,
                                            Grad grad) {
#pragma unroll
  for (int n = 0; n < Teacher<P>::N; ++n) {
    const int j = t + n * P;
    if (j < a.k) { ws[j] = te.weight(a, n); vs[j] = te.v[n]; }
  }
  row_sync<P>();
#pragma unroll
  for (int n = 0; n < Teacher<P>::N; ++n) {
    const int j = t + n * P, v = te.v[n];
    if (v < 0) continue;
    float p = 0.0f;
    bool first = true;
    for (int x = 0; x < a.k; ++x)
      if (vs[x] == v) {
        first &= x >= j;
        p += ws[x];
      }
    if (first) dz[v] = (T)(grad(te.z[n]) - w * (p / te.mass));
  }
}

// Longer rows: a workgroup each, U pieces a thread at a time; a piece past the end is loaded again from the last place and does not count
template <typename T, bool NT> __global__ __launch_bounds__(256) void distill_fwd_kernel(const DistillArgs a) {
  constexpr int P = 256, E = Piece<T>::E, U = 4;
  __shared__ float red[4];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  const Cut<T> cut(z, (int)a.V);
  Teacher<P> te;
  te.load(a, row, t);
  float m = -__builtin_inff(), l = 0.0f;
  auto take = [&](const float *x, int n) {
    float top = m;
    for (int e = 0; e < n; ++e) top = fmaxf(top, x[e]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    l *= __builtin_amdgcn_exp2f((m - base) * a.c2);
    for (int e = 0; e < n; ++e) l += power(x[e], base, a.c2);
    m = top;
  };
  const uint4 *pieces = reinterpret_cast<const uint4 *>(z + cut.head);
  uint4 u[U];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int n = 0; n < U; ++n) u[n] = load16<NT>(pieces + min(max(i0 + n * P, 0), cut.full - 1));
  };
  if (cut.full > 0) fetch(t - cut.skip);
  te.gather(a, z);                                         // (behind the row's first pieces, before its lines are gone)
  for (int i0 = t - cut.skip; i0 < cut.full; i0 += P * U) {
    if (i0 != t - cut.skip) fetch(i0);
    float x[U * E];
#pragma unroll
    for (int n = 0; n < U; ++n) {
      float y[E];
      widen<T>(u[n], y);
      const bool in = i0 + n * P >= 0 && i0 + n * P < cut.full;
#pragma unroll
      for (int e = 0; e < E; ++e) x[n * E + e] = in ? y[e] : -__builtin_inff();
    }
    float top = m;
#pragma unroll
    for (int e = 0; e < U * E; ++e) top = fmaxf(top, x[e]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    l *= __builtin_amdgcn_exp2f((m - base) * a.c2);
#pragma unroll
    for (int e = 0; e < U * E; ++e) l += power(x[e], base, a.c2);
    m = top;
  }
  {                                                        // the ends of the row: fewer than E elements each
    const int e = t < cut.head ? t : t - cut.head + cut.rest;
    if (t < cut.head + (int)a.V - cut.rest) {
      const float x = (float)z[e];
      take(&x, 1);
    }
  }
  const float M = row_max<P>(m, red), base = M == -__builtin_inff() ? 0.0f : M;
  const float L = row_sum<P>(l * __builtin_amdgcn_exp2f((m - base) * a.c2), red);
  const bool some = te.sum(a, red);
  const float s = row_sum<P>(some ? te.loss(a, base, L) : 0.0f, red);
  if (t == 0) {
    a.loss[row] = some ? a.T * a.T * s : 0.0f;
    if (a.stats) { a.stats[2 * row] = base; a.stats[2 * row + 1] = L; }
  }
}

template <typename T, bool NT> __global__ __launch_bounds__(256) void distill_bwd_kernel(const DistillArgs a) {
  constexpr int P = 256, E = Piece<T>::E, U = 4;
  __shared__ float ws[kDistillMax], red[4];
  __shared__ int vs[kDistillMax];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  T *dz = static_cast<T *>(a.dz) + row * a.V;
  const Cut<T> cut(z, (int)a.V);
  const bool vec = (reinterpret_cast<uintptr_t>(dz + cut.head) & 15) == 0;
  Teacher<P> te;
  te.load(a, row, t);
  const float w = a.g[row] * a.T, base = a.stats[2 * row], L = a.stats[2 * row + 1];
  const float f = w / L;
  const uint4 *pieces = reinterpret_cast<const uint4 *>(z + cut.head);
  uint4 u[U];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int n = 0; n < U; ++n) u[n] = load16<NT>(pieces + min(max(i0 + n * P, 0), cut.full - 1));
  };
  if (cut.full > 0) fetch(t - cut.skip);
  te.gather(a, z);
  const bool some = te.sum(a, red);
  auto grad = [&](float x) { return some ? f * power(x, base, a.c2) : 0.0f; };
  for (int i0 = t - cut.skip; i0 < cut.full; i0 += P * U) {
    if (i0 != t - cut.skip) fetch(i0);
#pragma unroll
    for (int n = 0; n < U; ++n) {
      if (i0 + n * P < 0 || i0 + n * P >= cut.full) continue;
      float x[E];
      widen<T>(u[n], x);
      T y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = (T)grad(x[e]);
      T *o = dz + cut.head + (int64_t)(i0 + n * P) * E;
      put_piece<T>(o, y, vec);
    }
  }
  if (t < cut.head + (int)a.V - cut.rest) {
    const int e = t < cut.head ? t : t - cut.head + cut.rest;
    dz[e] = (T)grad((float)z[e]);
  }
  if (some) put_entries<T, P>(a, te, t, ws, vs, w, dz, grad);        // (the same for all threads of the row)
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows that fit LDS: a wave each, R of them a workgroup.  The row comes straight into LDS, whole, past the registers, so its
// length and not U bounds what is under way, and the teacher's k places are read there: in memory those reads touched
// nearly half of a row's lines a second time.
template <bool NT> __device__ __forceinline__ void row_to_lds(const void *from, uint32_t lds_byte) {
  uint32_t m0;                                             // (the compiler's: put back)
  if (NT)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(lds_byte), "v"(from) : "memory");
  else
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"(lds_byte), "v"(from) : "memory");
}

// bytes of LDS of a row: 128 in front (the head and the line's start), whole pieces, the rest
template <typename T> constexpr int lds_row_bytes(int64_t V) { return 128 + (int)((V * (int64_t)sizeof(T) + 15) / 16 + 1) * 16; }

// sends for the row; element e will lie at x[e] of the returned pointer
template <typename T, bool NT>
__device__ __forceinline__ T *fetch_row(const T *z, const Cut<T> &cut, int V, unsigned char *lds, int lane) {
  constexpr int E = Piece<T>::E;
  const uint32_t base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)(lds)) + 128;
  T *x = reinterpret_cast<T *>(lds + 128) - cut.head;
  for (int i0 = -cut.skip; i0 < cut.full; i0 += 64) {
    const int i = i0 + lane;
    if (i >= 0 && i < cut.full) row_to_lds<NT>(z + cut.head + (int64_t)i * E, __builtin_amdgcn_readfirstlane(base + (uint32_t)(i0 * 16)));
  }
  if (lane < cut.head + V - cut.rest) {
    const int e = lane < cut.head ? lane : lane - cut.head + cut.rest;
    x[e] = z[e];
  }
  return x;
}
__device__ __forceinline__ void row_has_come() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                      // vmcnt(0) lgkmcnt(0): the row and its ends
  asm volatile("" ::: "memory");
}

template <typename T, bool NT> __global__ __launch_bounds__(256) void distill_fwd_row_kernel(const DistillArgs a) {
  constexpr int E = Piece<T>::E;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_rows[];
  const int t = threadIdx.x & 63, rw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + rw;
  if (row >= a.n) return;                                  // (no barrier of the workgroup follows)
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  const int V = (int)a.V;
  const Cut<T> cut(z, V);
  Teacher<64> te;
  te.load(a, row, t);
  const T *x = fetch_row<T, NT>(z, cut, V, lds_rows + rw * lds_row_bytes<T>(V), t);
  row_has_come();
  te.gather(a, x);
  const bool end = t < cut.head + V - cut.rest;
  const float xe = end ? (float)x[t < cut.head ? t : t - cut.head + cut.rest] : -__builtin_inff();
  const uint4 *pieces = reinterpret_cast<const uint4 *>(x + cut.head);
  float top = xe;
  for (int i = t; i < cut.full; i += 64) {
    float y[E];
    widen<T>(pieces[i], y);
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, y[e]);
  }
  top = row_max<64>(top, nullptr);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float l = end ? power(xe, base, a.c2) : 0.0f;
  for (int i = t; i < cut.full; i += 64) {
    float y[E];
    widen<T>(pieces[i], y);
#pragma unroll
    for (int e = 0; e < E; ++e) l += power(y[e], base, a.c2);
  }
  const float L = row_sum<64>(l, nullptr);
  const bool some = te.sum(a, nullptr);
  const float s = row_sum<64>(some ? te.loss(a, base, L) : 0.0f, nullptr);
  if (t == 0) {
    a.loss[row] = some ? a.T * a.T * s : 0.0f;
    if (a.stats) { a.stats[2 * row] = base; a.stats[2 * row + 1] = L; }
  }
}

template <typename T, bool NT> __global__ __launch_bounds__(256) void distill_bwd_row_kernel(const DistillArgs a) {
  constexpr int E = Piece<T>::E;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds_rows[];
  __shared__ float ws[4][kDistillMax];
  __shared__ int vs[4][kDistillMax];
  const int t = threadIdx.x & 63, rw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + rw;
  if (row >= a.n) return;
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  T *dz = static_cast<T *>(a.dz) + row * a.V;
  const int V = (int)a.V;
  const Cut<T> cut(z, V);
  Teacher<64> te;
  te.load(a, row, t);
  const float w = a.g[row] * a.T, base = a.stats[2 * row], L = a.stats[2 * row + 1];
  T *x = fetch_row<T, NT>(z, cut, V, lds_rows + rw * lds_row_bytes<T>(V), t);
  row_has_come();
  te.gather(a, x);
  const bool some = te.sum(a, nullptr);
  const float f = w / L;
  auto grad = [&](float v) { return some ? f * power(v, base, a.c2) : 0.0f; };
  // the gradient takes the logits' place in LDS, its k places are corrected there, and it leaves in whole lines
  uint4 *pieces = reinterpret_cast<uint4 *>(x + cut.head);
  for (int i = t; i < cut.full; i += 64) {
    float v[E];
    widen<T>(pieces[i], v);
    T y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = (T)grad(v[e]);
    __builtin_memcpy(&pieces[i], y, 16);
  }
  const bool end = t < cut.head + V - cut.rest;
  const int at = t < cut.head ? t : t - cut.head + cut.rest;
  if (end) x[at] = (T)grad((float)x[at]);
  if (some) put_entries<T, 64>(a, te, t, ws[rw], vs[rw], w, x, grad);
  row_sync<64>();
  const bool vec = (reinterpret_cast<uintptr_t>(dz + cut.head) & 15) == 0;
  for (int i = t - cut.skip; i < cut.full; i += 64) {
    if (i < 0) continue;
    T y[E];
    __builtin_memcpy(y, &pieces[i], 16);
    put_piece<T>(dz + cut.head + (int64_t)i * E, y, vec);
  }
  if (end) dz[at] = x[at];
}

// Rows of up to kDistillRow bytes go through LDS, longer ones take a workgroup each and no LDS (forward + backward, us, LDS
// and workgroup: 50176 rows of 8 KB 91 + 140 and 160 + 196; 12544 rows of 32 KB 145 + 184 and 81 + 156, too few waves fit).
constexpr int64_t kDistillRow = 10 * 1024;
constexpr int64_t kDistillCache = (int64_t)256 << 20;      // bytes; see load16

template <typename T, bool NT> static void distill_launch(const DistillArgs &a, bool backward, hipStream_t s) {
  if (a.V * (int64_t)sizeof(T) <= kDistillRow) {
    const unsigned grid = (unsigned)((a.n + 3) / 4), lds = 4 * lds_row_bytes<T>(a.V);
    if (backward) hipLaunchKernelGGL((distill_bwd_row_kernel<T, NT>), dim3(grid), dim3(256), lds, s, a);
    else hipLaunchKernelGGL((distill_fwd_row_kernel<T, NT>), dim3(grid), dim3(256), lds, s, a);
  } else {
    if (backward) hipLaunchKernelGGL((distill_bwd_kernel<T, NT>), dim3((unsigned)a.n), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((distill_fwd_kernel<T, NT>), dim3((unsigned)a.n), dim3(256), 0, s, a);
  }
}

constexpr int64_t kDistillRows = (int64_t)1 << 23;         // of a launch, which takes fewer than 2^32 threads

template <typename T> static int distill_run(const DistillArgs &a, bool backward, hipStream_t s) {
  const bool nt = a.n * a.V * (int64_t)sizeof(T) > kDistillCache;
  for (int64_t r = 0; r < a.n; r += kDistillRows) {
    DistillArgs b = a;
    b.n = a.n - r < kDistillRows ? a.n - r : kDistillRows;
    b.z = static_cast<const T *>(a.z) + r * a.stride;
    if (a.k) { b.t = a.t + r * a.k; b.idx = a.idx + r * a.k; }
    if (a.stats) b.stats = a.stats + 2 * r;
    if (backward) { b.g = a.g + r; b.dz = static_cast<T *>(a.dz) + r * a.V; }
    else b.loss = a.loss + r;
    if (nt) distill_launch<T, true>(b, backward, s);
    else distill_launch<T, false>(b, backward, s);
    HSGK_LAUNCH_CHECK();
  }
  return 0;
}

static int distill_check(const void *logits, int dtype, int64_t n, int64_t V, int64_t row_stride, const float *teacher,
                         const int64_t *index, int k, float temperature) {
  HSGK_REQUIRE(dtype >= 0 && dtype <= 2, "dtype: 0 float32, 1 bfloat16, 2 float16");
  HSGK_REQUIRE(n >= 0 && n < ((int64_t)1 << 31), "rows outside 0 .. 2^31 - 1");
  HSGK_REQUIRE(V >= 1 && V < ((int64_t)1 << 31), "classes outside 1 .. 2^31 - 1");
  HSGK_REQUIRE(k >= 0 && k <= kDistillMax, "teacher entries outside 0 .. HSGK_DISTILL_MAX_K");
  HSGK_REQUIRE(isfinite(temperature) && temperature > 0.0f && isfinite(1.4426950408889634f / temperature),
               "the temperature is positive and finite, and so is its inverse");
  HSGK_REQUIRE(n == 0 || (logits && (k == 0 || (teacher && index))), "null argument");
  HSGK_REQUIRE(row_stride >= 0, "negative stride");
  HSGK_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == 0 ? 4 : 2) == 0, "the logits are not aligned to their elements");
  return 0;
}

static int distill_go(int dtype, const DistillArgs &a, bool backward, hipStream_t s) {
  (void)hipGetLastError();
  return dtype == 0 ? distill_run<float>(a, backward, s)
                    : dtype == 1 ? distill_run<__bf16>(a, backward, s) : distill_run<_Float16>(a, backward, s);
}

}  // namespace hsgk

using namespace hsgk;

extern "C" {

int hsgk_topk_distill_fwd(const void *logits, int dtype, int64_t n, int64_t V, int64_t row_stride, const float *teacher,
                          const int64_t *index, int k, float temperature, float *loss, float *stats, hsgk_stream_t stream) {
  if (int rc = distill_check(logits, dtype, n, V, row_stride, teacher, index, k, temperature)) return rc;
  if (n == 0) return 0;
  HSGK_REQUIRE(loss, "null argument");
  DistillArgs a = {logits, n, V, row_stride, teacher, index, k, temperature, 1.4426950408889634f / temperature, loss, stats,
                   nullptr, nullptr};
  return distill_go(dtype, a, false, static_cast<hipStream_t>(stream));
}

int hsgk_topk_distill_bwd(const void *logits, int dtype, int64_t n, int64_t V, int64_t row_stride, const float *teacher,
                          const int64_t *index, int k, float temperature, const float *stats, const float *grad,
                          void *dlogits, hsgk_stream_t stream) {
  if (int rc = distill_check(logits, dtype, n, V, row_stride, teacher, index, k, temperature)) return rc;
  if (n == 0) return 0;
  HSGK_REQUIRE(stats && grad && dlogits, "null argument");
  HSGK_REQUIRE(reinterpret_cast<uintptr_t>(dlogits) % (dtype == 0 ? 4 : 2) == 0, "dlogits is not aligned to its elements");
  DistillArgs a = {logits, n, V, row_stride, teacher, index, k, temperature, 1.4426950408889634f / temperature, nullptr,
                   const_cast<float *>(stats), grad, dlogits};
  return distill_go(dtype, a, true, static_cast<hipStream_t>(stream));
}

}  // extern "C"
