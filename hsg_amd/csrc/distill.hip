// distill.hip -- distillation of a softmax over V classes (prototypes) from a teacher's k best of them.
//
// Per row: p = softmax over the k entries of t / T (an entry outside [0, V) or with t = -inf does not count),
//   q = softmax over all V of z / T,   loss = T^2 sum_j p_j (log p_j - log q_{idx_j})   (no entry: 0)
//   dz_v = g T (q_v - sum_{j: idx_j = v} p_j)                                            (no entry: 0)
// Both passes are bound by memory: the forward reads the row once (running maximum and sum per thread, joined at the
// end) and leaves (maximum, sum) for the backward, which reads the row and writes the gradient once; the k places
// where p enters are written again at the end of the row, out of the cache, by one thread for each different index.
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

// the E elements from e0 on of a row of V, 16 bytes at once where they are all inside (e0 is chosen so that the address
// is aligned); `fill` elsewhere
template <typename T>
__device__ __forceinline__ void get_piece(const T *row, int64_t e0, int64_t V, float fill, float (&x)[Piece<T>::E]) {
  constexpr int E = Piece<T>::E;
  if (e0 >= 0 && e0 + E <= V) {
    const uint4 u = *reinterpret_cast<const uint4 *>(row + e0);
    T y[E];
    __builtin_memcpy(y, &u, 16);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = (float)y[i];
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = e0 + i >= 0 && e0 + i < V ? (float)row[e0 + i] : fill;
  }
}

// teacher: probabilities of the row's entries into tp, their indices into ti (-1: does not count); returns whether any counts
template <int P>
__device__ __forceinline__ bool teacher_row(const DistillArgs &a, int64_t row, int t, float *tp, int64_t *ti, float *red,
                                            float &top, float &mass) {
  float m = -__builtin_inff();
  for (int j = t; j < a.k; j += P) {
    const float x = a.t[row * a.k + j];
    const int64_t v = a.idx[row * a.k + j];
    const bool ok = v >= 0 && v < a.V && !(x == -__builtin_inff());
    ti[j] = ok ? v : -1;
    tp[j] = x;
    if (ok) m = fmaxf(m, x != x ? __builtin_inff() : x);
  }
  m = row_max<P>(m, red);
  top = m;
  const bool some = m > -__builtin_inff();
  float s = 0.0f;
  for (int j = t; j < a.k; j += P) {
    const float p = ti[j] >= 0 ? __builtin_amdgcn_exp2f((tp[j] - m) * a.c2) : 0.0f;
    s += p;
  }
  mass = row_sum<P>(s, red);
  return some;
}

template <typename T, int P> __global__ __launch_bounds__(256) void distill_fwd_kernel(const DistillArgs a) {
  constexpr int E = Piece<T>::E, R = 256 / P, U = 4;
  __shared__ float tps[R][kDistillMax], red[4];
  __shared__ int64_t tis[R][kDistillMax];
  const int t = threadIdx.x % P, rw = threadIdx.x / P;
  const int64_t row = (int64_t)blockIdx.x * R + rw;
  if (P == 64 && row >= a.n) return;                       // (one wave a row: no barrier of the workgroup follows)
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  const int off = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int64_t pieces = (a.V + off + E - 1) / E;
  float m = -__builtin_inff(), l = 0.0f;
  for (int64_t i0 = t; i0 < pieces; i0 += (int64_t)P * U) {
    float x[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) get_piece<T>(z, (i0 + (int64_t)u * P) * E - off, a.V, -__builtin_inff(), x[u]);
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) top = fmaxf(top, x[u][e]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    l *= __builtin_amdgcn_exp2f((m - base) * a.c2);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) l += __builtin_amdgcn_exp2f((x[u][e] - base) * a.c2);
    m = top;
  }
  const float M = row_max<P>(m, red), base = M == -__builtin_inff() ? 0.0f : M;
  const float L = row_sum<P>(l * __builtin_amdgcn_exp2f((m - base) * a.c2), red);
  float top, mass;
  const bool some = teacher_row<P>(a, row, t, tps[rw], tis[rw], red, top, mass);
  float s = 0.0f;
  if (some) {
    const float lm = logf(mass), lL = logf(L);
    for (int j = t; j < a.k; j += P) {
      const int64_t v = tis[rw][j];
      if (v < 0) continue;
      const float d = (tps[rw][j] - top) / a.T;
      const float p = __builtin_amdgcn_exp2f((tps[rw][j] - top) * a.c2) / mass;
      if (p != 0.0f) s += p * ((d - lm) - (((float)z[v] - base) / a.T - lL));
    }
  }
  s = row_sum<P>(s, red);
  if (t == 0) {
    a.loss[row] = some ? a.T * a.T * s : 0.0f;
    if (a.stats) { a.stats[2 * row] = base; a.stats[2 * row + 1] = L; }
  }
}

template <typename T, int P> __global__ __launch_bounds__(256) void distill_bwd_kernel(const DistillArgs a) {
  constexpr int E = Piece<T>::E, R = 256 / P, U = 2;
  __shared__ float tps[R][kDistillMax], red[4];
  __shared__ int64_t tis[R][kDistillMax];
  const int t = threadIdx.x % P, rw = threadIdx.x / P;
  const int64_t row = (int64_t)blockIdx.x * R + rw;
  if (P == 64 && row >= a.n) return;
  const T *z = static_cast<const T *>(a.z) + row * a.stride;
  T *dz = static_cast<T *>(a.dz) + row * a.V;
  const int off = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const bool vec = off == (int)((reinterpret_cast<uintptr_t>(dz) & 15) / sizeof(T));
  const int64_t pieces = (a.V + off + E - 1) / E;
  float top, mass;
  const bool some = teacher_row<P>(a, row, t, tps[rw], tis[rw], red, top, mass);
  const float w = a.g[row] * a.T;
  const float base = a.stats[2 * row], f = some ? w / a.stats[2 * row + 1] : 0.0f;
  for (int64_t i0 = t; i0 < pieces; i0 += (int64_t)P * U) {
    float x[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) get_piece<T>(z, (i0 + (int64_t)u * P) * E - off, a.V, 0.0f, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e0 = (i0 + (int64_t)u * P) * E - off;
      T y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = (T)(some ? f * __builtin_amdgcn_exp2f((x[u][e] - base) * a.c2) : 0.0f);
      if (vec && e0 >= 0 && e0 + E <= a.V) {
        uint4 o;
        __builtin_memcpy(&o, y, 16);
        *reinterpret_cast<uint4 *>(dz + e0) = o;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e0 + e >= 0 && e0 + e < a.V) dz[e0 + e] = y[e];
      }
    }
  }
  if (!some) return;                                       // (the same for all threads of the row)
  row_sync<P>();                                           // the row is written before its k places are written again
  for (int j = t; j < a.k; j += P) {
    const int64_t v = tis[rw][j];
    if (v < 0) continue;
    float p = 0.0f;
    bool first = true;
    for (int x = 0; x < a.k; ++x)
      if (tis[rw][x] == v) {
        if (x < j) first = false;
        p += __builtin_amdgcn_exp2f((tps[rw][x] - top) * a.c2);
      }
    if (first) dz[v] = (T)(f * __builtin_amdgcn_exp2f(((float)z[v] - base) * a.c2) - w * (p / mass));
  }
}

// Rows of up to this many elements take a wave each, longer ones a workgroup.
constexpr int64_t kDistillWaveRow = 2048;

template <typename T> static int distill_run(const DistillArgs &a, bool backward, hipStream_t s) {
  const bool wave = a.V <= kDistillWaveRow;
  const unsigned grid = (unsigned)(wave ? (a.n + 3) / 4 : a.n);
  if (!backward) {
    if (wave) hipLaunchKernelGGL((distill_fwd_kernel<T, 64>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((distill_fwd_kernel<T, 256>), dim3(grid), dim3(256), 0, s, a);
  } else {
    if (wave) hipLaunchKernelGGL((distill_bwd_kernel<T, 64>), dim3(grid), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((distill_bwd_kernel<T, 256>), dim3(grid), dim3(256), 0, s, a);
  }
  HSGK_LAUNCH_CHECK();
  return 0;
}

static int distill_check(const void *logits, int dtype, int64_t n, int64_t V, int64_t row_stride, const float *teacher,
                         const int64_t *index, int k, float temperature) {
  HSGK_REQUIRE(dtype >= 0 && dtype <= 2, "dtype: 0 float32, 1 bfloat16, 2 float16");
  HSGK_REQUIRE(n >= 0 && n < ((int64_t)1 << 31), "rows outside 0 .. 2^31 - 1");
  HSGK_REQUIRE(V >= 1 && V < ((int64_t)1 << 31), "classes outside 1 .. 2^31 - 1");
  HSGK_REQUIRE(k >= 0 && k <= kDistillMax, "teacher entries outside 0 .. HSGK_DISTILL_MAX_K");
  HSGK_REQUIRE(isfinite(temperature) && temperature > 0.0f, "the temperature is positive and finite");
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
