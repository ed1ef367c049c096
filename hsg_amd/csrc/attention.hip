// attention.hip -- multi-head attention and its backward pass behind the C ABI: checks, work plan, launches.
// The kernels and their mathematics are in attention_tiles.h.
#include <math.h>

#include "attention_tiles.h"

namespace hsgk {

static int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }
// (float32, whose products cost seven times as much, also to 96: 30 heads x 930 x 930, width 72, forward, dq, dk and dv 123 + 169 +
// 222 us, 150 + 210 + 275 with 128; the 16-bit types have no such form, nor one of 48: not measured)
static int padded_width(const hsgk_attention_args &a) {
  return a.D <= 32 ? 32 : a.D <= 64 ? 64 : a.dtype == 0 && a.D <= 96 ? 96 : 128;
}

struct AttnPlan {
  AttnShape shape;
  int splits;          // parts of the streamed rows, joined by a second kernel
};

// Shared columns where all their workgroups run at once, one, two or three a CU by LDS (forward, dq, dk and dv, us, shared and
// with 128 columns: float32, 28 heads x 131 x 203, width 36, 126 workgroups 16 + 17 + 25 and 23 + 31 + 49; float16, 36 heads x
// 510 x 510, width 80, 576 workgroups 49 + 46 + 64 and 16 + 25 + 31), and for few columns anyway, of which 128 would be mostly
// empty (forward and dq; bfloat16, 1024 heads, width 64: 1 column x 2048 keys 106 and 124 forward, 16 x 512 28 + 27 and 26 +
// 32, 32 x 512 31 + 29 and 26 + 32; float32, 512 heads, width 48: 64 x 512 79 + 93 and 79 + 111, 96 x 512 117 + 139 and 82 +
// 117).
// Split rows where there are fewer workgroups than `room`, what the CUs hold at a time: more only add partial results (one token of
// 16 heads over 2 x 32768 keys, width 128: 256 workgroups 25 + 4 us, 512 30 + 4; 30 heads x 930 x 930, width 72, float32, 240
// workgroups 143 us, 480 153 + 9; narrower 16-bit heads, whose workgroups fit three times on a CU, have the same room without
// a measurement of their own).  Causal blocks differ in length: two for each CU there (dk and dv of 4 key heads, 8192 keys:
// 1105 us in one part, 760 + 16 in two).
static AttnPlan attn_plan(const hsgk_attention_args &a, AttnPass pass) {
  const bool dkv = pass == kAttnDkv;
  const int64_t heads = (int64_t)a.B * a.G, queries = (int64_t)a.L * (a.H / a.G);
  const int64_t columns = dkv ? a.S : queries, rows = dkv ? queries : a.S;
  const int bytes = padded_width(a) * elem_size(a.dtype);                 // of a row in LDS
  AttnPlan p;
  const int64_t shared = heads * ((columns + 31) / 32), at_once = bytes >= 256 ? 256 : bytes >= 128 ? 512 : 768;
  p.shape = columns <= (a.dtype == 0 ? 64 : 15) || shared <= at_once ? kAttnShared : kAttnWide;
  const int64_t groups = p.shape == kAttnWide ? heads * ((columns + 127) / 128) : shared;
  const int64_t room = (p.shape == kAttnWide || bytes >= 256) && !a.causal ? 256 : 512;
  int64_t s = groups > 0 ? room / groups : 1;
  const int64_t most = rows / 256;
  if (s < 1) s = 1;
  if (p.shape == kAttnShared && bytes >= 256 && !a.causal && groups <= room) {
    // rounds of the CUs over parts: 160 workgroups leave a hundred CUs idle, three times as many take two rounds of a third (one
    // token of 32 heads on 8, 20 x 8192 keys, width 128, bfloat16: 155 us, 134 + 5; two workgroups a CU fill it as they are)
    auto time = [&](int64_t parts) { return (double)((groups * parts + room - 1) / room) / (double)parts; };
    const int64_t first = s;
    for (int64_t t = first + 1; t <= first + 3; ++t)
      if (time(t) < 0.9 * time(s)) s = t;
  }
  if (s > most) s = most;
  if (s > kAttnMaxSplits) s = kAttnMaxSplits;
  p.splits = s > 1 ? (int)s : 1;
  return p;
}

// whether 16-byte pieces of the rows are aligned
static bool pieces(const void *p, const int64_t *st, int D, int size) {
  const int64_t e = 16 / size;
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && D % e == 0 && (!st || (st[0] % e == 0 && st[1] % e == 0 && st[2] % e == 0));
}

static int loaded_width(const hsgk_attention_args &a) { const int e = 16 / elem_size(a.dtype); return (a.D + e - 1) / e * e; }

struct AttnSpace {
  float *delta, *part, *part2, *ml;
  void *packed[4];                    // aligned copies of q, k, v, dout where their own rows are not aligned
  size_t bytes;
};

static AttnSpace attn_space(const hsgk_attention_args &a, bool backward, void *base) {
  Carver c(base);
  AttnSpace w = {};
  const int64_t heads = (int64_t)a.B * a.G, C = (int64_t)a.L * (a.H / a.G);
  const size_t dp = (size_t)padded_width(a);
  const AttnPlan f = attn_plan(a, backward ? kAttnDq : kAttnFwd);
  if (!backward) {
    if (f.splits > 1) {
      w.part = c.take<float>((size_t)f.splits * heads * C * dp);
      w.ml = c.take<float>((size_t)f.splits * heads * C * 2);
    }
  } else {
    const AttnPlan r = attn_plan(a, kAttnDkv);
    const size_t n1 = f.splits > 1 ? (size_t)f.splits * heads * C * dp : 0;
    const size_t n2 = r.splits > 1 ? (size_t)r.splits * heads * a.S * dp : 0;
    w.delta = c.take<float>((size_t)heads * C);
    w.part = c.take<float>(n1 > n2 ? n1 : n2);               // (the two passes follow each other)
    if (n2) w.part2 = c.take<float>(n2);
  }
  const void *from[4] = {a.q, a.k, a.v, a.dout};
  const int64_t *st[4] = {a.q_stride, a.k_stride, a.v_stride, a.dout_stride};
  for (int i = 0; i < (backward ? 4 : 3); ++i)
    if (!pieces(from[i], st[i], a.D, elem_size(a.dtype))) {
      const bool query = i == 0 || i == 3;
      w.packed[i] = c.take<char>((size_t)a.B * (query ? (size_t)a.L * a.H : (size_t)a.S * a.G) * loaded_width(a) * elem_size(a.dtype));
    }
  w.bytes = c.off;
  return w;
}

// workgroups of a pass
static int64_t attn_groups(const hsgk_attention_args &a, AttnPass pass) {
  const AttnPlan p = attn_plan(a, pass);
  const int64_t columns = pass == kAttnDkv ? a.S : (int64_t)a.L * (a.H / a.G), per = p.shape == kAttnWide ? 128 : 32;
  return (int64_t)a.B * a.G * ((columns + per - 1) / per) * p.splits;
}

static int attn_check(const hsgk_attention_args *p, bool backward) {
  HSGK_REQUIRE(p, "null argument");
  const hsgk_attention_args &a = *p;
  HSGK_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "dtype: 0 float32, 1 bfloat16, 2 float16");
  HSGK_REQUIRE(a.B >= 0 && a.L >= 0 && a.S >= 0, "negative size");
  HSGK_REQUIRE(a.H >= 1 && a.G >= 1 && a.H % a.G == 0, "the query heads are a multiple of the key heads");
  HSGK_REQUIRE(a.D >= 1 && a.D <= HSGK_ATTENTION_MAX_WIDTH, "head width outside 1 .. 128");
  HSGK_REQUIRE(a.scale > 0.0f && isfinite(a.scale * 1.4426950408889634f), "the scale is positive and finite");
  const int64_t C = (int64_t)a.L * (a.H / a.G), most = (int64_t)1 << 30;
  HSGK_REQUIRE(C <= most && a.S <= most, "more than 2^30 rows a head");
  const int64_t rows = (C > a.S ? C : a.S) + 128;
  HSGK_REQUIRE((int64_t)a.B * a.G <= most && (int64_t)a.B * a.G * rows <= ((int64_t)1 << 38) / padded_width(a),
               "more rows than one launch covers");
  const int64_t grid = ((int64_t)1 << 24) - 1;                // of 256 threads each
  HSGK_REQUIRE(attn_groups(a, kAttnFwd) <= grid && (!backward || attn_groups(a, kAttnDkv) <= grid), "more rows than one launch covers");
  const bool some = (int64_t)a.B * a.L > 0, keys = (int64_t)a.B * a.S > 0;
  HSGK_REQUIRE(!some || (a.q && a.out), "null argument");
  HSGK_REQUIRE(!keys || (a.k && a.v), "null argument");
  if (backward) {
    HSGK_REQUIRE(!some || (a.dout && a.lse && a.dq), "null argument");
    HSGK_REQUIRE((!a.dk) == (!a.dv), "dk and dv come together");
  }
  const int size = elem_size(a.dtype);
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                        (backward ? reinterpret_cast<uintptr_t>(a.dout) : 0);
  HSGK_REQUIRE(all % size == 0, "a tensor is not aligned to its elements");
  const uintptr_t outs = reinterpret_cast<uintptr_t>(a.out) |
                         (backward ? reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk) | reinterpret_cast<uintptr_t>(a.dv) : 0);
  HSGK_REQUIRE(outs % 16 == 0, "an output is not aligned to 16 bytes");
  const size_t need = attn_space(a, backward, nullptr).bytes;
  HSGK_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "workspace too small");
  HSGK_REQUIRE(need == 0 || reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "the workspace is not aligned to 16 bytes");
  return 0;
}

// Rows whose 16-byte pieces are not aligned, copied into aligned ones, zeros past their end: [B, n, heads, pieces].  A thread
// copies a piece in words of G bytes, 2^lg threads a row (10 x 4158 x 6 rows of 36 bfloat16: 9.2 us, 4.1 TB/s; 30 element by
// element).
template <int G> struct Word;
template <> struct Word<2> { using T = uint16_t; };
template <> struct Word<4> { using T = uint32_t; };
template <> struct Word<8> { using T = uint2; };

template <int G>
__global__ __launch_bounds__(256) void attn_pack_kernel(const char *from, int64_t sb, int64_t sl, int64_t sh, int64_t rows, int n, int heads,
                                                        int bytes, int pieces, int lg, uint4 *to) {
  using W = typename Word<G>::T;
  const int p = (int)threadIdx.x & ((1 << lg) - 1), per = 256 >> lg;
  if (p >= pieces) return;
  for (int64_t row = (int64_t)blockIdx.x * per + ((int)threadIdx.x >> lg); row < rows; row += (int64_t)gridDim.x * per) {
    int64_t b, i;
    int head;
    if (rows <= 0x7fffffff) {                              // (a division of 64 bits takes as long as the copy)
      const unsigned j = (unsigned)row / (unsigned)heads, c = j / (unsigned)n;
      head = (int)((unsigned)row - j * heads);
      b = c; i = j - c * n;
    } else {
      const int64_t j = row / heads;
      head = (int)(row - j * heads);
      b = j / n; i = j - b * n;
    }
    const char *src = from + b * sb + i * sl + head * sh + 16 * p;
    W x[16 / G];
#pragma unroll
    for (int c = 0; c < 16 / G; ++c) x[c] = 16 * p + c * G < bytes ? *reinterpret_cast<const W *>(src + c * G) : W{};
    uint4 y;
    __builtin_memcpy(&y, x, 16);
    to[row * pieces + p] = y;
  }
}

static int attn_pack(const void *from, const int64_t *st, int size, int64_t B, int n, int heads, int D, int DL, void *to, hipStream_t s) {
  const int64_t rows = B * n * heads;
  if (rows == 0) return 0;
  const int bytes = D * size, count = DL * size / 16;
  const uintptr_t all = reinterpret_cast<uintptr_t>(from) | (uintptr_t)(st[0] * size) | (uintptr_t)(st[1] * size) | (uintptr_t)(st[2] * size) |
                        (uintptr_t)bytes;
  int lg = 0;
  while ((1 << lg) < count) ++lg;
  const int64_t blocks = (rows + (256 >> lg) - 1) / (256 >> lg);
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384)), block(256);
  const auto kernel = all % 8 == 0 ? attn_pack_kernel<8> : all % 4 == 0 ? attn_pack_kernel<4> : attn_pack_kernel<2>;
  hipLaunchKernelGGL(kernel, grid, block, 0, s, static_cast<const char *>(from), st[0] * size, st[1] * size, st[2] * size, rows, n, heads,
                     bytes, count, lg, static_cast<uint4 *>(to));
  HSGK_LAUNCH_CHECK();
  return 0;
}

// the kernels' arguments; copies what they could not read in 16-byte pieces
static int attn_args(const hsgk_attention_args &p, const AttnSpace &w, bool backward, hipStream_t s, AttnArgs &a) {
  a = {};
  const int size = elem_size(p.dtype);
  a.B = p.B; a.L = p.L; a.S = p.S; a.H = p.H; a.G = p.G; a.HG = p.H / p.G; a.D = p.D; a.C = p.L * a.HG;
  a.DL = loaded_width(p);
  const void *from[4] = {p.q, p.k, p.v, p.dout};
  const int64_t *st[4] = {p.q_stride, p.k_stride, p.v_stride, p.dout_stride};
  const void **to[4] = {&a.q, &a.k, &a.v, &a.g};
  int64_t *ts[4] = {a.qs, a.ks, a.vs, a.gs};
  for (int i = 0; i < (backward ? 4 : 3); ++i) {
    if (!w.packed[i]) {
      *to[i] = from[i];
      for (int x = 0; x < 3; ++x) ts[i][x] = st[i][x];
      continue;
    }
    const bool query = i == 0 || i == 3;
    const int n = query ? p.L : p.S, heads = query ? p.H : p.G;
    const int rc = attn_pack(from[i], st[i], size, p.B, n, heads, p.D, a.DL, w.packed[i], s);
    if (rc) return rc;
    *to[i] = w.packed[i];
    ts[i][0] = (int64_t)n * heads * a.DL; ts[i][1] = (int64_t)heads * a.DL; ts[i][2] = a.DL;
  }
  a.o = p.out;
  a.pad = p.padding; a.pad_b = p.padding_stride;
  a.causal = p.causal != 0;
  a.ovec = pieces(a.o, nullptr, a.D, size);
  a.scale = p.scale; a.c2 = p.scale * 1.4426950408889634f;
  a.lse = p.lse;
  return 0;
}

static int attn_go(int dtype, AttnPass pass, const AttnArgs &a, AttnShape shape, hipStream_t s) {
  if (pass == kAttnDkv)
    return dtype == 0 ? attn_dkv_f32(pass, a, shape, s) : dtype == 1 ? attn_dkv_bf16(pass, a, shape, s) : attn_dkv_f16(pass, a, shape, s);
  return dtype == 0 ? attn_f32(pass, a, shape, s) : dtype == 1 ? attn_bf16(pass, a, shape, s) : attn_f16(pass, a, shape, s);
}

}  // namespace hsgk

using namespace hsgk;

extern "C" {

size_t hsgk_attention_workspace_bytes(const hsgk_attention_args *args, int backward) {
  if (!args || args->B < 0 || args->L < 0 || args->S < 0 || args->H < 1 || args->G < 1 || args->H % args->G || args->D < 1 ||
      args->D > HSGK_ATTENTION_MAX_WIDTH)
    return 0;
  return attn_space(*args, backward != 0, nullptr).bytes;
}

int hsgk_attention_fwd(const hsgk_attention_args *args, hsgk_stream_t stream) {
  if (int rc = attn_check(args, false)) return rc;
  if ((int64_t)args->B * args->L == 0) return 0;
  (void)hipGetLastError();
  hipStream_t s = static_cast<hipStream_t>(stream);
  const AttnSpace w = attn_space(*args, false, args->workspace);
  AttnArgs a;
  if (int rc = attn_args(*args, w, false, s, a)) return rc;
  const AttnPlan p = attn_plan(*args, kAttnFwd);
  a.splits = p.splits; a.part = w.part; a.ml = w.ml; a.out = args->out;
  return attn_go(args->dtype, kAttnFwd, a, p.shape, s);
}

int hsgk_attention_bwd(const hsgk_attention_args *args, hsgk_stream_t stream) {
  if (int rc = attn_check(args, true)) return rc;
  if (args->B == 0) return 0;
  (void)hipGetLastError();
  hipStream_t s = static_cast<hipStream_t>(stream);
  const AttnSpace w = attn_space(*args, true, args->workspace);
  AttnArgs a;
  if (int rc = attn_args(*args, w, true, s, a)) return rc;
  a.delta = w.delta; a.part = w.part; a.part2 = w.part2;
  if (a.C > 0) {
    const AttnPlan p = attn_plan(*args, kAttnDq);
    if (args->dtype != 0) a.have_delta = a.pad || a.S <= exact_keys(padded_width(*args)) ? 1 : a.causal ? 2 : 0;   // queries of few keys
    if (a.have_delta) {
      a.splits = 1;
      if (int rc = attn_go(args->dtype, kAttnDelta, a, p.shape, s)) return rc;
    }
    a.splits = p.splits; a.out = args->dq;
    if (int rc = attn_go(args->dtype, kAttnDq, a, p.shape, s)) return rc;
  }
  if (a.S > 0 && args->dk) {
    const AttnPlan p = attn_plan(*args, kAttnDkv);
    a.splits = p.splits; a.out = args->dk; a.out2 = args->dv;
    if (int rc = attn_go(args->dtype, kAttnDkv, a, p.shape, s)) return rc;
  }
  return 0;
}

}  // extern "C"
