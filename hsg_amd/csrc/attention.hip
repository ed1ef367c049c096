// attention.hip -- multi-head attention and its backward pass behind the C ABI: checks, work plan, launches.
// The kernels and their mathematics are in attention_tiles.h.
#include <math.h>

#include "attention_tiles.h"

namespace hsgk {

struct AttnPlan {
  bool wk;          // 32 columns a workgroup, its waves share the streamed rows (else 128 columns, 32 a wave)
  int splits;       // parts of the streamed rows, joined by a second kernel
};

// Workgroups the plan aims for: two for each of the 256 CUs.
constexpr int64_t kAttnGroups = 512;

static AttnPlan attn_plan(int64_t heads, int64_t columns, int64_t rows) {
  AttnPlan p;
  p.wk = columns <= 32 || heads * ((columns + 127) / 128) < kAttnGroups / 2;
  const int64_t groups = heads * ((columns + (p.wk ? 31 : 127)) / (p.wk ? 32 : 128));
  const int64_t tile = p.wk ? 128 : 64;
  int64_t s = groups > 0 ? (kAttnGroups + groups - 1) / groups : 1;
  const int64_t most = rows / (2 * tile);
  if (s > most) s = most;
  p.splits = s > 1 ? (int)s : 1;
  return p;
}

static int padded_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct AttnSpace {
  float *delta, *part, *part2, *ml;
  size_t bytes;
};

static AttnSpace attn_space(const hsgk_attention_args &a, bool backward, void *base) {
  Carver c(base);
  AttnSpace w = {};
  const int64_t heads = (int64_t)a.B * a.G, C = (int64_t)a.L * (a.H / a.G);
  const size_t dp = (size_t)padded_width(a.D);
  const AttnPlan f = attn_plan(heads, C, a.S);
  if (!backward) {
    if (f.splits > 1) {
      w.part = c.take<float>((size_t)f.splits * heads * C * dp);
      w.ml = c.take<float>((size_t)f.splits * heads * C * 2);
    }
  } else {
    const AttnPlan r = attn_plan(heads, a.S, C);
    const size_t n1 = f.splits > 1 ? (size_t)f.splits * heads * C * dp : 0;
    const size_t n2 = r.splits > 1 ? (size_t)r.splits * heads * a.S * dp : 0;
    w.delta = c.take<float>((size_t)heads * C);
    w.part = c.take<float>(n1 > n2 ? n1 : n2);               // (the two passes follow each other)
    if (n2) w.part2 = c.take<float>(n2);
  }
  w.bytes = c.off;
  return w;
}

// whether 16-byte pieces of the rows are aligned
static int pieces(const void *p, const int64_t *st, int D, int size) {
  const int64_t e = 16 / size;
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && D % e == 0 && (!st || (st[0] % e == 0 && st[1] % e == 0 && st[2] % e == 0));
}

static int attn_check(const hsgk_attention_args *p, bool backward) {
  HSGK_REQUIRE(p, "null argument");
  const hsgk_attention_args &a = *p;
  HSGK_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "dtype: 0 float32, 1 bfloat16, 2 float16");
  HSGK_REQUIRE(a.B >= 0 && a.L >= 0 && a.S >= 0, "negative size");
  HSGK_REQUIRE(a.H >= 1 && a.G >= 1 && a.H % a.G == 0, "the query heads are a multiple of the key heads");
  HSGK_REQUIRE(a.D >= 1 && a.D <= HSGK_ATTENTION_MAX_WIDTH, "head width outside 1 .. 128");
  HSGK_REQUIRE(isfinite(a.scale) && a.scale > 0.0f, "the scale is positive and finite");
  const int64_t C = (int64_t)a.L * (a.H / a.G), most = (int64_t)1 << 30;
  HSGK_REQUIRE(C <= most && a.S <= most, "more than 2^30 rows a head");
  const int64_t rows = (C > a.S ? C : a.S) + 128;
  HSGK_REQUIRE((int64_t)a.B * a.G <= most && (int64_t)a.B * a.G * rows <= ((int64_t)1 << 38) / padded_width(a.D),
               "more rows than one launch covers");
  const bool some = (int64_t)a.B * a.L > 0, keys = (int64_t)a.B * a.S > 0;
  HSGK_REQUIRE(!some || (a.q && a.out), "null argument");
  HSGK_REQUIRE(!keys || (a.k && a.v), "null argument");
  if (backward) {
    HSGK_REQUIRE(!some || (a.dout && a.lse && a.dq), "null argument");
    HSGK_REQUIRE((!a.dk) == (!a.dv), "dk and dv come together");
  }
  const int size = a.dtype == 0 ? 4 : 2;
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

static AttnArgs attn_args(const hsgk_attention_args &p) {
  AttnArgs a = {};
  const int size = p.dtype == 0 ? 4 : 2;
  a.q = p.q; a.k = p.k; a.v = p.v; a.g = p.dout; a.o = p.out;
  for (int i = 0; i < 3; ++i) { a.qs[i] = p.q_stride[i]; a.ks[i] = p.k_stride[i]; a.vs[i] = p.v_stride[i]; a.gs[i] = p.dout_stride[i]; }
  a.pad = p.padding; a.pad_b = p.padding_stride;
  a.B = p.B; a.L = p.L; a.S = p.S; a.H = p.H; a.G = p.G; a.HG = p.H / p.G; a.D = p.D; a.C = p.L * a.HG;
  a.causal = p.causal != 0;
  a.qvec = pieces(a.q, a.qs, a.D, size); a.kvec = pieces(a.k, a.ks, a.D, size); a.vvec = pieces(a.v, a.vs, a.D, size);
  a.gvec = pieces(a.g, a.gs, a.D, size); a.ovec = pieces(a.o, nullptr, a.D, size);
  a.scale = p.scale; a.c2 = p.scale * 1.4426950408889634f;
  a.lse = p.lse;
  return a;
}

static int attn_go(int dtype, AttnPass pass, const AttnArgs &a, bool wk, hipStream_t s) {
  return dtype == 0 ? attn_f32(pass, a, wk, s) : dtype == 1 ? attn_bf16(pass, a, wk, s) : attn_f16(pass, a, wk, s);
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
  AttnArgs a = attn_args(*args);
  const AttnPlan p = attn_plan((int64_t)a.B * a.G, a.C, a.S);
  const AttnSpace w = attn_space(*args, false, args->workspace);
  a.splits = p.splits; a.part = w.part; a.ml = w.ml; a.out = args->out;
  return attn_go(args->dtype, kAttnFwd, a, p.wk, static_cast<hipStream_t>(stream));
}

int hsgk_attention_bwd(const hsgk_attention_args *args, hsgk_stream_t stream) {
  if (int rc = attn_check(args, true)) return rc;
  if (args->B == 0) return 0;
  (void)hipGetLastError();
  hipStream_t s = static_cast<hipStream_t>(stream);
  AttnArgs a = attn_args(*args);
  const AttnSpace w = attn_space(*args, true, args->workspace);
  a.delta = w.delta; a.part = w.part; a.part2 = w.part2;
  if (a.C > 0) {
    const AttnPlan p = attn_plan((int64_t)a.B * a.G, a.C, a.S);
    a.splits = p.splits; a.out = args->dq;
    if (int rc = attn_go(args->dtype, kAttnDq, a, p.wk, s)) return rc;
  }
  if (a.S > 0 && args->dk) {
    const AttnPlan p = attn_plan((int64_t)a.B * a.G, a.S, a.C);
    a.splits = p.splits; a.out = args->dk; a.out2 = args->dv;
    if (int rc = attn_go(args->dtype, kAttnDkv, a, p.wk, s)) return rc;
  }
  return 0;
}

}  // extern "C"
