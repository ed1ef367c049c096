"""Attention (hsg_amd.models.embeddings.transformer_clusters.attention, MultiheadAttention) against the definition in
float64, element by element within bounds that are derived here from the roundings the kernels make."""
import ctypes
import math

import pytest

EPS32 = 2.0 ** -24            # half a step of float32


def _half_step(dtype):
  import torch
  return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------------------------------------------
# arguments that are refused (no GPU needed)
def _args():
  import torch
  return [torch.zeros(2, 5, 4, 8), torch.zeros(2, 7, 2, 8), torch.zeros(2, 7, 2, 8)]


@pytest.mark.parametrize('change, error', [
    (lambda t: [t[0][0], t[1], t[2]], ValueError),                               # three dimensions
    (lambda t: [t[0], t[1][:, :6], t[2]], ValueError),                           # key and value differ
    (lambda t: [t[0][:1], t[1], t[2]], ValueError),                              # batch
    (lambda t: [t[0][..., :7], t[1], t[2]], ValueError),                         # head width
    (lambda t: [t[0][:, :, :3], t[1], t[2]], ValueError),                        # 3 query heads over 2 key heads
    (lambda t: [t[0], t[1][:, :, :0], t[2][:, :, :0]], ValueError),              # no key head
    (lambda t: [x[..., :0] for x in t], ValueError),                             # width 0
    (lambda t: [x.repeat(1, 1, 1, 17) for x in t], ValueError),                  # width 136
    (lambda t: [t[0].double(), t[1].double(), t[2].double()], TypeError),
    (lambda t: [t[0], t[1].half(), t[2].half()], TypeError),
])
def test_attention_refuses(change, error):
  from hsg_amd.models.embeddings.transformer_clusters import attention
  with pytest.raises(error):
    attention(*change(_args()))


def test_attention_refuses_masks_scales_and_cpu_tensors():
  import torch
  from hsg_amd import _lib
  from hsg_amd.models.embeddings.transformer_clusters import attention
  q, k, v = _args()
  with pytest.raises(TypeError):
    attention(q, k, v, key_padding_mask=torch.zeros(2, 7))
  with pytest.raises(ValueError):
    attention(q, k, v, key_padding_mask=torch.zeros(2, 6, dtype=torch.bool))
  for scale in (0.0, -1.0, math.inf, math.nan):
    with pytest.raises(ValueError):
      attention(q, k, v, scale=scale)
  with pytest.raises(_lib.HsgkError):
    attention(q, k, v)


def test_the_torch_op_refuses_tangents():
  """(before it looks at the device: no GPU needed)"""
  import torch
  import torch.autograd.forward_ad as fwd
  from hsg_amd import _torch_ops
  ops = _torch_ops.ops()
  if ops is None:
    pytest.skip('the torch binding is not built')
  with fwd.dual_level():
    for i in range(3):
      t = _args()
      t[i] = fwd.make_dual(t[i], torch.ones_like(t[i]))
      with torch.no_grad(), pytest.raises(RuntimeError, match='forward-mode'):
        ops.attention(*t, None, False, 0.5)
      with pytest.raises(RuntimeError, match='forward-mode'):
        ops.attention(*t, None, False, 0.5)


def test_the_torch_op_refuses_heads_that_do_not_divide():
  """(the op itself, not its Python entry: no key head was a division by zero in the host's code)"""
  import torch
  from hsg_amd import _torch_ops
  ops = _torch_ops.ops()
  if ops is None:
    pytest.skip('the torch binding is not built')
  q, k, v = _args()
  for query, key, value in ((q, k[:, :, :0], v[:, :, :0]), (q[:, :, :3], k, v)):
    with pytest.raises(RuntimeError, match='multiple of the key heads'):
      ops.attention(query.requires_grad_(True), key, value, None, False, 0.5)
  with pytest.raises(RuntimeError, match='no CPU path'):
    ops.attention(q, k, v, None, False, 0.5)


def test_c_entry_refuses_bad_arguments():
  """The C entry returns -1 with a message before anything is launched."""
  from hsg_amd import _lib
  L = _lib.lib()
  buf = ctypes.create_string_buffer(1 << 16)
  base = (ctypes.addressof(buf) + 255) // 256 * 256

  def good():
    a = _lib.AttentionArgs()
    a.q = a.k = a.v = a.out = a.lse = a.dout = a.dq = a.dk = a.dv = a.workspace = base
    a.workspace_bytes = 1 << 14
    a.B, a.L, a.S, a.H, a.G, a.D, a.scale = 1, 2, 3, 4, 2, 8, 0.5
    return a

  for field, value in (('dtype', 3), ('B', -1), ('L', -1), ('S', -2), ('H', 3), ('G', 0), ('D', 0), ('D', 129), ('scale', 0.0),
                       ('scale', math.nan), ('q', None), ('k', None), ('out', None), ('q', base + 2), ('out', base + 4),
                       ('L', (1 << 30))):
    a = good()
    setattr(a, field, value)
    assert L.hsgk_attention_fwd(ctypes.byref(a), None) == -1, field
    assert L.hsgk_last_error()
  for field, value in (('dout', None), ('lse', None), ('dq', None), ('dk', None), ('workspace', None), ('workspace_bytes', 0)):
    a = good()
    setattr(a, field, value)
    assert L.hsgk_attention_bwd(ctypes.byref(a), None) == -1, field
  assert L.hsgk_attention_fwd(None, None) == -1
  a = good()
  a.L = 0                                                     # nothing to do: no pointer is looked at
  a.q = a.out = None
  assert L.hsgk_attention_fwd(ctypes.byref(a), None) == 0


def test_c_entry_refuses_more_than_a_launch_covers():
  from hsg_amd import _lib
  L = _lib.lib()
  buf = ctypes.create_string_buffer(1 << 16)
  base = (ctypes.addressof(buf) + 255) // 256 * 256
  for B, Lq, scale in ((1 << 24, 1, 0.5), (1 << 22, 129, 0.5), (1, 1, 3e38)):
    a = _lib.AttentionArgs()
    a.q = a.k = a.v = a.out = base
    a.B, a.L, a.S, a.H, a.G, a.D, a.scale = B, Lq, 3, 4, 4, 8, scale
    assert L.hsgk_attention_fwd(ctypes.byref(a), None) == -1
    assert (b'scale' if scale > 1 else b'launch') in L.hsgk_last_error()


def test_module_refuses_what_the_kernels_do_not_offer():
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  x = torch.zeros(3, 2, 8)
  m = torch.nn.MultiheadAttention(8, 2)
  assert tc.use_attention_kernels(torch.nn.Sequential(m)) == 1 and type(m) is tc.MultiheadAttention
  assert tc.use_attention_kernels(m) == 0                     # already switched
  with pytest.raises(ValueError):
    m(x, x, x, attn_mask=torch.zeros(3, 3, dtype=torch.bool))
  with pytest.raises(ValueError):
    m(x[:, 0], x[:, 0], x[:, 0])
  for kwargs in ({'dropout': 0.1}, {'add_bias_kv': True}, {'add_zero_attn': True}):
    keep, bad = torch.nn.MultiheadAttention(8, 2), torch.nn.MultiheadAttention(8, 2, **kwargs)
    with pytest.raises(ValueError):
      tc.use_attention_kernels(torch.nn.Sequential(keep, bad))
    assert type(keep) is torch.nn.MultiheadAttention          # nothing is switched by half
  with pytest.raises(ValueError):
    tc.use_attention_kernels(torch.nn.MultiheadAttention(512, 2))
  drop = tc.MultiheadAttention(8, 2, dropout=0.1)
  with pytest.raises(ValueError):
    drop(x, x, x)


@pytest.mark.parametrize('kind', ['encoder', 'decoder'])
@pytest.mark.parametrize('training', [True, False])
@pytest.mark.parametrize('batch_first', [True, False])
def test_torchs_layers_can_be_called_with_padding(kind, training, batch_first):
  """What use_attention_kernels switches can be called: torch's layers get as far as the device check (they hand a bool mask
  on as floating point)."""
  import torch
  from hsg_amd import _lib
  from hsg_amd.models.embeddings import transformer_clusters as tc
  x, pad = torch.zeros(2, 6, 32), torch.arange(6)[None] >= torch.tensor([6, 4])[:, None]
  x = x if batch_first else x.transpose(0, 1)
  if kind == 'encoder':
    layer = torch.nn.TransformerEncoderLayer(32, 4, dropout=0.0, batch_first=batch_first).train(training)
    args, kwargs, n = (x,), {'src_key_padding_mask': pad}, 1
  else:
    layer = torch.nn.TransformerDecoderLayer(32, 4, dropout=0.0, batch_first=batch_first).train(training)
    args, kwargs, n = (x, x), {'tgt_key_padding_mask': pad, 'memory_key_padding_mask': pad}, 2
  assert tc.use_attention_kernels(layer) == n
  with pytest.raises(_lib.HsgkError):
    layer(*args, **kwargs)


@pytest.mark.parametrize('batch_first', [True, False])
def test_causal_masks_of_torchs_layers(batch_first):
  """torch's layers pass a causal mask together with is_causal=True: such a call gets as far as the device check, a mask that
  is_causal cannot be true of is refused."""
  import torch
  from hsg_amd import _lib
  from hsg_amd.models.embeddings import transformer_clusters as tc
  x, mask = torch.zeros(2, 6, 32), torch.nn.Transformer.generate_square_subsequent_mask(6)
  y, z = (t if batch_first else t.transpose(0, 1) for t in (x, torch.zeros(2, 8, 32)))
  enc = torch.nn.TransformerEncoderLayer(32, 4, dropout=0.0, batch_first=batch_first)
  dec = torch.nn.TransformerDecoderLayer(32, 4, dropout=0.0, batch_first=batch_first)
  m = torch.nn.MultiheadAttention(32, 4, batch_first=batch_first)
  assert tc.use_attention_kernels(torch.nn.ModuleList([enc, dec, m])) == 4
  for call in (lambda: enc(y, src_mask=mask, is_causal=True), lambda: dec(y, y, tgt_mask=mask, tgt_is_causal=True),
               lambda: m(y, y, y, attn_mask=mask, is_causal=True)):
    with pytest.raises(_lib.HsgkError):
      call()
  for call in (lambda: m(y, y, y, attn_mask=mask), lambda: m(y, z, z, attn_mask=torch.zeros(6, 8), is_causal=True),
               lambda: m(y, y, y, attn_mask=torch.zeros(8, 8), is_causal=True), lambda: enc(y, src_mask=mask),
               lambda: m(y, z, z, attn_mask=mask, is_causal=True),
               lambda: m(y, y, y, attn_mask=torch.zeros(8, 6, 6), is_causal=True)):
    with pytest.raises(ValueError):
      call()


def test_dropout_counts_in_training_only():
  import torch
  from hsg_amd import _lib
  from hsg_amd.models.embeddings import transformer_clusters as tc
  x = torch.zeros(6, 2, 32)
  m = torch.nn.MultiheadAttention(32, 4, dropout=0.1)
  with pytest.raises(ValueError):
    tc.use_attention_kernels(m)
  assert type(m) is torch.nn.MultiheadAttention
  m.eval()
  assert tc.use_attention_kernels(m) == 1
  with pytest.raises(_lib.HsgkError):                        # as far as the device check
    m(x, x, x)
  m.train()
  with pytest.raises(ValueError, match='dropout'):
    m(x, x, x)


def test_weights_that_are_asked_for_are_refused():
  """(they were None without a word)"""
  import torch
  from hsg_amd import _lib
  from hsg_amd.models.embeddings import transformer_clusters as tc
  x = torch.zeros(6, 2, 32)
  m = torch.nn.MultiheadAttention(32, 4)
  tc.use_attention_kernels(m)
  with pytest.raises(ValueError, match='need_weights'):
    m(x, x, x, need_weights=True)
  for kwargs in ({}, {'need_weights': False}):
    with pytest.raises(_lib.HsgkError):                      # as far as the device check
      m(x, x, x, **kwargs)


# ---------------------------------------------------------------------------------------------------------------------
# the definition in float64 and the bounds
def _visible(B, L, S, mask, causal, device):
  import torch
  seen = torch.ones((B, 1, L, S), dtype=torch.bool, device=device)
  if causal:
    i, j = torch.arange(L, device=device)[:, None], torch.arange(S, device=device)[None]
    seen = seen & (j <= i + (S - L))
  if mask is not None:
    seen = seen & ~mask[:, None, None, :]
  return seen


def _exact(q, k, v, g, mask, causal, scale, few=False):
  """Outputs, gradients and the bound of each in float64.

  With u the half step of the element type (0 for float32 inside the products) and e = 2^-24:
  a score of D products is off by at most e (D + 3) scale sum |q k| =: ds, its exponent's argument by e |s| log2(e) more,
  numerator and denominator both: a probability is off by a relative r = 2 (ds + 3 e |s|max) + e (S + 16), and by u where
  it enters a product.  out: (r + u) sum p |v| + u |out|.  dp = do.v is off by e (D + 3) sum |do v|; delta = do.out by the
  same with out and by (error of the stored out) |do|; ds = p (dp - delta) by r (+ u) of itself, and so on.  Sums of n
  terms in float32 add e n times the sum of magnitudes.  The hardware's exp2 gives 0 where the result is below the smallest
  normal number, so a probability (of the row's largest, or of the row's sum) is off by another f = 2^-126 at most: f (|dp| +
  |delta|) in ds and f |do| in each term of dv, f |v| in each of out.
  few: delta is sum p dp, off by r + e (S + 4) of its terms and by theirs, and the rounding of ds by u of ds itself."""
  import torch
  dtype = q.dtype
  u = 0.0 if dtype is torch.float32 else _half_step(dtype)
  uo = _half_step(dtype)
  B, L, H, D = q.shape
  S, G = k.shape[1], k.shape[2]
  hg = H // G
  Q, GO = (x.double().permute(0, 2, 1, 3) for x in (q, g))                     # [B,H,L,D]
  K, V = (x.double().permute(0, 2, 1, 3).repeat_interleave(hg, 1) for x in (k, v))
  seen = _visible(B, L, S, mask, causal, q.device)
  if mask is not None:                                                         # a masked key may hold anything
    K = K.masked_fill(mask[:, None, :, None], 0.0)
    V = V.masked_fill(mask[:, None, :, None], 0.0)
  s = scale * (Q @ K.transpose(-1, -2).contiguous())
  some = seen.any(-1, keepdim=True)
  s = s.masked_fill(~seen, -math.inf)
  p = torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1).masked_fill(~seen, 0.0)
  out = p @ V
  dp = GO @ V.transpose(-1, -2).contiguous()
  delta = (GO * out).sum(-1, keepdim=True)
  ds = p * (dp - delta)
  dq, dk, dv = scale * (ds @ K), scale * (ds.transpose(-1, -2) @ Q), p.transpose(-1, -2) @ GO
  # bounds
  e = EPS32
  ab = scale * (Q.abs() @ K.abs().transpose(-1, -2).contiguous())
  zero = torch.zeros_like(s)
  far = torch.where(seen, s.abs() + ab, zero).amax(-1, keepdim=True) if S else torch.zeros_like(some, dtype=torch.float64)
  r = 2 * e * ((D + 3) * (ab.amax(-1, keepdim=True) if S else 0.0) + 3 * far) + e * (S + 16)
  A = p @ V.abs()
  f = 2.0 ** -126 * seen.double().expand(-1, H, -1, -1)
  e_out = (r + u) * A + f @ V.abs() + uo * out.abs()
  e_dp = e * (D + 3) * (GO.abs() @ V.abs().transpose(-1, -2).contiguous())
  e_delta = e * (D + 3) * (GO.abs() * out.abs()).sum(-1, keepdim=True) + (GO.abs() * e_out).sum(-1, keepdim=True)
  e_round = u * (dp.abs() + delta.abs())
  if few:
    e_delta = (p * (e_dp + (r + e * (S + 4)) * dp.abs()) + f * dp.abs()).sum(-1, keepdim=True)
    e_round = u * (dp - delta).abs()
  e_ds = p * ((r + 4 * e) * (dp.abs() + delta.abs()) + e_round + e_dp + e_delta) + f * (dp.abs() + delta.abs())
  if dtype is torch.float16:                      # below the type's normal range, after the scaling by powers of two
    e_ds = e_ds + 2.0 ** -34 * ds.abs().amax(-1, keepdim=True) if S else e_ds
    e_ds = e_ds + 2.0 ** -34 * ds.abs().amax(-2, keepdim=True) if L else e_ds
  e_dq = scale * (e_ds @ K.abs() + e * (S + 4) * (ds.abs() @ K.abs())) + uo * dq.abs()
  e_dk = scale * (e_ds.transpose(-1, -2) @ Q.abs() + e * (hg * L + 4) * (ds.abs().transpose(-1, -2) @ Q.abs()))
  e_dv = ((r + u) * p + f).transpose(-1, -2) @ GO.abs() + e * (hg * L + 4) * (p.transpose(-1, -2) @ GO.abs())
  if dtype is torch.float16:
    e_dv = e_dv + 2.0 ** -40 * GO.abs().sum(-2, keepdim=True)

  def back(x):
    return x.permute(0, 2, 1, 3)

  def shared(x):                                                               # [B,H,S,D] -> [B,S,G,D]
    return back(x.view(B, G, hg, S, D).sum(2))

  dk, dv = shared(dk), shared(dv)
  res = {'out': back(out), 'dq': back(dq), 'dk': dk, 'dv': dv}
  # 2 step of the smallest numbers: results below the normal range of the type
  tiny = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}[dtype]
  bound = {'out': back(e_out), 'dq': back(e_dq), 'dk': shared(e_dk) + uo * dk.abs(), 'dv': shared(e_dv) + uo * dv.abs()}
  return res, {n: b * 1.01 + tiny for n, b in bound.items()}


def _compare(got, want, bound):
  import torch
  for name in got:
    a = got[name].double()
    assert a.shape == want[name].shape, name
    off = (a - want[name]).abs() - bound[name]
    assert bool(torch.isfinite(a).all()), name + ' is not finite'
    assert not off.numel() or float(off.max()) <= 0, '%s: off by %g over the bound %g' % (
        name, float(off.max()), float(bound[name].flatten()[off.argmax()]))


def _make(seed, dtype, B, L, S, H, G, D, mask=None, spread=1.0):
  import torch
  g = torch.Generator().manual_seed(seed)
  t = [torch.randn(s, generator=g).mul(spread).to(dtype).cuda() for s in ((B, L, H, D), (B, S, G, D), (B, S, G, D))]
  go = torch.randn((B, L, H, D), generator=g).to(dtype).cuda()
  m = None
  if mask == 'ragged':                                                         # the last item has no key
    n = torch.tensor([max(0, S - (b * S) // max(B - 1, 1)) for b in range(B)])
    m = (torch.arange(S) >= n[:, None]).cuda()
  elif mask == 'scattered':
    m = (torch.rand((B, S), generator=g) < 0.4).cuda()
  elif mask == 'all':
    m = torch.ones((B, S), dtype=torch.bool).cuda()
  return t, go, m


def _run(t, go, m, causal=False, scale=None):
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  leaves = [x.detach().requires_grad_(True) for x in t]
  out = attention(*leaves, key_padding_mask=m, is_causal=causal, scale=scale)
  assert out.dtype == t[0].dtype and out.is_contiguous()
  grads = torch.autograd.grad(out, leaves, go)
  with torch.no_grad():
    assert torch.equal(attention(*t, key_padding_mask=m, is_causal=causal, scale=scale), out)
  torch.cuda.synchronize()
  return {'out': out.detach(), 'dq': grads[0], 'dk': grads[1], 'dv': grads[2]}


def _check(seed, name, B, L, S, H, G, D, mask=None, causal=False, scale=None, spread=1.0):
  import torch
  t, go, m = _make(seed, getattr(torch, name), B, L, S, H, G, D, mask, spread)
  want, bound = _exact(*t, go, m, causal, scale if scale is not None else D ** -0.5)
  _compare(_run(t, go, m, causal, scale), want, bound)


TYPES = ['float32', 'bfloat16', 'float16']
SHAPES = [                            # B, L, S, H, G, D, mask, causal
    (1, 1, 1, 1, 1, 1, None, False),
    (2, 1, 5, 2, 1, 7, None, False),
    (2, 5, 1, 2, 2, 32, None, False),
    (3, 33, 64, 4, 2, 36, 'ragged', False),
    (2, 64, 33, 3, 1, 64, 'scattered', False),
    (2, 130, 257, 2, 2, 64, 'ragged', False),
    (2, 200, 31, 6, 2, 72, None, True),          # the first queries see no key
    (2, 31, 200, 4, 4, 128, None, True),
    (2, 129, 129, 2, 1, 128, 'scattered', True),
    (2, 17, 40, 2, 2, 40, 'all', False),
    (1, 3, 1500, 4, 1, 64, 'ragged', False),     # few queries: the keys are split
    (1, 1500, 3, 4, 1, 64, None, False),         # few keys: the queries are split
    (1, 300, 700, 1, 1, 100, 'scattered', False),
    (2, 256, 256, 8, 8, 32, 'ragged', False),    # the clustering transformer's encoder
    (16, 130, 140, 16, 16, 33, 'ragged', False),   # enough heads: 128 columns a workgroup
    (16, 140, 130, 16, 16, 64, None, True),
    (17, 129, 150, 8, 8, 128, 'scattered', False),
    (8, 512, 300, 8, 8, 64, None, False),        # ... and the streamed rows in two parts
    (8, 300, 512, 16, 8, 48, None, True),
    (2, 400, 300, 2, 1, 64, None, True),         # the first 100 queries see no key, many see few
    (1, 900, 900, 2, 1, 36, None, True),         # few heads: both sides in parts
    (1, 3, 3000, 2, 1, 64, 'scattered', False),  # more than eight parts
    (5, 300, 600, 8, 8, 128, 'ragged', False),   # 128 columns a workgroup and parts
    (2, 512, 640, 16, 8, 100, None, True),
    (70, 40, 50, 8, 8, 64, 'ragged', False),     # many heads of few columns, shared by float32 alone
    (12, 129, 150, 8, 8, 80, 'ragged', False),   # float32: padded to 96
    (2, 300, 330, 12, 4, 96, None, True),
    (1, 3, 3000, 2, 1, 90, 'scattered', False),
    (3, 70, 600, 4, 2, 65, 'ragged', False),
    (20, 1, 900, 32, 8, 128, 'ragged', False),   # 160 workgroups: three parts
]


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(str(v) for v in s))
def test_attention_and_gradients(name, shape):
  _check(7, name, *shape)


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
def test_attention_scales_and_large_scores(name):
  """A scale of the caller's, and scores of several hundred: probabilities that are 1 for one key and 0 for the others."""
  _check(8, name, 2, 40, 70, 2, 2, 64, 'ragged', False, scale=0.03)
  _check(9, name, 2, 40, 70, 2, 2, 64, None, False, scale=1.0, spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize('offset', [0.0, 300.0, 3000.0, -30000.0])
@pytest.mark.parametrize('B, L, H', [(1, 1, 1), (1, 200, 2), (16, 130, 16), (1, 40, 1)])
def test_an_offset_of_all_scores_costs_nothing(B, L, H, offset):
  """Width 1 and queries of 1, so that the scores are the keys, without rounding.  What they have in common leaves the softmax,
  and the parts of a row that is summed in steps weigh alike: keys that grow by 10 once a tile with values that shrink as much.

  With e = 2^-24 and far the spread of the scores: an argument (s log2(e) fused with a reference, log2(e) rounded, the same
  reference throughout) is off by 4 e far, exp2 by 2 e here and 2 e for each of up to eight rescalings and joins, a sum of S terms
  by e S, twice (numerator and denominator), the value's product and the division by 4 e."""
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  S = 700
  gen = torch.Generator().manual_seed(51)
  step = torch.arange(S) // 130
  k = (offset + 10.0 * step + torch.rand((B, S), generator=gen))
  v = (1.0 + torch.rand((B, S), generator=gen)) * torch.exp(-10.0 * step.double()).float()
  k, v = k[:, :, None, None].cuda(), v[:, :, None, None].cuda()
  out = attention(torch.ones((B, L, H, 1), device='cuda'), k.expand(B, S, H, 1), v.expand(B, S, H, 1), scale=1.0)
  s = k[:, :, 0, 0].double()
  want = (torch.softmax(s, 1) * v[:, :, 0, 0].double()).sum(1)
  far = float((s.amax(1) - s.amin(1)).max())
  off = (out.double() - want[:, None, None, None]).abs() / want[:, None, None, None]
  assert float(off.max()) <= EPS32 * 2 * (4 * far + 2 + 16 + S + 4), float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('shape', [
    (2, 9, 1, 2, 1, 24, None, False),
    (3, 40, 2, 4, 2, 32, None, False),
    (2, 70, 5, 2, 2, 64, None, False),
    (2, 50, 50, 4, 1, 128, None, True),
    (3, 40, 640, 2, 2, 40, 'first three', False),    # the queries' keys would be split
    (16, 130, 60, 16, 16, 64, 'ragged', False),      # 128 columns a workgroup
    (16, 130, 130, 16, 16, 36, None, True),
    (17, 129, 256, 8, 8, 128, 'scattered', False),
    (2, 60, 700, 2, 1, 24, 'ragged', False),         # narrow heads: more keys are few
], ids=lambda s: 'x'.join(str(v) for v in s))
def test_gradients_over_few_keys(name, shape):
  """Values with a common part, which dp - delta cancels: the gradients have the roundings of ds and of the result alone
  (delta from the stored output would add its rounding of the common part)."""
  import torch
  B, L, S, H, G, D, mask, causal = shape
  (q, k, v), go, m = _make(31, getattr(torch, name), B, L, S, H, G, D, None if mask == 'first three' else mask)
  if mask == 'first three':
    m = (torch.arange(S) >= 3).expand(B, S).cuda()
  v = (v.float() + 8.0).to(v.dtype)
  want, bound = _exact(q, k, v, go, m, causal, D ** -0.5, few=name != 'float32')
  _compare(_run([q, k, v], go, m, causal), want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
def test_attention_without_queries_or_keys(name):
  import torch
  dtype = getattr(torch, name)
  for B, L, S in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
    t, go, m = _make(1, dtype, B, L, S, 2, 1, 8)
    got = _run(t, go, m)
    assert got['out'].shape == (B, L, 2, 8) and got['dk'].shape == (B, S, 1, 8)
    for x in got.values():
      assert not bool(x.any())


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
def test_masked_keys_may_hold_anything(name):
  """NaN, infinities and the type's lowest value in masked keys and values change no bit; their gradients are zero."""
  import torch
  dtype = getattr(torch, name)
  for L, S, causal in ((70, 90, False), (3, 600, False), (90, 90, True)):
    t, go, m = _make(11, dtype, 3, L, S, 4, 2, 40, 'scattered')
    m[1] = True
    clean = [t[0]] + [x.masked_fill(m[:, :, None, None], 0.0) for x in t[1:]]
    want = _run(clean, go, m, causal)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
      dirty = [t[0]] + [x.masked_fill(m[:, :, None, None], bad) for x in t[1:]]
      got = _run(dirty, go, m, causal)
      for n in want:
        assert torch.equal(got[n], want[n]), (n, bad)
    assert not bool(want['dk'][m].any()) and not bool(want['dv'][m].any())
    assert not bool(want['out'][1].any()) and not bool(want['dq'][1].any())


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
def test_attention_strides(name):
  """Heads before rows, a packed projection, rows that are not 16-byte aligned, expanded and reversed-order inputs, a
  last dimension that is not contiguous, an expanded incoming gradient: the bits of the contiguous call."""
  import torch
  dtype = getattr(torch, name)
  B, L, H, D = 2, 70, 4, 40
  t, go, m = _make(12, dtype, B, L, L, H, H, D, 'ragged')
  want = _run(t, go, m)

  def same(views, go=go, want=want):
    for v, x in zip(views, t):
      assert torch.equal(v, x)
    got = _run(views, go, m)
    for n in want:
      assert torch.equal(got[n], want[n]), n

  same([x.transpose(1, 2).contiguous().transpose(1, 2) for x in t])
  packed = torch.stack(t, 2)                                                   # [B, L, 3, H, D]
  same([packed[:, :, i] for i in range(3)])
  same([x.transpose(0, 1).contiguous().transpose(0, 1) for x in t])
  wide = [torch.cat([x.new_full((B, L, H, 1), math.nan), x], -1)[..., 1:] for x in t]
  same(wide)                                                                   # odd strides, misaligned start
  same([x.transpose(2, 3).contiguous().transpose(2, 3) for x in t])            # last dimension not contiguous
  same(t, go=go.transpose(1, 2).contiguous().transpose(1, 2))
  one = go[:1, :1].expand(B, L, H, D)
  ref = _run(t, one.contiguous(), m)
  same(t, go=one, want=ref)
  same(t, go=go[..., :1].expand(B, L, H, D), want=_run(t, go[..., :1].expand(B, L, H, D).contiguous(), m))
  lone = [t[0], t[1][:1].expand(B, -1, -1, -1), t[2][:1].expand(B, -1, -1, -1)]
  got = _run(lone, go, m)
  ref = _run([x.contiguous() for x in lone], go, m)
  for n in ref:
    assert torch.equal(got[n], ref[n]), n
  mt = m.t().contiguous().t()                                                  # a mask with other strides
  got = _run(t, go, mt)
  for n in want:
    assert torch.equal(got[n], want[n]), n


@pytest.mark.gpu
def test_gradients_against_differences():
  """A directional derivative of sum(out * g) by a central difference of the float64 definition equals <gradient, direction>;
  the difference of the kernel's own float32 outputs agrees too."""
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  t, go, m = _make(13, torch.float32, 2, 20, 30, 4, 2, 16, 'ragged')
  m[1, 0] = False
  got = _run(t, go, m)
  gen = torch.Generator().manual_seed(3)
  h = 2.0 ** -7
  for i, n in enumerate(('dq', 'dk', 'dv')):
    d = torch.randn(t[i].shape, generator=gen).cuda()
    d = d / d.norm()
    up, down = list(t), list(t)
    up[i], down[i] = t[i] + h * d, t[i] - h * d
    slope = float(((attention(*up, key_padding_mask=m).double() - attention(*down, key_padding_mask=m).double())
                   * go.double()).sum()) / (2 * h)
    inner = float((got[n].double() * d.double()).sum())
    # the difference leaves h^2 / 6 of the third derivative (scores move by about |k| h scale < 0.02 here: < 1e-3 of the
    # gradient's norm), float32 outputs 2^-23 * sqrt(count) * |go| / h < 1e-3
    assert abs(slope - inner) <= 2e-3 * (1 + float(got[n].double().norm())), (n, slope, inner)


@pytest.mark.gpu
def test_only_wanted_gradients():
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  t, go, m = _make(14, torch.float32, 2, 40, 50, 4, 2, 32, 'scattered')
  want = _run(t, go, m)
  for pick in ((0,), (1,), (2,), (0, 2), (1, 2)):
    leaves = [x.detach().requires_grad_(i in pick) for i, x in enumerate(t)]
    out = attention(*leaves, key_padding_mask=m)
    got = torch.autograd.grad(out, [leaves[i] for i in pick], go)
    for i, g in zip(pick, got):
      assert torch.equal(g, want[('dq', 'dk', 'dv')[i]])


@pytest.mark.gpu
@pytest.mark.parametrize('binding', ['torch', 'ctypes'])
def test_gradients_cannot_be_differentiated(binding, monkeypatch):
  """create_graph works, and a gradient of the gradient raises instead of counting as zero."""
  import torch
  if binding == 'ctypes':
    monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  from hsg_amd.models.embeddings.transformer_clusters import attention
  t, go, _ = _make(5, torch.float32, 2, 9, 11, 2, 2, 16)
  leaves = [x.requires_grad_(True) for x in t]
  want = torch.autograd.grad(attention(*leaves), leaves, go)
  got = torch.autograd.grad(attention(*leaves), leaves, go, create_graph=True)
  for a, b in zip(got, want):
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match='differentiable once'):
      torch.autograd.grad(a.sum(), leaves, allow_unused=True, retain_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize('binding', ['torch', 'ctypes'])
def test_tangents_are_refused(binding, monkeypatch):
  """Forward-mode differentiation raises under both bindings, whether or not the primal requires a gradient; so does a stack that
  was switched over to the kernels."""
  import torch
  import torch.autograd.forward_ad as fwd
  from hsg_amd.models.embeddings import transformer_clusters as tc
  if binding == 'ctypes':
    monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  t, _, _ = _make(5, torch.float32, 2, 9, 11, 2, 2, 16)
  m = torch.nn.MultiheadAttention(32, 2).cuda()
  tc.use_attention_kernels(m)
  x = torch.randn((9, 2, 32), generator=torch.Generator().manual_seed(1)).cuda()
  for grad in (False, True):
    for i in range(3):
      with fwd.dual_level():
        u = [y.detach().requires_grad_(grad) for y in t]
        u[i] = fwd.make_dual(u[i], torch.ones_like(u[i]))
        with pytest.raises(RuntimeError):
          tc.attention(*u)
        with torch.no_grad(), pytest.raises(RuntimeError):
          tc.attention(*u)
    m.requires_grad_(grad)
    with fwd.dual_level():
      y = fwd.make_dual(x, torch.ones_like(x))
      with pytest.raises(RuntimeError):
        m(y, y, y)
  with fwd.dual_level():
    u = [y.detach().requires_grad_(True) for y in t]
    out = tc.attention(*u)                                                       # (without a tangent it runs)
    assert torch.autograd.grad(out, u, torch.ones_like(out), retain_graph=True)[0].shape == t[0].shape
    with pytest.raises(RuntimeError, match='forward-mode'):                      # a tangent of the incoming gradient
      torch.autograd.grad(out, u, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.gpu
def test_a_dimension_that_32_bits_do_not_hold_is_refused():
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  q = torch.zeros((1, 2, 1, 4), device='cuda')
  k = torch.zeros((1, 1, 1, 4), device='cuda').expand(1, (1 << 32) + 5, 1, 4)
  with pytest.raises(RuntimeError):
    attention(q, k, k)


@pytest.mark.gpu
def test_both_bindings_give_the_same_bits(monkeypatch):
  import torch
  t, go, m = _make(15, torch.bfloat16, 2, 70, 600, 4, 2, 64, 'ragged')
  a = _run(t, go, m)
  monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  b = _run(t, go, m)
  for n in a:
    assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
def test_attention_on_another_stream_and_twice_at_once():
  import torch
  cases = [_make(20 + i, torch.float32, 2, 50, 900, 4, 2, 64, 'ragged') for i in range(2)]
  want = [_run(*c) for c in cases]
  streams = [torch.cuda.Stream() for _ in cases]
  torch.cuda.synchronize()
  got = []
  for c, s in zip(cases, streams):
    with torch.cuda.stream(s):
      from hsg_amd.models.embeddings.transformer_clusters import attention
      leaves = [x.detach().requires_grad_(True) for x in c[0]]
      out = attention(*leaves, key_padding_mask=c[2])
      got.append([out] + list(torch.autograd.grad(out, leaves, c[1])))
  torch.cuda.synchronize()
  for w, g in zip(want, got):
    for n, x in zip(('out', 'dq', 'dk', 'dv'), g):
      assert torch.equal(w[n], x), n


@pytest.mark.gpu
def test_attention_captured_and_replayed():
  """Forward and backward in one graph, replayed on new inputs, with eager calls and synchronisations in between; two
  captured graphs do not share their workspaces."""
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  shapes = [(2, 3, 900, 4, 2, 64), (2, 80, 120, 4, 4, 32)]
  graphs = []
  for i, sh in enumerate(shapes):
    t, go, m = _make(30 + i, torch.bfloat16, *sh, 'ragged')
    leaves = [x.detach().requires_grad_(True) for x in t]

    def step(leaves=leaves, go=go, m=m):
      out = attention(*leaves, key_padding_mask=m)
      return [out] + list(torch.autograd.grad(out, leaves, go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      res = step()
    graphs.append((graph, leaves, go, m, res))
  for n in range(4):
    for i, (graph, leaves, go, m, res) in enumerate(graphs):
      new, go2, _ = _make(40 + 10 * n + i, torch.bfloat16, *shapes[i])
      with torch.no_grad():
        for a, b in zip(leaves, new):
          a.copy_(b)
        go.copy_(go2)
    for graph, *_ in graphs:
      graph.replay()
    torch.cuda.synchronize()
    for graph, leaves, go, m, res in graphs:
      want = _run([x.detach() for x in leaves], go, m)
      for name, x in zip(('out', 'dq', 'dk', 'dv'), res):
        assert torch.equal(want[name], x), (n, name)


@pytest.mark.gpu
def test_long_strides_pass_32_bits():
  """Keys and values inside a buffer whose row offsets pass 2^31 elements."""
  import torch
  S, G, D = 130, 1, 32
  stride = (1 << 31) // 100 // 8 * 8                                           # the last rows start past 2^31 elements
  big = torch.zeros((S * stride,), dtype=torch.float16, device='cuda')
  views = [torch.as_strided(big, (1, S, G, D), (S * stride, stride, D, 1), storage_offset=o) for o in (0, 64)]
  t, go, m = _make(16, torch.float16, 1, 40, S, 2, G, D)
  for v, x in zip(views, t[1:]):
    v.copy_(x)
  assert (S - 1) * stride > 1 << 31
  want = _run(t, go, m)
  got = _run([t[0]] + views, go, m)
  for n in want:
    assert torch.equal(want[n], got[n]), n


# ---------------------------------------------------------------------------------------------------------------------
# the module
def _transformer(E, heads, seed):
  """The shape of the clustering transformer: self-attention over the segments, queries that attend to them."""
  import torch
  torch.manual_seed(seed)

  class Stack(torch.nn.Module):
    def __init__(self):
      super().__init__()
      self.self_attn = torch.nn.MultiheadAttention(E, heads)
      self.norm = torch.nn.BatchNorm1d(E)
      self.cross = torch.nn.MultiheadAttention(E, heads)

    def forward(self, src, mask, query_embed, pos_embed):
      x, pos = src.permute(2, 0, 1), pos_embed.permute(2, 0, 1)
      q = query_embed[:, None].expand(-1, src.shape[0], -1)
      y = self.self_attn(x + pos, x + pos, value=x, key_padding_mask=mask)[0]
      x = self.norm((x + y).permute(1, 2, 0)).permute(2, 0, 1)
      c = self.cross(q, x + pos, value=x, key_padding_mask=mask)[0]
      return c.permute(1, 2, 0), x.permute(1, 2, 0)

  return Stack()


@pytest.mark.gpu
def test_clustering_transformer_on_the_kernels():
  """TransformerClustering.forward over a stack whose attention runs in libhsgk, against the same stack of torch modules:
  outputs and parameter gradients."""
  import copy
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  B, C, sl, tl, heads = 4, 64, 90, 8, 8

  class Clustering(tc.TransformerClusteringMixin, torch.nn.Module):
    def __init__(self, stack):
      super().__init__()
      self._transformer, self._num_clusters = stack, tl
      self.centroid_fc, self.centroid_feat_fc = torch.nn.Linear(C, C), torch.nn.Linear(C, C)

  ours = Clustering(_transformer(C, heads, 5)).cuda()
  plain = copy.deepcopy(ours)
  assert tc.use_attention_kernels(ours) == 2
  assert list(ours.state_dict()) == list(plain.state_dict())
  g = torch.Generator().manual_seed(6)
  src, pos = (torch.randn((B, C, sl), generator=g).cuda() for _ in range(2))
  query = torch.randn((tl, C), generator=g).cuda()
  mask = (torch.arange(sl)[None] >= torch.tensor([90, 60, 33, 1])[:, None]).cuda()
  res = []
  for net, double in ((ours, False), (plain, True)):
    args = [src, mask, query, pos]
    stack = net._transformer
    if double:
      stack, args = stack.double(), [x.double() if x.is_floating_point() else x for x in args]
    c, nodes = stack(*args)
    gen = torch.Generator().manual_seed(9)
    weights = [torch.randn(t.shape, generator=gen).cuda() for t in (c, nodes)]
    loss = sum((a * b.to(a.dtype)).sum() for a, b in zip((c, nodes), weights))
    grads = torch.autograd.grad(loss, list(stack.parameters()))
    res.append([c, nodes] + list(grads))
  # A chain of a dozen float32 products of at most a few hundred terms each: 2^-24 * 12 * 300 of the norm at the worst.
  # What BatchNorm takes out again (self_attn.out_proj.bias and the values' bias shift every node alike) has gradient 0,
  # and float32 leaves the rounding of a sum of n = B * sl terms: 2^-24 n of their norm, that of the weights of the nodes.
  floor = 2.0 ** -24 * B * sl * float(weights[1].norm())
  for a, b in zip(*res):
    assert float((a.double() - b).detach().norm()) <= 2.2e-4 * float(b.detach().norm()) + floor
  cent, feats, logits, nodes = ours(src, mask, query, pos)                     # the tail runs on the kernels' output
  assert cent.shape == (B, C, tl) and logits.shape == (B, tl, sl) and bool(torch.isfinite(logits).all())


@pytest.mark.gpu
@pytest.mark.parametrize('batch_first', [False, True])
def test_module_equals_torchs(batch_first):
  import copy
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  torch.manual_seed(2)
  for kwargs in ({}, {'kdim': 24, 'vdim': 40}, {'bias': False}):
    ref = torch.nn.MultiheadAttention(48, 4, batch_first=batch_first, **kwargs).cuda()
    ours = copy.deepcopy(ref)
    tc.use_attention_kernels(ours)
    q = torch.randn(3, 20, 48).cuda()
    k, v = torch.randn(3, 30, kwargs.get('kdim', 48)).cuda(), torch.randn(3, 30, kwargs.get('vdim', 48)).cuda()
    mask = (torch.arange(30)[None] >= torch.tensor([30, 17, 2])[:, None]).cuda()
    io = [x if batch_first else x.transpose(0, 1) for x in (q, k, v)]
    a, w = ours(*io, key_padding_mask=mask)
    b, _ = ref.double()(*[x.double() for x in io], key_padding_mask=mask)
    assert w is None and a.shape == b.shape
    a, b = a.detach(), b.detach()
    assert float((a.double() - b).norm()) <= 2.0 ** -24 * 400 * float(b.norm())   # three products of 24 .. 48 terms and the rows


def _norm_close(got, want, terms):
  """Norms: 2^-24 * terms of what a chain of float32 products and sums leaves."""
  a, b = got.detach().double(), want.detach()
  assert a.shape == b.shape and bool((a - b).isfinite().all())
  assert float((a - b).norm()) <= 2.0 ** -24 * terms * float(b.norm()), (float((a - b).norm()), float(b.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize('training', [True, False])
@pytest.mark.parametrize('batch_first', [True, False])
def test_torchs_encoder_layer_with_padding(training, batch_first):
  """A stock layer that was switched, with a bool mask that torch makes floating point: the rows that count and the gradients
  of what they add up to equal the unswitched layer's in float64."""
  import copy
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  torch.manual_seed(3)
  ours = torch.nn.TransformerEncoderLayer(32, 4, 48, dropout=0.0, batch_first=batch_first).cuda().train(training)
  plain = copy.deepcopy(ours).double()
  assert tc.use_attention_kernels(ours) == 1
  x = torch.randn(3, 20, 32).cuda()
  pad = (torch.arange(20)[None] >= torch.tensor([20, 13, 1])[:, None]).cuda()
  w = torch.randn(3, 20, 32).cuda().masked_fill(pad[..., None], 0.0)
  res = []
  for net, dtype in ((ours, torch.float32), (plain, torch.float64)):
    y = x.to(dtype).requires_grad_(True)
    out = net(y if batch_first else y.transpose(0, 1), src_key_padding_mask=pad)
    out = out if batch_first else out.transpose(0, 1)
    g = torch.autograd.grad((out * w.to(dtype)).sum(), [y, net.linear1.weight, net.self_attn.in_proj_weight,
                                                        net.self_attn.out_proj.weight])
    res.append([out.masked_fill(pad[..., None], 0.0)] + list(g))
  # a chain of ten products and norms of at most 60 rows or 48 terms each, whose errors a layer norm may double
  for a, b in zip(*res):
    _norm_close(a, b, 2 * 10 * 60)


@pytest.mark.gpu
@pytest.mark.parametrize('padded', [False, True])
def test_torchs_decoder_layer_with_causality(padded):
  """A stock decoder layer: causal self-attention (mask and is_causal), padded keys from elsewhere, against float64."""
  import copy
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  torch.manual_seed(5)
  ours = torch.nn.TransformerDecoderLayer(32, 4, 48, dropout=0.0, batch_first=True).cuda()
  plain = copy.deepcopy(ours).double()
  assert tc.use_attention_kernels(ours) == 2
  x, memory, w = torch.randn(3, 20, 32).cuda(), torch.randn(3, 33, 32).cuda(), torch.randn(3, 20, 32).cuda()
  mask = torch.nn.Transformer.generate_square_subsequent_mask(20).cuda()
  pad = (torch.arange(33)[None] >= torch.tensor([33, 13, 1])[:, None]).cuda() if padded else None
  res = []
  for net, dtype in ((ours, torch.float32), (plain, torch.float64)):
    y, z = (t.to(dtype).requires_grad_(True) for t in (x, memory))
    out = net(y, z, tgt_mask=mask.to(dtype), tgt_is_causal=True, memory_key_padding_mask=pad)
    res.append([out] + list(torch.autograd.grad((out * w.to(dtype)).sum(), [y, z, net.self_attn.in_proj_weight])))
  for a, b in zip(*res):                                       # fifteen products and norms of at most 60 rows or 48 terms each
    _norm_close(a, b, 2 * 15 * 60)


@pytest.mark.gpu
def test_torchs_encoder_layer_in_evaluation():
  """With dropout and without gradients, torch's fused path off: the module is called and its rows are torch's."""
  import copy
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  torch.manual_seed(6)
  ours = torch.nn.TransformerEncoderLayer(32, 4, 48, dropout=0.1, batch_first=True).cuda().eval()
  plain = copy.deepcopy(ours).double()
  assert tc.use_attention_kernels(ours) == 1
  x = torch.randn(3, 20, 32).cuda()
  pad = (torch.arange(20)[None] >= torch.tensor([20, 13, 1])[:, None]).cuda()
  calls = []
  ours.self_attn.register_forward_hook(lambda *a: calls.append(1))
  want = plain(x.double().requires_grad_(True), src_key_padding_mask=pad)     # (with gradients: torch's plain path)
  try:
    torch.backends.mha.set_fastpath_enabled(False)
    with torch.no_grad():
      got = ours(x, src_key_padding_mask=pad)
  finally:
    torch.backends.mha.set_fastpath_enabled(True)
  assert len(calls) == 1
  _norm_close(got.masked_fill(pad[..., None], 0.0), want.masked_fill(pad[..., None], 0.0), 2 * 6 * 60)


@pytest.mark.gpu
def test_floating_point_padding_mask():
  """0 and -inf: the bits of the bool mask, gradients too; any other value: NaN for its batch item and no other."""
  import torch
  from hsg_amd.models.embeddings import transformer_clusters as tc
  torch.manual_seed(4)
  for dtype in (torch.float32, torch.bfloat16):
    m = torch.nn.MultiheadAttention(32, 4, batch_first=True).cuda().to(dtype)
    tc.use_attention_kernels(m)
    x = torch.randn(3, 20, 32).cuda().to(dtype).requires_grad_(True)
    pad = (torch.arange(20)[None] >= torch.tensor([20, 13, 0])[:, None]).cuda()
    soft = torch.zeros(pad.shape, device='cuda', dtype=dtype).masked_fill(pad, -math.inf)
    res = []
    for mask in (pad, soft):
      out, _ = m(x, x, x, key_padding_mask=mask)
      res.append([out] + list(torch.autograd.grad(out.float().square().sum(), [x] + list(m.parameters()))))
    for a, b in zip(*res):
      assert torch.equal(a, b)
    for value in (-1.0, 1.0, torch.finfo(dtype).min, math.inf, math.nan):
      bad = soft.clone()
      bad[1, 2] = value
      out, _ = m(x, x, x, key_padding_mask=bad)
      assert bool(torch.isnan(out[1]).all()) and torch.equal(out[[0, 2]], res[0][0][[0, 2]])
