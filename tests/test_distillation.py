"""topk_distillation_loss (hsg_amd.utils.segsort.loss) against the definition in float64."""
import ctypes
import math

import pytest

EPS32 = 2.0 ** -24            # half a step of float32


# ---------------------------------------------------------------------------------------------------------------------
# arguments that are refused (no GPU needed)
def _args():
  import torch
  return dict(logits=torch.zeros(3, 10), teacher_logits=torch.zeros(3, 4), teacher_indices=torch.zeros(3, 4, dtype=torch.long))


@pytest.mark.parametrize('change, error', [
    (lambda a: a.update(logits=a['logits'].double()), TypeError),
    (lambda a: a.update(teacher_logits=a['teacher_logits'].long()), TypeError),
    (lambda a: a.update(teacher_indices=a['teacher_indices'].int()), TypeError),
    (lambda a: a.update(logits=a['logits'][:, :0]), ValueError),
    (lambda a: a.update(logits=a['logits'][:2]), ValueError),
    (lambda a: a.update(teacher_logits=a['teacher_logits'][:, :3]), ValueError),
    (lambda a: a.update(logits=a['logits'][None]), ValueError),
    (lambda a: a.update({n: a[n].repeat(1, 65) for n in ('teacher_logits', 'teacher_indices')}), ValueError),   # 260 entries
    (lambda a: a.update(teacher_logits=a['teacher_logits'].requires_grad_(True)), ValueError),
    (lambda a: a.update(temperature=0.0), ValueError),
    (lambda a: a.update(temperature=-1.0), ValueError),
    (lambda a: a.update(temperature=math.nan), ValueError),
    (lambda a: a.update(temperature=math.inf), ValueError),
    (lambda a: a.update(reduction='average'), ValueError),
])
def test_distillation_refuses(change, error):
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  a = _args()
  change(a)
  with pytest.raises(error):
    topk_distillation_loss(**a)


def test_distillation_refuses_cpu_tensors():
  from hsg_amd import _lib
  from hsg_amd.utils.segsort.loss import TopKDistillationLoss
  with pytest.raises(_lib.HsgkError):
    TopKDistillationLoss(2.0)(**_args())
  assert '2.00' in repr(TopKDistillationLoss(2.0))


def test_the_torch_op_refuses_tangents():
  """(before it looks at the device: no GPU needed)"""
  import torch
  import torch.autograd.forward_ad as fwd
  from hsg_amd import _torch_ops
  ops = _torch_ops.ops()
  if ops is None:
    pytest.skip('the torch binding is not built')
  for i in range(2):
    with fwd.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
      t = list(_args().values())
      t[i] = fwd.make_dual(t[i], torch.ones_like(t[i]))
      ops.topk_distill(*t, 1.0)


def test_the_torch_op_refuses_more_entries_than_32_bits_count():
  """(the op itself, not its Python entry: 2^32 + 4 entries a row were taken for 4)"""
  import torch
  from hsg_amd import _torch_ops
  ops = _torch_ops.ops()
  if ops is None:
    pytest.skip('the torch binding is not built')
  z, t, idx = _args().values()
  for k in (257, (1 << 32) + 4):
    with pytest.raises(RuntimeError, match='at most 256'):
      ops.topk_distill(z, t[:, :1].expand(3, k), idx[:, :1].expand(3, k), 1.0)
  with pytest.raises(RuntimeError, match='no CPU path'):
    ops.topk_distill(z, t, idx, 1.0)


def test_c_entry_refuses_bad_arguments():
  from hsg_amd import _lib
  L = _lib.lib()
  buf = ctypes.create_string_buffer(4096)
  p = (ctypes.addressof(buf) + 255) // 256 * 256
  good = [p, 0, 2, 8, 8, p, p, 4, 1.0, p, p]
  for i, value in ((0, None), (0, p + 2), (1, 3), (2, -1), (3, 0), (3, 1 << 31), (4, -8), (5, None), (6, None), (7, -1), (7, 257),
                   (8, 0.0), (8, math.nan), (9, None)):
    args = list(good)
    args[i] = value
    assert L.hsgk_topk_distill_fwd(*args, None) == -1, (i, value)
    assert L.hsgk_last_error()
  for i in (9, 10, 11):
    args = good[:9] + [p, p, p]
    args[i] = None
    assert L.hsgk_topk_distill_bwd(*args, None) == -1, i
  assert L.hsgk_topk_distill_fwd(None, 0, 0, 8, 8, None, None, 4, 1.0, None, None, None) == 0     # no rows
  assert L.hsgk_topk_distill_fwd(*good[:8], 1e-39, *good[9:], None) == -1                         # 1 / T is infinite


# ---------------------------------------------------------------------------------------------------------------------
def _exact(z, t, idx, T, g):
  """loss, dz and the bound of each in float64.

  With e = 2^-24: an exponent's argument x log2(e) / T is off by e (|x| / T + 1) twice over (the difference, the factor),
  exp2 by 2 e, a sum of n terms by e (n / 64 + 16) (64 lanes or more sum side by side), so q is off by a relative
  rq = e (4 span + n / 64 + 32), span = the spread of the row's arguments that matter (probabilities below 2^-60 count
  through their absolute size), and p alike; the loss adds terms of size T^2 p (|log p| + |log q|), each off by
  e (span + 32) and its factor; dz = g T (q - p): g T (q rq + p rp + 4 e |q - p|), and half a step of the type at the end."""
  import torch
  z, t = z.double(), t.double()
  n, V = z.shape
  k = t.shape[1]
  ok = (idx >= 0) & (idx < V) & (t != -math.inf)
  some = ok.any(1, keepdim=True) if k else torch.zeros((n, 1), dtype=torch.bool, device=z.device)
  tt = torch.where(ok, t / T, torch.full_like(t, -math.inf))
  tt = torch.where(some, tt, torch.zeros_like(tt))
  logp = torch.log_softmax(tt, 1) if k else tt
  p = torch.where(ok, logp.exp(), torch.zeros_like(tt))
  logq = torch.log_softmax(z / T, 1)
  at = logq.gather(1, idx.clamp(0, V - 1)) if k else tt
  loss = T * T * torch.where(p > 0, p * (logp - at), torch.zeros_like(p)).sum(1)
  q = logq.exp()
  hits = torch.zeros_like(z)
  if k:
    hits.scatter_add_(1, idx.clamp(0, V - 1), p)
  dz = g.double()[:, None] * T * (q - hits) * some
  e = EPS32
  top = (z / T).amax(1, keepdim=True)
  far = (top - z / T).clamp(max=60.0)
  rq = e * (4 * far + V / 64 + 32)
  rq_row = (rq * q).sum(1, keepdim=True)
  rp = e * (4 * 60.0 + k + 32)
  mag = torch.where(p > 0, p * (logp.abs() + at.abs() + (top - z / T).gather(1, idx.clamp(0, V - 1)).abs()), torch.zeros_like(p)).sum(1) if k \
      else torch.zeros_like(loss)
  e_loss = T * T * ((rp + 8 * e) * mag + torch.where(some[:, 0], (rq_row[:, 0] + rp + 40 * e) * 1.0, torch.zeros_like(loss)))
  e_dz = g.double().abs()[:, None] * T * (q * (rq + rq_row) + hits * rp + 4 * e * (q - hits).abs() + 2.0 ** -100) * some
  return loss, dz, e_loss * 1.01, e_dz * 1.01


def _make(seed, dtype, n, V, k, spread=3.0):
  import torch
  gen = torch.Generator().manual_seed(seed)
  z = (torch.randn((n, V), generator=gen) * spread).to(dtype).cuda()
  t = (torch.randn((n, k), generator=gen) * spread).cuda()
  idx = torch.randint(0, V, (n, k), generator=gen).cuda()          # the same index twice now and then
  g = torch.randn((n,), generator=gen).cuda()
  return z, t, idx, g


def _run(z, t, idx, g, T=1.0):
  import torch
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  leaf = z.detach().requires_grad_(True)
  loss = topk_distillation_loss(leaf, t, idx, temperature=T, reduction='none')
  (dz,) = torch.autograd.grad(loss, leaf, g)
  with torch.no_grad():
    again = topk_distillation_loss(z, t, idx, temperature=T, reduction='none')
    assert torch.equal(again.view(torch.int32), loss.detach().view(torch.int32))
  assert loss.dtype == torch.float32 and dz.dtype == z.dtype
  torch.cuda.synchronize()
  return loss.detach(), dz


def _check(z, t, idx, g, T=1.0):
  import torch
  loss, dz = _run(z, t, idx, g, T)
  w_loss, w_dz, e_loss, e_dz = _exact(z, t, idx, T, g)
  u = torch.finfo(z.dtype).eps / 2
  tiny = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}[z.dtype]
  assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(dz).all())
  off = (loss.double() - w_loss).abs() - e_loss
  assert float(off.max()) <= 0, float(off.max())
  off = (dz.double() - w_dz).abs() - (e_dz + u * w_dz.abs() + tiny)
  assert float(off.max()) <= 0, float(off.max())


TYPES = ['float32', 'bfloat16', 'float16']


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('n, V, k, T', [
    (1, 1, 1, 1.0), (1, 2, 1, 1.0), (5, 3, 7, 2.0), (3, 64, 8, 1.0), (7, 65, 64, 0.5), (130, 257, 20, 1.0), (9, 2047, 32, 2.0),
    (9, 2048, 32, 2.0), (9, 2049, 1, 1.0), (6, 4099, 256, 1.0), (3, 40001, 65, 1.0), (2, 17, 256, 1.0), (4, 100, 0, 1.0)])
def test_loss_and_gradient(name, n, V, k, T):
  import torch
  _check(*_make(3, getattr(torch, name), n, V, k), T=T)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [100, 3001])
def test_rows_without_entries_and_entries_that_do_not_count(V):
  """Entries outside [0, V), unfilled slots (-inf), rows without any: zeros, whatever the row's logits are."""
  import torch
  z, t, idx, g = _make(4, torch.float32, 40, V, 9)
  idx[0] = -1
  t[1] = -math.inf
  idx[2, :5], idx[2, 5:] = V, 1 << 40
  idx[3, 1:] = -7
  t[4, ::2] = -math.inf
  idx[5] = 6                                                       # one class in every slot
  idx[6, :4] = torch.tensor([2, 2, 3, 2])
  _check(z, t, idx, g)
  loss, dz = _run(z, t, idx, g)
  assert not bool(loss[:3].any()) and not bool(dz[:3].any())
  z[0], z[1, 3] = math.nan, math.inf                               # a row without entries passes nothing on
  loss, dz = _run(z, t, idx, g)
  assert not bool(loss[:3].any()) and not bool(dz[:3].any()) and bool(torch.isfinite(dz).all())


@pytest.mark.gpu
def test_masked_classes_and_non_finite_values():
  """Classes that the student masks with -inf or the type's lowest value have q = 0; NaN stays NaN in its row only."""
  import torch
  for V in (120, 2600):
    z, t, idx, g = _make(5, torch.float32, 6, V, 4)
    hide = torch.arange(V).cuda() % 3 == 0
    idx = torch.where(idx % 3 == 0, idx + 1, idx).clamp(max=V - 1)
    idx = torch.where(idx % 3 == 0, idx - 1, idx)
    for low in (-math.inf, torch.finfo(torch.float32).min):
      zz = z.masked_fill(hide, low)
      loss, dz = _run(zz, t, idx, g)
      keep = torch.arange(V).cuda()[~hide]
      pos = torch.full((V,), -1, dtype=torch.long, device='cuda')
      pos[keep] = torch.arange(keep.numel(), device='cuda')
      w_loss, w_dz, e_loss, e_dz = _exact(z[:, keep], t, pos[idx], 1.0, g)
      assert not bool(dz[:, hide].any())
      assert bool(((loss.double() - w_loss).abs() <= e_loss).all())
      assert bool(((dz[:, keep].double() - w_dz).abs() <= e_dz + EPS32 * w_dz.abs()).all())
    z[2, 5] = math.nan
    loss, dz = _run(z, t, idx, g)
    bad = torch.arange(6).cuda() == 2
    assert bool(torch.isnan(loss[bad]).all()) and bool(torch.isnan(dz[bad]).all())
    assert bool(torch.isfinite(loss[~bad]).all()) and bool(torch.isfinite(dz[~bad]).all())
    one = z[3:4].masked_fill(torch.arange(V).cuda() == idx[3, 0], -math.inf)   # the student excludes what the teacher names
    loss, _ = _run(one, t[3:4], idx[3:4], g[3:4])
    assert float(loss[0]) == math.inf


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('V', [1000, 5200, 100003])
@pytest.mark.parametrize('offset', [100.0, 1000.0, -10000.0])
def test_an_offset_of_the_whole_row_costs_nothing(name, V, offset):
  """Softmax does not see what all logits of a row have in common: the bounds, which count the row's spread and not its
  size, hold as they do around zero.  (_make's logits are rounded to the type after the offset is added.)"""
  import torch
  z, t, idx, g = _make(41, torch.float32, 9, V, 32)
  _check((z + offset).to(getattr(torch, name)), t, idx, g, T=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('more', [-1, 0, 1])
@pytest.mark.parametrize('lead', [0, 1, 3])
def test_longest_rows_that_go_through_lds(name, more, lead):
  """One class either side of 10 KB, where a workgroup takes over from a wave, with the most entries, row starts that are
  aligned or not, and a last workgroup that is not full."""
  import torch
  dtype = getattr(torch, name)
  V = 10240 // torch.empty((), dtype=dtype).element_size() + more
  z, t, idx, g = _make(44, dtype, 7, V, 256)
  idx[:, :4] = torch.tensor([0, V - 1, 0, V - 1])                    # both ends of the row, twice
  wide = torch.full((7, V + 5), math.nan, dtype=dtype, device='cuda')
  view = wide[:, lead:lead + V]
  view.copy_(z)
  _check(view, t, idx, g, T=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('V', [200, 1000, 6000])
@pytest.mark.parametrize('offset', [0.0, 300.0, 1000.0, -3000.0])
def test_loss_of_one_entry_next_to_an_offset(name, V, offset):
  """One entry: p = 1, loss = T^2 (log L - (z_i - top) / T), so that the row's log L stands alone.  With e = 2^-24 and far the
  row's spread over T: an exponent's argument (difference, log2(e) / T, product) is off by 3 e far, exp2 by 2 e, a sum of V terms
  by e (V / 64 + 16); the logarithm, the two divisions and the difference by 4 e (log V + far) + 8 e."""
  import torch
  z, t, idx, g = _make(43, torch.float32, 64, V, 1)
  z, T = (z + offset).to(getattr(torch, name)), 0.5
  loss, _ = _run(z, t, idx, g, T)
  want, _, _, _ = _exact(z, t, idx, T, g)
  x = z.double() / T
  far = x.amax(1) - x.amin(1)
  bound = T * T * EPS32 * (3 * far + V / 64 + 18 + 4 * (math.log(V) + far) + 8)
  off = (loss.double() - want).abs() - bound
  assert float(off.max()) <= 0, float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('V', [40, 2600, 9000])
def test_rows_at_the_types_lowest_value(name, V):
  """Every class of a row masked with the lowest value, or the highest: uniform, as for any other common value."""
  import torch
  dtype = getattr(torch, name)
  z, t, idx, g = _make(42, dtype, 6, V, 4)
  z[1], z[4] = torch.finfo(dtype).min, torch.finfo(dtype).max
  for T in (1.0, 0.25):
    _check(z, t, idx, g, T=T)


@pytest.mark.gpu
@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('V', [99, 2500])
def test_strides_and_alignment(name, V):
  """Rows of a wider buffer, misaligned starts, expanded rows, a transposed view, leading dimensions: the same bits."""
  import torch
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  z, t, idx, g = _make(6, getattr(torch, name), 12, V, 8)
  want = _run(z, t, idx, g)
  for lead in range(4):
    wide = torch.full((12, V + 9), math.nan, dtype=z.dtype, device='cuda')
    view = wide[:, lead:lead + V]
    view.copy_(z)
    got = _run(view, t, idx, g)
    for a, b in zip(got, want):
      # (pieces start elsewhere, so the sums of a row may differ in their last bits)
      assert float((a.double() - b.double()).abs().max()) <= 4e-6 * float(b.abs().max()) + \
          2 * torch.finfo(a.dtype).eps * float(b.abs().max())
    _check(view, t, idx, g)
  got = _run(z.t().contiguous().t(), t, idx, g)
  for a, b in zip(got, want):
    assert torch.equal(a, b)
  one = z[:1].expand(12, V)
  for a, b in zip(_run(one, t, idx, g), _run(one.contiguous(), t, idx, g)):
    assert a.shape == b.shape and float((a.double() - b.double()).abs().max()) <= 8 * torch.finfo(a.dtype).eps * float(b.abs().max())
  leaf = z.view(3, 4, V).detach().requires_grad_(True)
  loss = topk_distillation_loss(leaf, t.view(3, 4, 8), idx.view(3, 4, 8), reduction='none')
  assert loss.shape == (3, 4) and torch.equal(loss.view(-1), want[0])
  (dz,) = torch.autograd.grad(loss, leaf, g.view(3, 4))
  assert torch.equal(dz.view(12, V), want[1])


@pytest.mark.gpu
def test_reductions_and_teacher_types():
  import torch
  from hsg_amd.utils.segsort.loss import TopKDistillationLoss, topk_distillation_loss
  z, t, idx, g = _make(7, torch.float32, 33, 70, 5)
  rows = topk_distillation_loss(z, t, idx, 2.0, 'none')
  assert torch.equal(topk_distillation_loss(z, t, idx, 2.0), rows.mean())
  assert torch.equal(TopKDistillationLoss(2.0, reduction='sum')(z, t, idx), rows.sum())
  half = t.half()
  assert torch.equal(topk_distillation_loss(z, half, idx, 2.0, 'none'), topk_distillation_loss(z, half.float(), idx, 2.0, 'none'))
  assert topk_distillation_loss(z[:0], t[:0], idx[:0], reduction='none').shape == (0,)


@pytest.mark.gpu
def test_gradient_against_differences():
  import torch
  z, t, idx, g = _make(8, torch.float32, 6, 50, 6)
  _, dz = _run(z, t, idx, g)
  d = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).cuda()
  h = 1e-4
  up, _, _, _ = _exact(z.double() + h * d, t, idx, 1.0, g)
  down, _, _, _ = _exact(z.double() - h * d, t, idx, 1.0, g)
  slope = float(((up - down) * g.double()).sum()) / (2 * h)
  inner = float((dz.double() * d.double()).sum())
  assert abs(slope - inner) <= 1e-5 * (1 + float(dz.double().norm()) * float(d.double().norm()))


@pytest.mark.gpu
def test_more_rows_than_one_launch_takes():
  import torch
  _check(*_make(23, torch.float16, (1 << 23) + 3, 6, 2))


@pytest.mark.gpu
@pytest.mark.parametrize('binding', ['torch', 'ctypes'])
def test_gradient_cannot_be_differentiated(binding, monkeypatch):
  import torch
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  if binding == 'ctypes':
    monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  z, t, idx, _ = _make(3, torch.float32, 5, 40, 3)
  z.requires_grad_(True)
  (want,) = torch.autograd.grad(topk_distillation_loss(z, t, idx), z)
  (got,) = torch.autograd.grad(topk_distillation_loss(z, t, idx), z, create_graph=True)
  assert torch.equal(got, want)
  with pytest.raises(RuntimeError, match='differentiable once'):
    torch.autograd.grad(got.sum(), z)


@pytest.mark.gpu
@pytest.mark.parametrize('binding', ['torch', 'ctypes'])
def test_tangents_are_refused(binding, monkeypatch):
  """Forward-mode differentiation raises under both bindings, of the logits and of the teacher."""
  import torch
  import torch.autograd.forward_ad as fwd
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  if binding == 'ctypes':
    monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  z, t, idx, _ = _make(3, torch.float32, 5, 40, 3)
  for grad in (False, True):
    for which in (0, 1):
      with fwd.dual_level():
        u = [z.detach().requires_grad_(grad), t.detach()]
        u[which] = fwd.make_dual(u[which], torch.ones_like(u[which]))
        for shape in ((5, -1), (1, 5, -1)):
          v = [x.view(*shape) for x in u] + [idx.view(*shape)]
          with pytest.raises(RuntimeError):
            topk_distillation_loss(*v)
          with torch.no_grad(), pytest.raises(RuntimeError):
            topk_distillation_loss(*v)
  with fwd.dual_level():
    leaf = z.detach().requires_grad_(True)
    loss = topk_distillation_loss(leaf, t, idx, reduction='none')                # (without a tangent it runs)
    one = torch.ones_like(loss)
    assert torch.autograd.grad(loss, leaf, one, retain_graph=True)[0].shape == z.shape
    with pytest.raises(RuntimeError, match='forward-mode'):                      # a tangent of the incoming gradient
      torch.autograd.grad(loss, leaf, fwd.make_dual(one, one))


@pytest.mark.gpu
def test_bindings_streams_and_graphs(monkeypatch):
  import torch
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  z, t, idx, g = _make(9, torch.bfloat16, 40, 2500, 16)
  want = _run(z, t, idx, g)
  with torch.cuda.stream(torch.cuda.Stream()):
    got = _run(z, t, idx, g)
  assert all(torch.equal(a, b) for a, b in zip(got, want))
  leaf = z.detach().clone().requires_grad_(True)

  def step():
    loss = topk_distillation_loss(leaf, t, idx, reduction='none')
    return [loss] + list(torch.autograd.grad(loss, leaf, g))

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    res = step()
  for n in range(3):
    z2 = _make(50 + n, torch.bfloat16, 40, 2500, 16)[0]
    with torch.no_grad():
      leaf.copy_(z2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(res, _run(z2, t, idx, g))), n
  monkeypatch.setenv('HSGK_BINDING', 'ctypes')
  got = _run(z, t, idx, g)
  assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_retrieval_attention_and_distillation_together():
  """One training step as it is used: tokens attend to each other, their rows are scored against prototypes, a teacher's
  retrieved prototypes (top_k_indices, with a group that holds fewer than k) supervise them; gradients against float64."""
  import torch
  from hsg_amd.models.embeddings.transformer_clusters import attention
  from hsg_amd.utils.segsort.eval import top_k_indices
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  gen = torch.Generator().manual_seed(11)
  B, n, H, D, P, k, kappa = 2, 40, 2, 16, 30, 6, 8.0
  x, teacher = (torch.randn((B, n, H * D), generator=gen).cuda() for _ in range(2))
  protos = torch.nn.functional.normalize(torch.randn((P, H * D), generator=gen), dim=1).cuda()
  groups, pgroups = torch.arange(B).repeat_interleave(n).cuda(), (torch.arange(P) >= 3).long().cuda()   # 3 and 27 prototypes
  idx, val = top_k_indices(teacher.view(-1, H * D), protos, k, groups, pgroups)
  mask = (torch.arange(n)[None] >= torch.tensor([n, 25])[:, None]).cuda()

  def step(x, protos, plain):
    heads = x.view(B, n, H, D)
    if plain:
      q = heads.transpose(1, 2)
      s = (q @ q.transpose(-1, -2)) * D ** -0.5
      y = (torch.softmax(s.masked_fill(mask[:, None, None], -math.inf), -1) @ q).transpose(1, 2)
    else:
      y = attention(heads, heads, heads, key_padding_mask=mask)
    z = kappa * (y.reshape(-1, H * D) @ protos.t())
    if not plain:
      return topk_distillation_loss(z, val, idx, 2.0, 'sum')
    t = torch.where(val == -math.inf, torch.full_like(val, -math.inf), val).double() / 2.0
    logp = torch.log_softmax(t, 1)
    logq = torch.log_softmax(z / 2.0, 1).gather(1, idx)
    p = logp.exp()
    return 4.0 * torch.where(p > 0, p * (logp.clamp_min(-1e30) - logq), torch.zeros_like(p)).sum()

  a, b = x.requires_grad_(True), protos.requires_grad_(True)
  loss = step(a, b, False)
  got = torch.autograd.grad(loss, (a, b))
  a64, b64 = x.detach().double().requires_grad_(True), protos.detach().double().requires_grad_(True)
  want_loss = step(a64, b64, True)
  want = torch.autograd.grad(want_loss, (a64, b64))
  # products of at most 40 terms, a softmax each way, kappa 8: 2^-24 * 500 of the norm
  assert abs(float(loss.detach()) - float(want_loss.detach())) <= 3e-5 * abs(float(want_loss.detach()))
  for u, v in zip(got, want):
    assert float((u.double() - v).norm()) <= 3e-5 * float(v.norm())
