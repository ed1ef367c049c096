"""What is measured of the attention and teacher-distillation operators: the cases, their inputs, the plain forms and the
values from the definition in 64 bits.

Sizes: the clustering transformer (eight queries and 256 padded segment tokens an image, 256 channels in eight heads of
32), ViT-S/16 tokens (384 channels in six heads of 64, one class token) of the 224, 448 and 768 pixel crops that bench.py
runs, pixel rows of the training resolutions (28 x 28 and 56 x 56 embeddings) against tables of prototypes, and generic
long ones."""
import math

import torch

own = False

TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


# ---- the cases ------------------------------------------------------------------------------------------------------
def _attention(name, dtype, B, L, S, H, G, D, pad, causal, backward):
  return {'name': name, 'op': 'attention', 'dtype': dtype, 'B': B, 'L': L, 'S': S, 'H': H, 'G': G, 'D': D, 'pad': pad,
          'causal': causal, 'backward': backward}


def _distill(name, dtype, N, V, k, T, backward):
  return {'name': name, 'op': 'distill', 'dtype': dtype, 'N': N, 'V': V, 'k': k, 'T': T, 'backward': backward}


def listed():
  return [
      # the decoder of the clustering transformer: eight learned queries on the padded segments of 24 images
      _attention('queries_on_segments', 'float32', 24, 8, 256, 8, 8, 32, True, False, False),
      # its encoder, trained: the segments of an image attend to each other
      _attention('segments_train', 'float32', 24, 256, 256, 8, 8, 32, True, False, True),
      # ragged lengths and a head width that fills no tile, trained
      _attention('ragged_train', 'float32', 7, 131, 203, 4, 2, 36, True, False, True),
      # ViT-S/16 tokens of 224 x 224 crops, trained in bfloat16
      _attention('vit224_train', 'bfloat16', 32, 197, 197, 6, 6, 64, False, False, True),
      # the same of 448 x 448 crops, inference in float16
      _attention('vit448', 'float16', 16, 785, 785, 6, 6, 64, False, False, False),
      # the same of 768 x 768 crops, trained
      _attention('vit768_train', 'bfloat16', 4, 2305, 2305, 6, 6, 64, False, False, True),
      # a long causal sequence with shared key heads, trained
      _attention('long_causal_train', 'bfloat16', 1, 8192, 8192, 16, 4, 128, False, True, True),
      # one new token over long keys and values that four heads share
      _attention('one_token', 'bfloat16', 2, 1, 32768, 16, 4, 128, True, False, False),
      # one 28 x 28 map against the 64 segments of its image: the smallest call
      _distill('one_map', 'float32', 784, 64, 8, 1.0, False),
      # the pixels of 48 such maps against a table of prototypes, trained
      _distill('pixels_train', 'float32', 37632, 2048, 20, 1.0, True),
      # 16 maps of 56 x 56 against an odd table, trained in bfloat16
      _distill('pixels_odd_train', 'bfloat16', 50176, 4099, 32, 2.0, True),
      # few rows, a memory bank of prototypes
      _distill('bank_train', 'float16', 1031, 100003, 64, 0.5, True),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  if rng.random() < 0.4:
    V = _log(rng, 32, 100003)
    N = _log(rng, 256, max(257, min(60000, 200000000 // V)))
    return _distill('', rng.choice(['float32', 'bfloat16', 'float16']), N, V, rng.choice([1, 4, 8, 20, 32, 64]),
                    rng.choice([0.5, 1.0, 2.0]), rng.random() < 0.6) | {'name': 'drawn'}
  kind = rng.choice(['self', 'self', 'cross', 'single', 'causal'])
  dtype = rng.choice(['float32', 'bfloat16', 'float16'])
  D = rng.choice([24, 32, 36, 40, 48, 64, 64, 72, 80, 96, 128])
  G = rng.choice([1, 2, 3, 4, 6, 8])
  H = G * rng.choice([1, 1, 2, 4])
  if kind == 'single':
    L, S = rng.randint(1, 4), _log(rng, 512, 40000)
  elif kind == 'cross':
    L, S = _log(rng, 4, 128), _log(rng, 32, 4096)
  else:
    S = L = _log(rng, 16, 2400)
    if kind == 'causal' and rng.random() < 0.5:
      S = L + rng.randint(1, 300)
  backward = kind != 'single' and rng.random() < 0.6
  # no more than a sixteenth of the scores of the longest case in 32 bits, whose products are the slowest
  B = max(1, min(32, 64000000 // (H * L * S)))
  B = rng.randint(max(1, B // 4), B)
  return _attention('drawn', dtype, B, L, S, H, G, D, kind != 'causal' and rng.random() < 0.6, kind == 'causal', backward)


def _lengths(case):
  """Keys of every batch item: spread evenly from all down to a quarter; of eight and more items the last has none."""
  B, S = case['B'], case['S']
  if not case['pad']:
    return [S] * B
  got = [max(1, S - (b * (3 * S // 4)) // max(B - 1, 1)) for b in range(B)]
  if B >= 8:
    got[-1] = 0
  return got


def work(case):
  size = torch.empty((), dtype=TYPES[case['dtype']]).element_size()
  if case['op'] == 'distill':
    N, V, k = case['N'], case['V'], case['k']
    rows = N * V * size
    return {'bytes': rows + N * k * 12 + 4 * N + (rows + 4 * N if case['backward'] else 0),
            'flops': N * V * (8.0 if case['backward'] else 4.0)}
  B, L, S, H, G, D = (case[n] for n in 'BLSHGD')
  keys = sum(_lengths(case))
  if case['causal']:
    seen = sum(max(0, min(S, i + 1 + S - L)) for i in range(L))
    pairs = B * seen
  else:
    pairs = L * keys
  rows_q, rows_k = B * L * H * D, keys * G * D
  moved = 2 * rows_q + 2 * rows_k                      # q and out, k and v
  if case['backward']:
    moved += 2 * rows_q + 2 * B * S * G * D            # the incoming gradient and dq, dk and dv
  return {'bytes': moved * size + (B * S if case['pad'] else 0),
          'flops': (14.0 if case['backward'] else 4.0) * pairs * H * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
  g = torch.Generator(device='cuda').manual_seed(seed)
  dtype = TYPES[case['dtype']]

  def normal(*shape):
    return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)

  state = {'case': case}
  if case['op'] == 'distill':
    N, V, k = case['N'], case['V'], min(case['k'], case['V'])
    z = normal(N, V).mul_(2.5)
    # a teacher that agrees with the student in part; the last rows' images hold fewer prototypes than k
    # (those slots are index 0 with value -inf), the very last rows are pixels without any
    t, at = torch.topk(z + 2.0 * normal(N, V), k, dim=1)
    few, none = N - N // 16, N - N // 64
    t[few:, (k + 1) // 2:] = -math.inf
    at[few:, (k + 1) // 2:] = 0
    t[none:] = -math.inf
    at[none:] = 0
    state.update(z=z.to(dtype), t=t.contiguous(), at=at.contiguous())
    if case['backward']:
      # a mean over the rows with weights; training in float16 scales its loss
      state['g'] = (torch.rand((N,), generator=g, device='cuda') + 0.5) * ((65536.0 if dtype == torch.float16 else 1.0) / N)
      state['z'].requires_grad_(True)
    return state
  B, L, S, H, G, D = (case[n] for n in 'BLSHGD')
  for name, shape in (('q', (B, L, H, D)), ('k', (B, S, G, D)), ('v', (B, S, G, D))):
    state[name] = normal(*shape).to(dtype)
  state['mask'] = None
  if case['pad']:
    order = torch.randperm(B, generator=g, device='cuda')
    n = torch.tensor(_lengths(case), device='cuda')[order]
    state['mask'] = torch.arange(S, device='cuda') >= n[:, None]
  if case['backward']:
    state['g'] = normal(B, L, H, D).to(dtype)
    for name in 'qkv':
      state[name].requires_grad_(True)
  return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
  case = state['case']
  if case['op'] == 'distill':
    return _run_distill(case, state) if own else _plain_distill(case, state)
  return _run_attention(case, state) if own else _plain_attention(case, state)


def _run_attention(case, s):
  from hsg_amd.models.embeddings.transformer_clusters import attention
  out = attention(s['q'], s['k'], s['v'], key_padding_mask=s['mask'], is_causal=case['causal'])
  if not case['backward']:
    return {'out': out}
  dq, dk, dv = torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['g'])
  return {'out': out, 'dq': dq, 'dk': dk, 'dv': dv}


def _run_distill(case, s):
  from hsg_amd.utils.segsort.loss import topk_distillation_loss
  loss = topk_distillation_loss(s['z'], s['t'], s['at'], temperature=case['T'], reduction='none')
  if not case['backward']:
    return {'loss': loss}
  (dz,) = torch.autograd.grad(loss, (s['z'],), s['g'])
  return {'loss': loss, 'dz': dz}


def _heads(x, G):
  """[B, n, H, D] -> [B, G, H / G * n, D] in 32 bits: the queries of the heads that share a key head lie together."""
  B, n, H, D = x.shape
  return x.float().view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * n, D)


def _rows(x, n):
  """The reverse of _heads."""
  B, G, m, D = x.shape
  return x.view(B, G, m // n, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, G * (m // n), D)


def _hidden(case, mask, device):
  """[B or 1, 1, H / G * L or 1, S] true where a query does not see a key, or None."""
  L, S = case['L'], case['S']
  hidden = None
  if mask is not None:
    hidden = mask[:, None, None, :]
  if case['causal']:
    i, j = torch.arange(L, device=device)[:, None], torch.arange(S, device=device)[None, :]
    ahead = (j > i + (S - L)).repeat(case['H'] // case['G'], 1)[None, None]
    hidden = ahead if hidden is None else hidden | ahead
  return hidden


def _plain_attention(case, s):
  G, D, dtype = case['G'], case['D'], s['q'].dtype
  q, k, v = (_heads(s[n].detach(), G) for n in 'qkv')
  p = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5)
  hidden = _hidden(case, s['mask'], p.device)
  if hidden is not None:
    p.masked_fill_(hidden, -math.inf)
  top = p.amax(dim=-1, keepdim=True)
  p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
  total = p.sum(dim=-1, keepdim=True)
  p.div_(torch.where(total == 0, torch.ones_like(total), total))
  o = torch.matmul(p, v)
  out = _rows(o, case['L']).to(dtype)
  if not case['backward']:
    return {'out': out}
  g = _heads(s['g'], G)
  dv = torch.matmul(p.transpose(-1, -2), g)
  dp = torch.matmul(g, v.transpose(-1, -2))
  ds = dp.sub_((g * o).sum(dim=-1, keepdim=True)).mul_(p).mul_(D ** -0.5)
  dq = torch.matmul(ds, k)
  dk = torch.matmul(ds.transpose(-1, -2), q)
  return {'out': out, 'dq': _rows(dq, case['L']).to(dtype), 'dk': _rows(dk, case['S']).to(dtype),
          'dv': _rows(dv, case['S']).to(dtype)}


def _plain_distill(case, s):
  T, dtype = case['T'], s['z'].dtype
  z = s['z'].detach().float() / T
  z = z - z.amax(dim=1, keepdim=True)
  e = z.exp()
  total = e.sum(dim=1, keepdim=True)
  t, at = s['t'] / T, s['at']
  top = t.amax(dim=1, keepdim=True)
  p = (t - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
  mass = p.sum(dim=1, keepdim=True)
  p = p / torch.where(mass == 0, torch.ones_like(mass), mass)
  logp = torch.where(p > 0, p, torch.ones_like(p)).log()
  logq = z.gather(1, at) - total.log()
  loss = T * T * (p * (logp - logq)).sum(dim=1)
  if not case['backward']:
    return {'loss': loss}
  w = s['g'][:, None] * T
  dz = e.mul_(torch.where(mass > 0, w / total, torch.zeros_like(total)))
  dz.scatter_add_(1, at, -w * p)
  return {'loss': loss, 'dz': dz.to(dtype)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
  s = prepare(case, seed)
  return _exact_distill(case, s) if case['op'] == 'distill' else _exact_attention(case, s)


def _exact_attention(case, s):
  """One batch item at a time by torch's own differentiation in float64."""
  B, L, S, H, G, D = (case[n] for n in 'BLSHGD')
  got = {'out': []} if not case['backward'] else {'out': [], 'dq': [], 'dk': [], 'dv': []}
  for b in range(B):
    seen = torch.ones((L, S), dtype=torch.bool, device='cuda')
    if case['causal']:
      seen = torch.tril(seen, diagonal=S - L)
    if s['mask'] is not None:
      seen = seen & ~s['mask'][b][None, :]
    some = seen.any(dim=1, keepdim=True)
    parts = {name: [] for name in got}
    for h in range(G):                                 # one key head and the heads that share it
      own_heads = slice(h * (H // G), (h + 1) * (H // G))
      q = s['q'].detach()[b, :, own_heads].double().transpose(0, 1).contiguous().requires_grad_(case['backward'])
      k = s['k'].detach()[b, :, h].double().requires_grad_(case['backward'])
      v = s['v'].detach()[b, :, h].double().requires_grad_(case['backward'])
      score = (q.reshape(-1, D) @ k.t()).view(H // G, L, S) / math.sqrt(D)
      # a row that sees nothing is computed with every key and replaced by zeros afterwards
      score = score.masked_fill(~(seen | ~some), -math.inf)
      o = (torch.softmax(score, dim=-1).view(-1, S) @ v).view(H // G, L, D)
      o = torch.where(some, o, torch.zeros_like(o))
      parts['out'].append(o.detach().transpose(0, 1))
      if case['backward']:
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), s['g'][b, :, own_heads].double().transpose(0, 1))
        parts['dq'].append(dq.transpose(0, 1))
        parts['dk'].append(dk[:, None])
        parts['dv'].append(dv[:, None])
    for name in got:
      got[name].append(torch.cat(parts[name], dim=1))
  return {name: torch.stack(rows) for name, rows in got.items()}


def _exact_distill(case, s):
  T = case['T']
  z = s['z'].detach().double().requires_grad_(case['backward'])
  t = s['t'].double()
  some = (t > -math.inf).any(dim=1)
  logp = torch.log_softmax(torch.where(some[:, None], t, torch.zeros_like(t)) / T, dim=1)
  p = logp.exp()
  logq = torch.log_softmax(z / T, dim=1).gather(1, s['at'])
  each = torch.where(p > 0, p * (logp.clamp_min(-1e300) - logq), torch.zeros_like(p))
  loss = torch.where(some, T * T * each.sum(dim=1), torch.zeros_like(some, dtype=torch.float64))
  if not case['backward']:
    return {'loss': loss.detach()}
  (dz,) = torch.autograd.grad(loss, (z,), s['g'].double())
  return {'loss': loss.detach(), 'dz': dz}
