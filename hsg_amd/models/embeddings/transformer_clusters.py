"""`TransformerClustering.forward` of the reference
(hsg/models/embeddings/transformer_clusters.py:60-114) with its tail -- logits, the
`num_clusters` queries of largest activation, the three gathers -- on libhsgk
(`hsgk_cluster_topk`).  The transformer stack and the two FC + BN heads are the module's own
(stock PyTorch-ROCm); `forward` below is bound onto the reference class by
`hsg_amd.patch_reference()` or inherited through `TransformerClusteringMixin`.

`attention` is the operator between the projections of the stack's attention modules
(hsg/models/heads/transformer.py builds them from torch.nn.MultiheadAttention), forward and backward on libhsgk;
`use_attention_kernels(module)` switches the attention modules of a built stack over to it.
"""
import math

import torch
import torch.nn.functional as F

from hsg_amd import ops
from hsg_amd.models.embeddings import hierarchy

MAX_HEAD_WIDTH = 128    # include/hsgk.h HSGK_ATTENTION_MAX_WIDTH


def attention(query, key, value, key_padding_mask=None, is_causal=False, scale=None):
  """softmax(scale * query key^T) value per head, differentiable (once, in reverse mode) in the three.

  query [B, L, H, D], key and value [B, S, G, D] with H a multiple of G (query head h uses key head h // (H // G)), all
  float32, bfloat16 or float16 with D <= 128, on one ROCm device; any strides (a last dimension that is not contiguous
  is copied).  key_padding_mask [B, S] bool: True = not a key, as in torch.nn.MultiheadAttention; such keys and values
  may hold anything, NaN included.  is_causal: query i sees the keys j <= i + S - L (the last query sees every key).
  scale: positive, 1 / sqrt(D) when None.  Returns [B, L, H, D], contiguous, of the inputs' type.

  A query that sees no key has output 0 and passes no gradient (torch's softmax gives NaN there).  Sums and statistics are
  float32; between 16-bit inputs a probability, and its gradient, is rounded to their type where it enters the second
  product, so that an output is off by about 1.4 roundings and not one.  A score is float32 too: a probability's relative
  error is 2^-23 of the row's largest score or so, and scores past 2^22 leave float16's range.  Causality hides what is
  finite: a NaN or an infinity in a row that some query of the batch item sees may reach queries next to it that do not.
  The backward pass recomputes the probabilities, uses no atomics and repeats bit for bit.
  Under graph capture take gradients with torch.autograd.grad, which adds nothing to leaves that another graph holds.
  """
  for name, t in (('query', query), ('key', key), ('value', value)):
    if t.dim() != 4:
      raise ValueError('%s must be [batch, length, heads, width] (got %d dimensions)' % (name, t.dim()))
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) or t.dtype is not query.dtype:
      raise TypeError('query, key and value must share one type of float32, bfloat16, float16 (%s is %s)' % (name, t.dtype))
    if t.device != query.device:
      raise ValueError('query, key and value must be on one device')
  B, _, H, D = query.shape
  if key.shape != value.shape:
    raise ValueError('key and value must have the same shape: %s and %s' % (tuple(key.shape), tuple(value.shape)))
  if key.shape[0] != B or key.shape[3] != D:
    raise ValueError('query and key disagree on the batch or the head width: %s and %s'
                     % (tuple(query.shape), tuple(key.shape)))
  G = key.shape[2]
  if G < 1 or H < 1 or H % G:
    raise ValueError('the query heads (%d) must be a multiple of the key heads (%d)' % (H, G))
  if not 1 <= D <= MAX_HEAD_WIDTH:
    raise ValueError('the head width must be 1 .. %d (got %d)' % (MAX_HEAD_WIDTH, D))
  if key_padding_mask is not None:
    if key_padding_mask.dtype is not torch.bool:
      raise TypeError('key_padding_mask must be bool (got %s)' % key_padding_mask.dtype)
    if tuple(key_padding_mask.shape) != (B, key.shape[1]) or key_padding_mask.device != query.device:
      raise ValueError('key_padding_mask must be [%d, %d] on the device of the keys' % (B, key.shape[1]))
  scale = D ** -0.5 if scale is None else float(scale)
  if not (scale > 0.0 and math.isfinite(scale)):
    raise ValueError('scale must be positive and finite (got %r)' % scale)
  ops.require_gpu(query, 'query')
  return ops.attention(query, key, value, key_padding_mask, bool(is_causal), scale)


class MultiheadAttention(torch.nn.MultiheadAttention):
  """torch.nn.MultiheadAttention (same parameters, state_dict and call) whose softmax(q k^T) v runs in libhsgk.  Returns
  (output, None): the probabilities are never stored, so there are no weights to return (and need_weights is False unless
  it is asked for).  A call that needs what the kernels do not offer raises: need_weights=True, any other attn_mask than
  the causal one, dropout in training, bias_k / bias_v, add_zero_attn, unbatched inputs.

  attn_mask [length, length] with is_causal=True, over as many queries as keys, is taken for the causal mask, as is_causal
  says of it in torch.nn.MultiheadAttention; its values are not read.  is_causal without a mask is `attention`'s.

  key_padding_mask is bool, or floating point with 0 for a key and -inf for none, which is what torch's own layers make
  of a bool mask.  Any other value would be added to the scores, which the kernels do not offer; it is not looked for on
  the host: a query that sees such a key gets NaN."""

  def forward(self, query, key, value, key_padding_mask=None, need_weights=False, attn_mask=None,
              average_attn_weights=True, is_causal=False):
    if need_weights:
      raise ValueError('MultiheadAttention: need_weights=True is not supported, the probabilities are never stored')
    if self.dropout and self.training:
      raise ValueError('MultiheadAttention: dropout of the probabilities is not supported in training')
    if self.bias_k is not None or self.bias_v is not None or self.add_zero_attn:
      raise ValueError('MultiheadAttention: bias_k, bias_v and add_zero_attn are not supported')
    if query.dim() != 3:
      raise ValueError('MultiheadAttention: batched inputs only (got %d dimensions)' % query.dim())
    if attn_mask is not None:
      L, S = (t.shape[1 if self.batch_first else 0] for t in (query, key))
      if not (is_causal and L == S and tuple(attn_mask.shape) == (L, S)):
        raise ValueError('MultiheadAttention: attn_mask is not supported, but for the [length, length] one with is_causal=True')
    E = self.embed_dim
    if self._qkv_same_embed_dim:
      wq, wk, wv = self.in_proj_weight.split(E)
    else:
      wq, wk, wv = self.q_proj_weight, self.k_proj_weight, self.v_proj_weight
    bq, bk, bv = self.in_proj_bias.split(E) if self.in_proj_bias is not None else (None, None, None)
    q, k, v = F.linear(query, wq, bq), F.linear(key, wk, bk), F.linear(value, wv, bv)
    if not self.batch_first:                            # [length, batch, channels]: the heads are views, nothing is moved
      q, k, v = q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1)
    if key_padding_mask is not None and key_padding_mask.is_floating_point():
      k = k.masked_fill((key_padding_mask != 0)[..., None], math.nan)   # (what a hidden key holds does not matter)
      key_padding_mask = key_padding_mask == -math.inf
    heads = [t.unflatten(-1, (self.num_heads, self.head_dim)) for t in (q, k, v)]
    out = attention(*heads, key_padding_mask=key_padding_mask, is_causal=is_causal).flatten(2)
    if not self.batch_first:
      out = out.transpose(0, 1)
    return self.out_proj(out), None


def use_attention_kernels(module):
  """Switches every torch.nn.MultiheadAttention inside `module` (a TransformerClustering, its `_transformer`, a ViT) over
  to MultiheadAttention above, in place and without touching its parameters.  Returns how many were switched; a module
  that could not be called afterwards (dropout in training mode, bias_k / bias_v, add_zero_attn, heads wider than
  MAX_HEAD_WIDTH) raises and nothing is switched.  One with dropout that is in evaluation mode is switched and raises when
  it is called in training mode.

  torch.nn.TransformerEncoderLayer in evaluation, with batch_first and without gradients, takes a fused path of torch's own
  and does not call its attention module; torch.backends.mha.set_fastpath_enabled(False) makes it."""
  found = [m for m in module.modules() if type(m) is torch.nn.MultiheadAttention]
  for m in found:
    if (m.dropout and m.training) or m.bias_k is not None or m.bias_v is not None or m.add_zero_attn:
      raise ValueError('use_attention_kernels: an attention module uses dropout in training, bias_k / bias_v or add_zero_attn')
    if m.head_dim > MAX_HEAD_WIDTH:
      raise ValueError('use_attention_kernels: head width %d, at most %d' % (m.head_dim, MAX_HEAD_WIDTH))
  for m in found:
    m.__class__ = MultiheadAttention
  return len(found)


def forward(self, src, mask, query_embed, pos_embed):
  """Same arguments and results as the reference: src [B,C,sl], mask [B,sl] bool, query_embed
  [tl,C] or [B,C,tl], pos_embed [B,C,sl] -> (centroids [B,C,k], centroid_feats [B,C,k],
  logits [B,k,sl], node_features [B,C,sl])."""
  bs, cs, _ = src.shape
  centroids, node_features = self._transformer(src, mask, query_embed, pos_embed)   # :81-84
  tl = centroids.shape[-1]
  flat_centroids = centroids.transpose(1, 2).flatten(0, 1)                          # :86
  centroids = self.centroid_fc(flat_centroids).view(bs, tl, cs).transpose(1, 2)
  centroid_feats = self.centroid_feat_fc(flat_centroids).view(bs, tl, cs).transpose(1, 2)
  c_sel, cf_sel, logits, _order = hierarchy.transformer_clustering_tail(               # :91-112
      centroids, centroid_feats, node_features, self._num_clusters)
  return c_sel, cf_sel, logits, node_features


class TransformerClusteringMixin:
  """class TransformerClustering(TransformerClusteringMixin, reference.TransformerClustering)"""
  forward = forward
