"""``sequence_attention``: attention over token sequences with gradients, beside
``dot_product_attention`` (``xfold/fastnn/attention.py:45-98``), which has additive biases and key masks and
serves inference."""

from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import config as fastnn_config
from . import native_hip as nh


def _integers(t, shape, what):
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"sequence_attention: {what} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def sequence_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False,
                       prefix: Optional[Union[int, torch.Tensor]] = None, documents: Optional[torch.Tensor] = None,
                       lengths: Optional[torch.Tensor] = None, softcap: Optional[float] = None,
                       slopes: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax over the visible keys of ``c(scale q.k) - slopes[h] * |p_i - j|``, times v, with
    ``c(x) = softcap * tanh(x / softcap)`` (or x), in FP32 between FP32 or BF16 tensors.

    ``q`` [B, H, Nq, D], ``k`` [B, Hk, Nk, D], ``v`` [B, Hk, Nk, Dv], or all without B; D and Dv at most
    128, H a multiple of Hk (neighbouring heads share a key head); any strides. The queries are the last Nq
    tokens of a sequence of n tokens, n = ``lengths[b]`` or Nk: query i is token ``p_i = n - Nq + i``. So Nq =
    Nk is a whole sequence, Nq = 1 the next token of one whose keys are in a cache, k and v being the cache.
    Query i sees key j if all of these hold:

    * j < n (keys from n on are not read);
    * with ``causal``: j <= p_i, or j < ``prefix`` (an int, or int32 [B]);
    * with ``documents`` (int32 [B, Nk] or [Nk]): tokens p_i and j have the same number, and it is not
      negative (a negative number is a token of no document: padding);
    * with ``lengths`` (int32 [B], held to 0..Nk): p_i >= 0.

    A query that sees no key gives zeros, and no gradient. What a masked place holds does not
    matter, be it NaN. ``slopes`` [H] (FP32/BF16) and ``scale`` (default D^-0.5) as in the formula.

    Gradients (once) of q, k, v and slopes, summed in a fixed order. The output has q's order of
    heads and tokens in memory. Under autocast q, k and v are taken in its type, as in
    ``dot_product_attention``. ValueError for other types, shapes, devices, and for Nq > Nk with a
    causal, document or length mask."""
    if fastnn_config.dot_product_attention_implementation != fastnn_config.HIP:
        raise ValueError("Unknown dot_product_attention_implementation for xfold_cpu_amd: "
                         f"{fastnn_config.dot_product_attention_implementation!r} (only 'hip')")
    if q.dim() == 3 and k.dim() == 3 and v.dim() == 3:
        out = sequence_attention(q[None], k[None], v[None], causal=causal, prefix=prefix, documents=documents,
                                 lengths=lengths, softcap=softcap, slopes=slopes, scale=scale)
        return out.squeeze(0)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("sequence_attention: q, k and v must be [B, H, N, D], or all [H, N, D]")
    batch, heads, queries, dim = q.shape
    kv_heads, keys, value_dim = k.shape[1], k.shape[2], v.shape[3]
    if tuple(k.shape) != (batch, kv_heads, keys, dim) or tuple(v.shape) != (batch, kv_heads, keys, value_dim):
        raise ValueError(f"sequence_attention: shapes do not match: q {list(q.shape)}, k {list(k.shape)}, v {list(v.shape)}")
    if not 1 <= dim <= 128 or not 1 <= value_dim <= 128:
        raise ValueError("sequence_attention: head dims must be 1 to 128")
    if heads % kv_heads if kv_heads else heads:
        raise ValueError("sequence_attention: the number of heads must be a multiple of the key heads")
    if prefix is not None and not causal:
        raise ValueError("sequence_attention: a prefix needs causal=True")
    if queries > keys and (causal or documents is not None or lengths is not None):
        raise ValueError("sequence_attention: more queries than keys with a causal, document or length mask")
    softcap = 0.0 if softcap is None else float(softcap)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale) or not 0.0 <= softcap < math.inf:
        raise ValueError("sequence_attention: scale must be finite, softcap finite and not negative")
    prefix_all = 0
    if isinstance(prefix, torch.Tensor):
        prefix = _integers(prefix, (batch,), "prefix")
    elif prefix is not None:
        prefix, prefix_all = None, min(max(int(prefix), 0), keys)
    if documents is not None and documents.dim() == 1:
        documents = documents.expand(batch, documents.shape[0])
        if documents.dtype != torch.int32 or documents.shape[1] != keys:
            raise ValueError(f"sequence_attention: documents must be int32 {[batch, keys]} or {[keys]}")
        if documents.stride(1) != 1:
            documents = documents.contiguous()
    else:
        documents = _integers(documents, (batch, keys), "documents")
    lengths = _integers(lengths, (batch,), "lengths")
    if slopes is not None and (tuple(slopes.shape) != (heads,) or slopes.dtype not in (torch.float32, torch.bfloat16)):
        raise ValueError(f"sequence_attention: slopes must be FP32/BF16 [{heads}]")
    nh.check_gpu(q, k, v, slopes, prefix, documents, lengths)
    dtype = nh.compute_dtype(q, k, v)
    return nh.autograd().sequence_attention(q, k, v, slopes, prefix, documents, lengths, bool(causal), prefix_all, softcap, scale,
                                            dtype == torch.bfloat16)
