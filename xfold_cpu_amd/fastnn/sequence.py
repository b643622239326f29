"""``sequence_attention``: attention over token sequences with gradients, beside
``dot_product_attention`` (``xfold/fastnn/attention.py:45-98``), which has additive biases and key masks and
serves inference."""

from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import config as fastnn_config
from . import native_hip as nh

_NO_STRIDES = (0, 0, 0)
_CODES = {torch.float32: nh.F32, torch.bfloat16: nh.BF16}
# nh.SequenceAttention as bytes: 15 addresses, 33 sizes and strides, scale, softcap, causal, dtype.
_PACKED = struct.Struct("15Q33q2f2i")
assert _PACKED.size == ctypes.sizeof(nh.SequenceAttention)


def _cast(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    t = t.contiguous()
    out = torch.empty(t.shape, dtype=dtype, device=t.device)
    nh.launch(t.device, "xfh_convert", t.data_ptr(), _CODES[t.dtype], out.data_ptr(), _CODES[dtype], t.numel())
    return out


def _rows(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``t`` in ``dtype`` with a contiguous last dim (any strides before it)."""
    if t.dtype != dtype:
        return _cast(t, dtype)
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _empty(like: torch.Tensor, heads: int, tokens: int, dim: int) -> torch.Tensor:
    """[B, heads, tokens, dim] in the memory order of ``like``: token by token where its heads lie side by
    side, else head by head."""
    batch = like.shape[0]
    if like.stride(1) < like.stride(2):
        return torch.empty((batch, tokens, heads, dim), dtype=like.dtype, device=like.device).transpose(1, 2)
    return torch.empty((batch, heads, tokens, dim), dtype=like.dtype, device=like.device)


def _address(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _strides(t: Optional[torch.Tensor]) -> tuple:
    return _NO_STRIDES if t is None else t.stride()[:3]


def _call(name, q, k, v, out, lse, low, slopes, masks, options, dout=None, dq=None, dk=None, dv=None, dslopes=None):
    prefix, documents, lengths = masks
    causal, prefix_all, softcap, scale = options
    device = q.device
    batch, heads, queries, dim = q.shape
    kv_heads, keys, value_dim = v.shape[1:]
    args = _PACKED.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _address(lse), _address(low), _address(slopes), _address(prefix),
        _address(documents), _address(lengths), _address(dout), _address(dq), _address(dk), _address(dv),
        _address(dslopes), batch, heads, kv_heads, queries, keys, dim, value_dim,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3],
        *_strides(dout), *_strides(dq), *_strides(dk), *_strides(dv),
        0 if documents is None else documents.stride(0), prefix_all, scale, softcap, causal, _CODES[q.dtype])
    size = nh.function(name + "_workspace_size")(args)
    if size <= 0:                                        # (none needed, or arguments that the call refuses)
        return nh.launch(device, name, args, None, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    nh.launch(device, name, args, ws.data_ptr(), size)


def _forward(q, k, v, slopes, masks, options, keep):
    out = _empty(q, q.shape[1], q.shape[2], v.shape[3])
    lse = low = None
    if keep:                                             # for the backward pass: row sums, and what rounding left out
        single = q.dtype == torch.float32
        lse = torch.empty((1 + single, *q.shape[:3]), dtype=torch.float32, device=q.device)
        if not single:
            low = torch.empty((*q.shape[:3], v.shape[3]), dtype=torch.bfloat16, device=q.device)
    _call("xfh_sequence_attention", q, k, v, out, lse, low, slopes, masks, options)
    return out, lse, low


class _SequenceAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, documents, lengths, options, dtype):
        ctx.dtypes = q.dtype, k.dtype, v.dtype, None if slopes is None else slopes.dtype
        q, k, v = (_rows(t, dtype) for t in (q, k, v))
        s = None if slopes is None else slopes.to(torch.float32).contiguous()
        out, lse, low = _forward(q, k, v, s, (prefix, documents, lengths), options, True)
        ctx.save_for_backward(q, k, v, s, out, lse, low, prefix, documents, lengths)
        ctx.options = options
        return out

    @staticmethod
    def backward(ctx, dout):
        # Gradients that are to be differentiated again get the node that refuses it.
        return _backward_once(ctx, dout) if torch.is_grad_enabled() else _backward(ctx, dout)


def _backward(ctx, dout):
    q, k, v, slopes, out, lse, low, *masks = ctx.saved_tensors
    dout = _rows(dout, q.dtype)
    needs = ctx.needs_input_grad
    dq, dk, dv = _empty(q, *q.shape[1:]), None, None
    if needs[1] or needs[2]:
        dk, dv = _empty(k, *k.shape[1:]), _empty(v, *v.shape[1:])
    dslopes = torch.empty_like(slopes) if needs[3] else None
    _call("xfh_sequence_attention_backward", q, k, v, out, lse, low, slopes, masks, ctx.options, dout, dq, dk, dv, dslopes)
    grads = [dq, dk, dv, dslopes]
    for i, dtype in enumerate(ctx.dtypes):
        if not needs[i]:
            grads[i] = None
        elif grads[i].dtype != dtype:
            grads[i] = _cast(grads[i], dtype)
    return (*grads, None, None, None, None, None)


_backward_once = once_differentiable(_backward)


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
    options = (bool(causal), prefix_all, softcap, scale)
    if nh.needs_gradient(q, k, v, slopes):
        return _SequenceAttention.apply(q, k, v, slopes, prefix, documents, lengths, options, dtype)
    if slopes is not None:
        slopes = slopes.to(torch.float32).contiguous()
    return _forward(*(_rows(t, dtype) for t in (q, k, v)), slopes, (prefix, documents, lengths), options, False)[0]
