"""Attention of a batch over a prefix that all its rows share (no reference
counterpart): the prefix's K and V are kept once, unquantised, and read once
for the whole batch; each row's own tokens stay in the cache (or in a prompt
chunk) and their attention is joined with the prefix's as one softmax.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib


def check_prefix(prefix, heads: int, head_dim: int, dtype, device):
    """Refuse a (k, v) that prefix_attention would not take behind `heads` query heads."""
    if len(prefix) != 2:
        raise ValueError(f"prefix must be (k, v); got {len(prefix)} values")
    k, v = prefix
    if k.dim() != 3 or k.shape[2] != head_dim or v.shape != k.shape or not k.shape[0] or heads % k.shape[0]:
        raise ValueError(f"prefix k {tuple(k.shape)} and v {tuple(v.shape)} must be (kv heads, P, {head_dim}) alike, "
                         f"with kv heads dividing {heads}")
    if head_dim not in (64, 128):
        raise ValueError(f"a prefix needs head_dim 64 or 128 (got {head_dim})")
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"prefix k and v must be {dtype} (got {k.dtype}, {v.dtype})")
    if k.device != device or v.device != device:
        raise _lib.CarekvError(f"prefix on {k.device} / {v.device}, the queries on {device}")


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     own: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, sm_scale: Optional[float] = None,
                     return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of every row of q over the one prefix k, v (Hkv, P, D), joined
    with the row's attention over tokens of its own.

    q (B, Hq, D), one token a sequence, or (B, Hq, T, D); fp16 or bf16, any
    strides, Hq a multiple of Hkv.  Every row sees the whole prefix (its tokens
    come before all of q's).  ``own`` = (o, lse): the row's attention over its
    own tokens, o like q and lse (B, Hq) or (B, Hq, T) fp32, as
    ``decode_attention(..., return_lse=True)`` or ``prefill_attention(...,
    return_lse=True)`` gives them, with -inf where a row has no token of its own
    (that row of o is not used).  Returns o like q and, with ``return_lse``, the
    joint log-sum-exp.  A row that sees nothing is 0 with lse -inf.  ``out`` may
    be own's o itself.  The results carry no autograd history."""
    one = q.dim() == 3
    o_own, l_own = (None, None) if own is None else own
    if one:
        q = q.unsqueeze(2)
        out = None if out is None else out.unsqueeze(2)
        if own is not None:
            o_own, l_own = o_own.unsqueeze(2), l_own.unsqueeze(2)
    if q.dim() != 4 or k.dim() != 3:
        raise ValueError(f"q must be (B, Hq, D) or (B, Hq, T, D) and k (Hkv, P, D); got {tuple(q.shape)} / "
                         f"{tuple(k.shape)}")
    B, Hq, T, D = q.shape
    Hkv, P = k.shape[:2]
    if k.shape[2] != D or v.shape != k.shape or Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if D not in (64, 128):
        raise ValueError(f"prefix_attention: head_dim 64 or 128 (got {D})")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"prefix_attention: q, k and v all fp16 or all bf16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    if own is not None:
        if o_own.shape != q.shape or o_own.dtype != q.dtype or l_own.shape != q.shape[:3] or \
                l_own.dtype != torch.float32:
            raise ValueError(f"own must be an output like q and its fp32 log-sum-exp {tuple(q.shape[:3])}; got "
                             f"{tuple(o_own.shape)} {o_own.dtype}, {tuple(l_own.shape)} {l_own.dtype}")
        o_own = o_own if o_own.stride(3) == 1 else o_own.contiguous()
        l_own = l_own.contiguous()
    if out is not None:
        _lib.check_out(out, q.shape, q.dtype, "out", q, k, v, *(() if own is None else (o_own, l_own)))
    dev = _lib.same_device("prefix_attention", q, k, v, o_own, l_own, out)
    if out is None:
        out = q.new_empty(q.shape)
    lse = q.new_empty((B, Hq, T), dtype=torch.float32) if return_lse else None
    if out.numel():
        q, k, v = _lib.aligned_rows(q), _lib.aligned_rows(k, near=True), _lib.aligned_rows(v, near=True)
        pp = _lib.PrefixParams(B, Hq, Hkv, T, P, D, _lib.DTYPE_CODE[q.dtype],
                               1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), *q.stride()[:3],
                               *k.stride()[:2], *v.stride()[:2], *out.stride()[:3],
                               *((0, 0, 0) if own is None else o_own.stride()[:3]))
        lib = _lib.load()
        nbytes = lib.carekv_prefix_attn_workspace_bytes(pp)
        if nbytes < 0:
            _lib.check(-1, "carekv_prefix_attn_workspace_bytes")
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _lib.call(dev, "carekv_prefix_attn", lib.carekv_prefix_attn, pp, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  None if own is None else o_own.data_ptr(), None if own is None else l_own.data_ptr(), out.data_ptr(),
                  None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    if one:
        out, lse = out.squeeze(2), None if lse is None else lse.squeeze(2)
    return (out, lse) if return_lse else out
