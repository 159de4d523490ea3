"""Attention inside a window and over a few first tokens (no reference
counterpart; ``prefill_attention`` is the full causal form of equal lengths): of
prompts, of their later chunks and of single tokens over unquantised rows.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .pages import check_window


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: Optional[int] = None, sink: int = 0,
                     lengths=None, q_lengths=None, q_start=None, sm_scale: Optional[float] = None,
                     return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Causal attention of q (B, Hq, Tq, D) over k, v (B, Hkv, Tk, D), fp16 or
    bf16, any strides, Hq a multiple of Hkv; (Hq, Tq, D) and (Hkv, Tk, D) of one
    sequence work alike.  Query row i of sequence b stands at position
    ``q_start[b] + i`` and sees the keys below ``lengths[b]`` (default Tk) up to
    its own position, with ``window`` only the last ``window`` of those positions
    and the first ``sink`` keys.  Rows from ``q_lengths[b]`` on are padding and see
    nothing.  Default of q_lengths: Tq, but where neither it nor q_start is given
    and Tq = Tk, the lengths (row i of q and of k are one token of a right-padded
    prompt); of q_start: the rows are the last of the sequence, lengths[b] -
    q_lengths[b] + i.  lengths, q_lengths and q_start: a device tensor of B
    integers, one int for all, or (not in captured code) a host sequence.

    Returns o like q and, with ``return_lse``, the natural log-sum-exp of each
    row's scaled scores, fp32 (B, Hq, Tq), as ``attention_mass`` and
    ``prefix_attention`` take it.  Rows that see nothing are 0 with lse -inf; a
    score of -inf has no weight.  What keys that a row does not see hold (NaN
    included) is never used; an infinite value that it sees is its result whatever
    the weight.  ``out`` may be q itself.  The results carry no autograd
    history.

    Scores, the softmax's sums and the output's are 32 bits; the weights are
    rounded to the operands' type (half a step of each, 2^-11 in fp16, 2^-8 in
    bf16) before their product with v."""
    squeeze = q.dim() == 3
    if squeeze:
        q, k, v = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
        out = None if out is None else out.unsqueeze(0)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"q must be (B, Hq, Tq, D), k and v (B, Hkv, Tk, D); got {tuple(q.shape)} / {tuple(k.shape)} / "
                         f"{tuple(v.shape)}")
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D or Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}")
    if D not in (64, 128):
        raise ValueError(f"window_attention: head_dim 64 or 128 (got {D})")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"window_attention: q, k and v all fp16 or all bf16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    window, sink = check_window(window, sink)
    if out is not None:
        _lib.check_out(out, q.shape, q.dtype, "out", q)
        if _lib.overlap(out, k) or _lib.overlap(out, v):
            raise ValueError("out must not overlap k or v")
    dev = _lib.same_device("window_attention", q, k, v, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, Tq), dtype=torch.float32) if return_lse else None
    if out.numel():
        if not q.is_contiguous() or q.data_ptr() % 16:
            q = _lib.aligned_rows(q)
        k, v = (x if x.is_contiguous() and x.data_ptr() % 16 == 0 else _lib.aligned_rows(x, near=True) for x in (k, v))
        ln = _lib.row_counts(lengths, B, dev, "lengths")
        qs = _lib.row_counts(q_start, B, dev, "q_start")
        ql = ln if q_lengths is None and q_start is None and Tq == Tk else \
            _lib.row_counts(q_lengths, B, dev, "q_lengths")
        pp = _lib.window_params(B, Hq, Hkv, Tq, Tk, D, _lib.DTYPE_CODE[q.dtype], window, sink,
                               1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), *q.stride()[:3],
                               *k.stride()[:3], *v.stride()[:3], *out.stride()[:3])
        lib = _lib.load()
        nbytes = lib.carekv_window_attn_workspace_bytes(pp)
        if nbytes < 0:
            _lib.check(-1, "carekv_window_attn_workspace_bytes")
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        _lib.call(dev, "carekv_window_attn", lib.carekv_window_attn, pp, q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(ln),
                  ptr(ql), ptr(qs), out.data_ptr(), ptr(lse), ptr(ws), nbytes)
    if squeeze:
        out, lse = out[0], None if lse is None else lse[0]
    return (out, lse) if return_lse else out
