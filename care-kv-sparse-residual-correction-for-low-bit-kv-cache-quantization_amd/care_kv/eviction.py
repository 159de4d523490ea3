"""Rows of a prompt kept by the attention they get (no reference counterpart):
``attention_mass`` adds up the weight that each key gathers from the query
rows that see it, ``evict_rows`` keeps the first, the last and the heaviest
rows and gathers their K and V for ``CAREKVCache.write_prefill`` or as the
shared prefix of ``prefix_attention``.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib


class EvictedRows(NamedTuple):
    """What ``evict_rows`` kept, in index order; places past a sequence's kept
    rows hold zeros and index -1.  ``write_prefill`` and ``prefix_attention``
    know no lengths and would take those zeros for rows: of a sequence shorter
    than keep they are given k[b, :, :n] and v[b, :, :n], n = lengths[b]."""
    k: torch.Tensor        # (B, Hkv, keep, D)
    v: torch.Tensor
    mass: torch.Tensor     # (B, Hkv, keep) fp32
    index: torch.Tensor    # (B, Hkv, keep) int32 row of each in the prompt
    lengths: torch.Tensor  # (B,) int32 min(length, keep)


def attention_mass(q: torch.Tensor, k: torch.Tensor, *, lse: Optional[torch.Tensor] = None, causal: bool = True,
                   sm_scale: Optional[float] = None, q_start=None, lengths=None, q_lengths=None,
                   out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The attention weight each key has gathered, fp32 (B, Hkv, Tk):
    mass[b, g, j] = sum over the query heads of kv head g and the query rows i
    that see key j of exp(sm_scale q_i . k_j - lse_i).

    q (B, Hq, Tq, D) and k (B, Hkv, Tk, D), fp16 or bf16, any strides; (Hq, Tq,
    D) and (Hkv, Tk, D) of one sequence work alike.  Query row i of sequence b
    stands at position ``q_start[b] + i`` and sees the keys below ``lengths[b]``
    (default Tk) and, with ``causal``, up to its own position: Tq = Tk is a
    prompt, a few last rows are a voting window, Tq = 1 a decode step.  Rows from
    ``q_lengths[b]`` on are padding and see nothing.  Default of q_lengths: Tq,
    but where neither it nor q_start is given and Tq = Tk, the lengths (row i of
    q and of k are one token of a right-padded prompt); of q_start: the rows are
    the last of the sequence, lengths[b] - q_lengths[b] + i.  q_start, lengths
    and q_lengths: a device tensor of B integers, one int for all, or (not in
    captured code) a host sequence.  lse (B, Hq, Tq) fp32: the
    rows' log-sum-exp as ``prefill_attention(..., return_lse=True)`` gives it;
    without it an extra pass computes it.  ``accumulate`` adds to ``out``, whose
    values of a head must lie next to each other.

    Rows that see nothing, or whose lse is infinite, add nothing; what they and
    the keys behind a length hold is never used (NaN included).  Sums run in a fixed
    order.  The result carries no autograd history."""
    squeeze = q.dim() == 3
    if squeeze:
        q, k = q.unsqueeze(0), k.unsqueeze(0)
        lse = None if lse is None else lse.unsqueeze(0)
        out = None if out is None else out.unsqueeze(0)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q must be (B, Hq, Tq, D) and k (B, Hkv, Tk, D); got {tuple(q.shape)} / {tuple(k.shape)}")
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D or Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}")
    if D not in (64, 128):
        raise ValueError(f"attention_mass: head_dim 64 or 128 (got {D})")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype:
        raise ValueError(f"attention_mass: q and k both fp16 or both bf16 (got {q.dtype}, {k.dtype})")
    if lse is not None:
        if lse.shape != (B, Hq, Tq) or lse.dtype != torch.float32:
            raise ValueError(f"lse must be {(B, Hq, Tq)} fp32; got {tuple(lse.shape)} {lse.dtype}")
        lse = lse.contiguous()
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    if out is not None:
        _lib.check_out(out, (B, Hkv, Tk), torch.float32, "out")
        if any(_lib.overlap(out, x) for x in (q, k, lse) if x is not None):
            raise ValueError("out must not overlap q, k or lse")
    dev = _lib.same_device("attention_mass", q, k, lse, out)
    if out is None:
        out = q.new_empty((B, Hkv, Tk), dtype=torch.float32)
    if B and Tk:
        q, k = _lib.aligned_rows(q, near=True), _lib.aligned_rows(k, near=True)
        pp = _lib.MassParams(B, Hq, Hkv, Tq, Tk, D, _lib.DTYPE_CODE[q.dtype], bool(causal), bool(accumulate),
                             1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), *q.stride()[:3],
                             *k.stride()[:3], *out.stride()[:2])
        lib = _lib.load()
        qs = _lib.row_counts(q_start, B, dev, "q_start")
        ln = _lib.row_counts(lengths, B, dev, "lengths")
        ql = ln if q_lengths is None and q_start is None and Tq == Tk else \
            _lib.row_counts(q_lengths, B, dev, "q_lengths")
        pp.q_lengths = None if ql is None else ql.data_ptr()
        nbytes = lib.carekv_attention_mass_workspace_bytes(pp, lse is not None)
        if nbytes < 0:
            _lib.check(-1, "carekv_attention_mass_workspace_bytes")
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _lib.call(dev, "carekv_attention_mass", lib.carekv_attention_mass, pp, q.data_ptr(), k.data_ptr(),
                  None if lse is None else lse.data_ptr(), None if qs is None else qs.data_ptr(),
                  None if ln is None else ln.data_ptr(), out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return out[0] if squeeze else out


def evict_rows(mass: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, keep: int, sink: int = 0, recent: int = 0,
               lengths=None) -> EvictedRows:
    """The ``keep`` rows of each (sequence, kv head) that stay: the first
    ``sink``, the last ``recent`` and of the others those of largest ``mass``
    (equal weights: the lower index; NaN below everything), in index order.

    mass (B, Hkv, T) fp32; k and v (B, Hkv, T, D) of any 2- or 4-byte type and
    any strides ((Hkv, T) and (Hkv, T, D) of one sequence work alike, and give
    results without the batch dim, lengths with one value).  ``lengths``: rows of each sequence that
    count (default T), a device tensor of B integers or (not in captured code) a
    host sequence; what the rows behind them hold is not used.  The results have min(keep, T) places;
    sequences that are shorter keep every row."""
    squeeze = mass.dim() == 2
    if squeeze:
        mass, k, v = mass.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
    if mass.dim() != 3 or mass.dtype != torch.float32:
        raise ValueError(f"mass must be (B, Hkv, T) fp32; got {tuple(mass.shape)} {mass.dtype}")
    B, H, T = mass.shape
    if k.dim() != 4 or k.shape[:3] != mass.shape or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"k and v must be ({B}, {H}, {T}, D) of one type; got {tuple(k.shape)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    D, e = k.shape[3], k.element_size()
    if D == 0 or D * e % 4:
        raise ValueError(f"rows of {D} {k.dtype} values are not a multiple of 4 bytes")
    if keep <= 0 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError(f"keep must be positive, sink and recent not negative and at most keep together "
                         f"(got keep={keep}, sink={sink}, recent={recent})")
    dev = _lib.same_device("evict_rows", mass, k, v)
    n = min(int(keep), T)
    sink = min(int(sink), n)  # (with keep > T every row stays)
    recent = min(int(recent), n - sink)
    kk = k.new_empty((B, H, n, D))
    vv = k.new_empty((B, H, n, D))
    mm = mass.new_empty((B, H, n))
    index = mass.new_empty((B, H, n), dtype=torch.int32)
    kept = (mass.new_empty if B * H * n else mass.new_zeros)(B, dtype=torch.int32)
    if B * H * n:
        mass, k, v = _lib.aligned_rows(mass, 4), _lib.aligned_rows(k, 4), _lib.aligned_rows(v, 4)
        sk, sv = k.stride(), v.stride()
        pp = _lib.EvictParams(B, H, T, D * e, n, sink, recent, *mass.stride()[:2], sk[0] * e, sk[1] * e, sk[2] * e,
                              sv[0] * e, sv[1] * e, sv[2] * e)
        ln = _lib.row_counts(lengths, B, dev, "lengths")
        lib = _lib.load()
        nbytes = lib.carekv_evict_rows_workspace_bytes(pp)
        if nbytes < 0:
            _lib.check(-1, "carekv_evict_rows_workspace_bytes")
        ws = k.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _lib.call(dev, "carekv_evict_rows", lib.carekv_evict_rows, pp, mass.data_ptr(), k.data_ptr(), v.data_ptr(),
                  None if ln is None else ln.data_ptr(), kk.data_ptr(), vv.data_ptr(), mm.data_ptr(), index.data_ptr(),
                  kept.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    got = EvictedRows(kk, vv, mm, index, kept)
    return EvictedRows(*(x[0] for x in got[:4]), kept) if squeeze else got
