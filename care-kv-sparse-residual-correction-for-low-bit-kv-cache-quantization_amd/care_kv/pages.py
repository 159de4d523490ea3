"""Pages of 4-bit rows whose lengths live on the device (no reference
counterpart): several new tokens a sequence are written in one call, read back
by attention that may be bounded to a window and a few first tokens, and taken
back by counting them no more.  Beside ``CAREKVCache``, which keeps residual
slots, one token a step and its lengths on the host, this is the cache of a
serving loop that runs as a captured graph or verifies drafted tokens
(``verify_drafts``)::

    q = append_pages(pages, table, lengths, k, v, q=q, plan=plan)
    o = paged_attention(q, pages, table, lengths + T, window=4096, sink=4)

A page holds 16 tokens of a sequence.  Of a row every 32 values are kept as
``quantize_rows(x, 4)`` gives them: a scale s = half(max|x| / 7) and codes
clamp(round(half(x / s)), -8, 7), which stand for half(code * s); a group with a
value that is not finite stands for NaN.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .rotary import RotaryPlan

PAGE = 16


@dataclass(frozen=True)
class Int4Pages:
    """A pool of pages of one layer: ``data`` uint8 (n_pages, kv heads, bytes of
    a block), zeros at first.  Which pages a sequence has is its row of a page
    table, int32 (B, max_pages) on the device: entry i is the page of its tokens
    16 i .. 16 i + 15.  An entry outside 0 .. n_pages - 1 is a page that is not
    there (one behind a window that was given back, say): what is appended to it
    is dropped, its tokens are seen by no row.  Sequences may share pages that
    none of them writes to any more."""
    data: torch.Tensor
    head_dim: int

    def __post_init__(self):
        if self.head_dim not in (64, 128):
            raise ValueError(f"pages of 4-bit rows need head_dim 64 or 128 (got {self.head_dim})")
        n = block_bytes(self.head_dim)
        d = self.data
        if d.dim() != 3 or d.shape[2] != n or not d.shape[1] or d.dtype != torch.uint8 or not d.is_contiguous() or \
                d.data_ptr() % 16:
            raise ValueError(f"pages must be packed uint8 (n_pages, kv heads, {n}) on 16 bytes; got {tuple(d.shape)} "
                             f"{d.dtype}")

    @property
    def n_pages(self) -> int:
        return self.data.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.data.shape[1]


def block_bytes(head_dim: int) -> int:
    """Bytes of 16 tokens of one kv head, K and V with their scales: 4.5 bits a value."""
    return 2 * PAGE * (head_dim // 2 + head_dim // 32 * 2)


def int4_pages(n_pages: int, n_kv_heads: int, head_dim: int, *, device=None) -> Int4Pages:
    """A pool of ``n_pages`` pages for ``n_kv_heads`` heads of ``head_dim`` (64 or 128)."""
    if n_pages < 0 or n_kv_heads < 1 or head_dim not in (64, 128):
        raise ValueError(f"int4_pages: n_pages not negative, n_kv_heads positive, head_dim 64 or 128 (got {n_pages}, "
                         f"{n_kv_heads}, {head_dim})")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    return Int4Pages(torch.zeros(n_pages, n_kv_heads, block_bytes(head_dim), dtype=torch.uint8, device=device), head_dim)


_NONE = (0, 0, 0)


def _ptr(x: Optional[torch.Tensor]):
    return None if x is None else x.data_ptr()


def _check_table(table: torch.Tensor, batch: int) -> torch.Tensor:
    if table.dim() != 2 or table.shape[0] != batch or table.dtype != torch.int32:
        raise ValueError(f"table must be ({batch}, max_pages) int32; got {tuple(table.shape)} {table.dtype}")
    return table if table.stride(1) == 1 or table.shape[1] < 2 else table.contiguous()


def check_window(window, sink) -> tuple:
    """(window, 0: no bound; sink), refused where they are no counts."""
    if window is not None and window < 1:
        raise ValueError(f"window must be None or at least 1 (got {window})")
    if sink < 0:
        raise ValueError(f"sink must not be negative (got {sink})")
    top = 2 ** 30  # (more keys than a call takes)
    return 0 if window is None else min(int(window), top), min(int(sink), top)


def append_pages(pages: Int4Pages, table: torch.Tensor, start, k: torch.Tensor, v: torch.Tensor, *,
                 q: Optional[torch.Tensor] = None, plan: Optional[RotaryPlan] = None,
                 positions: Optional[torch.Tensor] = None, counts=None, return_hat: bool = False):
    """Write T new tokens of every sequence to its pages, k (and q) turned to
    their positions on the way, in one launch; returns q turned (None without q)
    and, with ``return_hat``, (q, k_hat, v_hat).

    k and v (B, Hkv, T, D), q (B, Hq, T, D), fp16 or bf16 of one type, any strides
    (a projection's (B, T, heads, D) seen through ``transpose(1, 2)`` is read in
    place).  Token t of sequence b goes to place ``start[b] + t``; of a ragged
    batch the first ``counts[b]`` tokens do (default T), q's are turned all.
    start, counts: a device tensor of B integers, one int for all, or (not in
    captured code) a host sequence.  ``plan``: turned as by ``rotate_heads`` at
    ``positions`` (int32 or int64 (B, T), (1, T) or (T,); default start + t), in 64
    bits, rounded to 32 and then, q to the type, k to fp16; without a plan k and q
    are taken as they are.  k_hat, v_hat: fp16 (B, Hkv, T, D), the values that the new rows
    stand for, zeros behind the counts.

    Tokens before place 0, behind the table or on pages that are not there are
    dropped.  A call may write to a page for one sequence only, and for one entry of
    its table.  The results carry no autograd history."""
    kd, ks, dev = k.dtype, k.shape, k.device
    if len(ks) != 4 or v.shape != ks or v.dtype != kd:
        raise ValueError(f"k and v must be (B, Hkv, T, D) of one type; got {tuple(ks)} {kd}, {tuple(v.shape)} {v.dtype}")
    B, Hkv, T, D = ks
    if kd != torch.float16 and kd != torch.bfloat16:
        raise ValueError(f"append_pages: fp16 or bf16 rows (got {kd})")
    data = pages.data
    n_pages, heads, _ = data.shape
    if Hkv != heads or D != pages.head_dim:
        raise ValueError(f"k {tuple(ks)} does not fit pages of {heads} kv heads, head_dim {pages.head_dim}")
    Hq, qo, sq, so = 0, None, _NONE, _NONE
    if q is not None:
        if q.dim() != 4 or q.dtype != kd or (q.shape[0], q.shape[2], q.shape[3]) != (B, T, D):
            raise ValueError(f"q must be ({B}, heads, {T}, {D}) {kd}; got {tuple(q.shape)} {q.dtype}")
        Hq = q.shape[1]
    table = _check_table(table, B)
    R, layout, scale, freqs = 0, False, 1.0, None
    if plan is not None:
        R, layout, scale, freqs = plan.rotary_dim, plan.layout == "interleaved", plan.scale, plan.freqs
        if R > D:
            raise ValueError(f"head_dim {D} must be at least the plan's rotary_dim {R}")
    elif positions is not None:
        raise ValueError("positions need a plan")
    pos, pos_bits, pos_batch = positions, 64, 0
    if pos is not None:
        pos = pos.unsqueeze(0) if pos.dim() == 1 else pos
        if pos.dtype not in (torch.int32, torch.int64) or pos.dim() != 2 or pos.shape[0] not in (1, B) or pos.shape[1] != T:
            raise ValueError(f"positions must be int32 or int64 ({B}, {T}), (1, {T}) or ({T},); got "
                             f"{tuple(positions.shape)} {positions.dtype}")
        pos = pos if pos.stride(1) == 1 or T == 1 else pos.contiguous()
        pos_bits, pos_batch = 64 if pos.dtype == torch.int64 else 32, pos.stride(0) if pos.shape[0] > 1 else 0
    _lib.same_device("append_pages", k, v, q, data, table, pos, freqs)
    if start is None:
        raise ValueError("append_pages needs start, the tokens that the sequences hold")
    if q is not None:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    kh = vh = None
    if return_hat:
        kh = torch.empty_like(k, dtype=torch.float16, memory_format=torch.contiguous_format)
        vh = torch.empty_like(kh)
    if B and T:
        sk, sv = k.stride(), v.stride()
        if sk[3] != 1:
            k = k.contiguous()
            sk = k.stride()
        if sv[3] != 1:
            v = v.contiguous()
            sv = v.stride()
        if q is not None:
            if q.stride(3) != 1:
                q = q.contiguous()
            sq, so = q.stride(), qo.stride()
        st, ct = _lib.row_counts(start, B, dev, "start"), _lib.row_counts(counts, B, dev, "counts")
        pp = _lib.append_params(B, Hq, Hkv, T, D, R, _lib.DTYPE_CODE[kd], layout, pos_bits, n_pages, table.shape[1], scale,
                               pos_batch, table.stride(0), sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                               so[0], so[1], so[2])
        _lib.call(dev, "carekv_append_pages", _lib.load().carekv_append_pages, pp, _ptr(q), k.data_ptr(), v.data_ptr(),
                  _ptr(pos), _ptr(freqs), st.data_ptr(), _ptr(ct), table.data_ptr(), data.data_ptr(), _ptr(qo), _ptr(kh),
                  _ptr(vh))
    return (qo, kh, vh) if return_hat else qo


def paged_attention(q: torch.Tensor, pages: Int4Pages, table: torch.Tensor, lengths, *, q_lengths=None,
                    window: Optional[int] = None, sink: int = 0, sm_scale: Optional[float] = None,
                    return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """Attention of each sequence's last rows over its pages.

    q (B, Hq, T, D), or (B, Hq, D) for one row a sequence; fp16 or bf16, any
    strides, Hq a multiple of the pages' kv heads.  ``lengths``: the tokens of
    each sequence, those of q among them (written by ``append_pages`` before);
    row t < ``q_lengths[b]`` (default T) is token lengths[b] - q_lengths[b] + t
    and sees the tokens up to itself, with ``window`` only the last ``window`` of
    them and the sequence's first ``sink``.  Lengths past the table count as its
    end.  lengths, q_lengths: as ``start`` of ``append_pages``.

    Returns o like q and, with ``return_lse``, the natural log-sum-exp of each
    row's scaled scores, fp32 (B, Hq, T).  Rows of padding and rows that see
    nothing are 0 with lse -inf; a score of -inf has no weight.  What places that a
    row does not see hold (NaN included) is never used; a group that stands for NaN
    is NaN in the rows that see it.  ``out`` may be q itself.  The results carry no
    autograd history.

    Scores, the softmax's sums and the output's are 32 bits; the weights are
    rounded to fp16 (half a step, 2^-11 of each) before their product with V, and
    bf16 rows of q are scaled by a power of two into fp16."""
    one = q.dim() == 3
    if one:
        q = q.unsqueeze(2)
        out = None if out is None else out.unsqueeze(2)
    if q.dim() != 4:
        raise ValueError(f"q must be (B, Hq, D) or (B, Hq, T, D); got {tuple(q.shape)}")
    B, Hq, T, D = q.shape
    if D != pages.head_dim or Hq == 0 or Hq % pages.n_kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit pages of {pages.n_kv_heads} kv heads, head_dim {pages.head_dim}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"paged_attention: fp16 or bf16 queries (got {q.dtype})")
    table = _check_table(table, B)
    window, sink = check_window(window, sink)
    if out is not None:
        _lib.check_out(out, q.shape, q.dtype, "out", q)
        if _lib.overlap(out, pages.data):
            raise ValueError("out must not overlap the pages")
    dev = _lib.same_device("paged_attention", q, pages.data, table, out)
    if lengths is None:
        raise ValueError("paged_attention needs lengths")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, T), dtype=torch.float32) if return_lse else None
    if out.numel():
        qq = _lib.aligned_rows(q) if not q.is_contiguous() or q.data_ptr() % 16 else q
        ln = _lib.row_counts(lengths, B, dev, "lengths")
        ql = _lib.row_counts(q_lengths, B, dev, "q_lengths")
        pp = _lib.paged_params(B, Hq, pages.n_kv_heads, T, D, _lib.DTYPE_CODE[q.dtype], pages.n_pages, table.shape[1],
                              window, sink, 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), table.stride(0),
                              *qq.stride()[:3], *out.stride()[:3])
        lib = _lib.load()
        nbytes = lib.carekv_paged_attn_workspace_bytes(pp)
        if nbytes < 0:
            _lib.check(-1, "carekv_paged_attn_workspace_bytes")
        ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _lib.call(dev, "carekv_paged_attn", lib.carekv_paged_attn, pp, qq.data_ptr(), pages.data.data_ptr(),
                  table.data_ptr(), ln.data_ptr(), None if ql is None else ql.data_ptr(), out.data_ptr(),
                  None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    if one:
        out, lse = out.squeeze(2), None if lse is None else lse.squeeze(2)
    return (out, lse) if return_lse else out
