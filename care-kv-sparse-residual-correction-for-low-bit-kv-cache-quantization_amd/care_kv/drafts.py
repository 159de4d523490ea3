"""Drafted tokens against the model's probabilities (no reference counterpart):
which of them stay, and the token behind them, so that what comes out is
distributed as the model's own sampling."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class VerifiedDrafts(NamedTuple):
    """What ``verify_drafts`` found."""
    tokens: torch.Tensor    # (B, T + 1) int32: the accepted tokens, the next one, -1 behind
    accepted: torch.Tensor  # (B,) int32: how many were accepted


def verify_drafts(draft: torch.Tensor, target_probs: torch.Tensor, u: torch.Tensor, u_next: torch.Tensor, *,
                  draft_probs: Optional[torch.Tensor] = None, counts=None) -> VerifiedDrafts:
    """draft (B, T) int32 or int64 tokens x_t that were drawn from ``draft_probs``
    (B, T, V), q_t; target_probs (B, T + 1, V), p_t: the model's probabilities
    behind each of them, of one type (fp32, fp16 or bf16).  Without draft_probs the
    tokens were guessed (looked up in the text, say): all of q_t is on x_t.  u (B,
    T) and u_next (B,): fp32 random numbers, uniform in [0, 1).

    Token t is accepted while u[b, t] q_t(x_t) < p_t(x_t); of a ragged batch the
    first ``counts[b]`` tokens are looked at (default T).  Behind the n accepted
    ones comes the smallest token i with w_0 + .. + w_i > u_next[b] sum(w): w = p_n
    where all were accepted, max(p_n - q_n, 0) where x_n was rejected (p_n if none
    of that is over 0).  Products and sums are 64 bits.

    Weights that are NaN or below 0 count as 0; a row without any weight gives
    token -1.  A token outside the vocabulary is rejected.  T may be 0: a token
    is drawn for each sequence."""
    if draft.dim() != 2 or target_probs.dim() != 3:
        raise ValueError(f"draft must be (B, T) and target_probs (B, T + 1, V); got {tuple(draft.shape)} / "
                         f"{tuple(target_probs.shape)}")
    B, T = draft.shape
    V = target_probs.shape[2]
    if draft.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"draft must be int32 or int64 (got {draft.dtype})")
    if tuple(target_probs.shape) != (B, T + 1, V) or V == 0:
        raise ValueError(f"target_probs must be ({B}, {T + 1}, V), V not 0; got {tuple(target_probs.shape)}")
    if target_probs.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"verify_drafts: fp32, fp16 or bf16 probabilities (got {target_probs.dtype})")
    if draft_probs is not None and (tuple(draft_probs.shape) != (B, T, V) or draft_probs.dtype != target_probs.dtype):
        raise ValueError(f"draft_probs must be ({B}, {T}, {V}) {target_probs.dtype}; got {tuple(draft_probs.shape)} "
                         f"{draft_probs.dtype}")
    if tuple(u.shape) != (B, T) or tuple(u_next.shape) != (B,) or u.dtype != torch.float32 or u_next.dtype != torch.float32:
        raise ValueError(f"u and u_next must be fp32 ({B}, {T}) and ({B},); got {tuple(u.shape)} {u.dtype}, "
                         f"{tuple(u_next.shape)} {u_next.dtype}")
    dev = _lib.same_device("verify_drafts", target_probs, draft, u, u_next, draft_probs)
    tokens = target_probs.new_empty((B, T + 1), dtype=torch.int32)
    accepted = target_probs.new_empty(B, dtype=torch.int32)
    if B:
        def packed(x):  # the values of a row next to each other
            return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()
        draft, p, u, u_next = packed(draft.to(torch.int64)), packed(target_probs), packed(u), packed(u_next)
        q = None if draft_probs is None or T == 0 else packed(draft_probs)
        pp = _lib.verify_params(B, T, V, _lib.DTYPE_CODE[p.dtype], *p.stride()[:2],
                               *((0, 0) if q is None else q.stride()[:2]), draft.stride(0), u.stride(0))
        lib = _lib.load()
        nbytes = lib.carekv_verify_drafts_workspace_bytes(pp)
        if nbytes < 0:
            _lib.check(-1, "carekv_verify_drafts_workspace_bytes")
        ws = p.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        ct = _lib.row_counts(counts, B, dev, "counts")
        _lib.call(dev, "carekv_verify_drafts", lib.carekv_verify_drafts, pp, draft.data_ptr(), p.data_ptr(),
                  None if q is None else q.data_ptr(), u.data_ptr(), u_next.data_ptr(),
                  None if ct is None else ct.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
                  None if ws is None else ws.data_ptr(), nbytes)
    return VerifiedDrafts(tokens, accepted)
