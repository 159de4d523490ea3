"""Heads under rotary positions given as positions (no reference counterpart
beyond the fp16 tables of ``CAREKVLayer``): both pair layouts, a part of the
head, contexts stretched past the trained length.

For pair i of a head's first ``rotary_dim`` values at position p, with
t = p f_i and the plan's factor a::

    y1 = a (x1 cos t - x2 sin t)        y2 = a (x2 cos t + x1 sin t)

``layout="half"`` pairs (i, i + rotary_dim / 2), ``"interleaved"`` (2i, 2i+1).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib

LAYOUTS = ("half", "interleaved")
SCALINGS = ("none", "linear", "ntk", "yarn", "bands")


@dataclass(frozen=True)
class RotaryPlan:
    """What ``rotate_heads`` turns by: made once by ``rotary_plan`` and kept."""
    rotary_dim: int
    layout: str
    freqs: torch.Tensor  # fp64 (rotary_dim / 2,), radians per position, on the device
    scale: float         # factor on the rotated values

    def __post_init__(self):
        if self.layout not in LAYOUTS:
            raise ValueError(f"layout={self.layout!r} not in {LAYOUTS}")
        if self.rotary_dim < 2 or self.rotary_dim % 2 or self.freqs.dtype != torch.float64 or \
                self.freqs.shape != (self.rotary_dim // 2,) or not self.freqs.is_contiguous():
            raise ValueError(f"a plan needs an even rotary_dim and rotary_dim / 2 packed fp64 angles (got "
                             f"{self.rotary_dim}, {tuple(self.freqs.shape)} {self.freqs.dtype})")


def rotary_plan(rotary_dim: int, base: float = 10000.0, *, layout: str = "half", scaling: str = "none",
                factor: float = 1.0, original_len: Optional[int] = None, scale: Optional[float] = None,
                fast_turns: float = 32.0, slow_turns: float = 1.0, low_band: float = 1.0, high_band: float = 4.0,
                device=None) -> RotaryPlan:
    """The angles per position f_i = base^(-2i / rotary_dim), i < rotary_dim / 2,
    stretched for contexts ``factor`` >= 1 times the trained length
    ``original_len``:

    * ``linear``: f_i / factor;
    * ``ntk``: the base times factor^(rotary_dim / (rotary_dim - 2)), which
      keeps the fastest pair and stretches the slowest by factor;
    * ``yarn``: pairs that turn more than ``fast_turns`` times over
      original_len kept, those that turn less than ``slow_turns`` times
      divided by factor, a linear ramp over the pair index between; the
      rotated values times 0.1 ln(factor) + 1;
    * ``bands``: the same by wavelength, kept below original_len / high_band,
      divided above original_len / low_band, between them mixed linearly in
      original_len / wavelength.

    ``scale`` overrides the factor on the rotated values."""
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"rotary_dim must be even and positive (got {rotary_dim})")
    if layout not in LAYOUTS:
        raise ValueError(f"layout={layout!r} not in {LAYOUTS}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling={scaling!r} not in {SCALINGS}")
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"base must be above 1 and factor at least 1 (got {base}, {factor})")
    if scaling in ("yarn", "bands") and (original_len is None or original_len <= 0):
        raise ValueError(f"scaling={scaling!r} needs original_len")
    if scaling == "ntk" and r < 4:
        raise ValueError("scaling='ntk' needs rotary_dim of at least 4")
    if scaling == "yarn" and not fast_turns > slow_turns > 0:
        raise ValueError("yarn needs fast_turns > slow_turns > 0")
    if scaling == "bands" and not high_band > low_band > 0:
        raise ValueError("bands needs high_band > low_band > 0")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    i = torch.arange(0, r, 2, dtype=torch.float64)
    b = base * factor ** (r / (r - 2)) if scaling == "ntk" else base
    f = b ** (-i / r)
    amp = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair(turns):  # the pair index that turns so often over original_len
            return r * math.log(original_len / (2 * math.pi * turns)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast_turns)), 0), min(math.ceil(pair(slow_turns)), r - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - ramp) + f / factor * ramp
        amp = 0.1 * math.log(factor) + 1.0
    elif scaling == "bands":
        mix = ((original_len * f / (2 * math.pi) - low_band) / (high_band - low_band)).clamp(0.0, 1.0)
        f = f * mix + f / factor * (1.0 - mix)
    return RotaryPlan(r, layout, f.to(device), float(amp if scale is None else scale))


def rotate_heads(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, plan: RotaryPlan, *,
                 inverse: bool = False, out=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q (B, Hq, T, D) and k (B, Hkv, T, D) (or None) under the plan's rotary
    positions, in one launch; fp16, bf16 or fp32, any strides (a projection's
    (B, T, heads, D) seen through ``transpose(1, 2)`` is read in place).
    (Hq, T, D) heads of one sequence work alike.  positions: int32 or int64
    device tensor (B, T), (1, T) or (T,), any values (negative, far, repeated).

    Angles are reduced in 64 bits and products taken in fp32, rounded once.
    ``inverse`` turns back by the same angles (times the plan's scale): the
    gradient of the forward call, and with scale 1 its inverse.  ``out``: (q_out,
    k_out), which may be (q, k) themselves; by default new contiguous tensors.
    The results carry no autograd history."""
    if out is not None and (len(out) != 2 or out[0] is None or (out[1] is None) != (k is None)):
        raise ValueError("out must be (q_out, k_out), k_out None only without k")
    squeeze = q.dim() == 3
    if squeeze:
        qo, ko = (None, None) if out is None else out
        a, b = rotate_heads(q.unsqueeze(0), None if k is None else k.unsqueeze(0), positions, plan, inverse=inverse,
                            out=None if out is None else (qo.unsqueeze(0), None if ko is None else ko.unsqueeze(0)))
        return a[0], None if b is None else b[0]
    if q.dim() != 4:
        raise ValueError(f"q must be (B, heads, T, D) or (heads, T, D); got {tuple(q.shape)}")
    B, Hq, T, D = q.shape
    if q.dtype not in _lib.DTYPE_CODE:
        raise ValueError(f"rotate_heads: fp16, bf16 or fp32 heads (got {q.dtype})")
    if k is not None and (k.dim() != 4 or (k.shape[0], k.shape[2], k.shape[3]) != (B, T, D) or k.dtype != q.dtype):
        raise ValueError(f"k must be ({B}, heads, {T}, {D}) {q.dtype}; got {tuple(k.shape)} {k.dtype}")
    if D % 2 or plan.rotary_dim > D:
        raise ValueError(f"head_dim {D} must be even and at least rotary_dim {plan.rotary_dim}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64 (got {positions.dtype})")
    pos = positions.unsqueeze(0) if positions.dim() == 1 else positions
    if pos.dim() != 2 or pos.shape[0] not in (1, B) or pos.shape[1] != T:
        raise ValueError(f"positions must be ({B}, {T}), (1, {T}) or ({T},); got {tuple(positions.shape)}")
    if out is not None:
        _lib.check_out(out[0], q.shape, q.dtype, "q_out", q)
        if k is not None:
            _lib.check_out(out[1], k.shape, k.dtype, "k_out", k)
            if any(_lib.overlap(a, b) for a, b in ((out[0], out[1]), (out[0], k), (out[1], q))):
                raise ValueError("q_out must not overlap k or k_out, nor k_out q")
    dev = _lib.same_device("rotate_heads", q, k, positions, plan.freqs, *(() if out is None else out))
    if out is None:
        qo = q.new_empty(q.shape)
        ko = None if k is None else k.new_empty(k.shape)
    else:
        qo, ko = out
    pos = pos if pos.stride(1) == 1 or T == 1 else pos.contiguous()
    if q.stride(3) != 1:
        q = q.contiguous()
    sq, so = q.stride(), qo.stride()
    if k is None:
        hk, kp, kop, sk, sko = 0, None, None, (0, 0, 0), (0, 0, 0)
    else:
        if k.stride(3) != 1:
            k = k.contiguous()
        hk, kp, kop, sk, sko = k.shape[1], k.data_ptr(), ko.data_ptr(), k.stride(), ko.stride()
    pp = _lib.RotaryParams(B, T, Hq, hk, D, plan.rotary_dim, _lib.DTYPE_CODE[q.dtype], plan.layout == "interleaved",
                           bool(inverse), 64 if pos.dtype == torch.int64 else 32, plan.scale,
                           pos.stride(0) if pos.shape[0] > 1 else 0, *sq[:3], *sk[:3], *so[:3], *sko[:3])
    _lib.call(dev, "carekv_rotate_heads", _lib.load().carekv_rotate_heads, pp, q.data_ptr(), kp, pos.data_ptr(),
              plan.freqs.data_ptr(), qo.data_ptr(), kop)
    return qo, ko
