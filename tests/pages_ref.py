"""Plain forms for the tests of 4-bit pages and windowed attention, in 64 bits."""
import math

import torch

INF = float("inf")


def round4(x):
    """fp16 rows (.., D) -> (codes, scales, values), each from its definition; a group that is not finite: NaN."""
    w = x.double().unflatten(-1, (-1, 32))
    top = w.abs().amax(-1)
    top = torch.where(torch.isfinite(w).all(-1), top, math.nan)
    s = (top / 7).float().half()
    r = (w / s.double()[..., None]).float().half().double()
    c = torch.where(torch.isnan(r), 0.0, r.round().clamp(-8, 7))
    c = torch.where(torch.isnan(top)[..., None], 0.0, c)
    hat = (c * s.double()[..., None]).float().half()
    return c.flatten(-2), s, hat.flatten(-2)


def turn(x, positions, plan):
    """Heads (B, H, T, D) at positions (B or 1, T), in 64 bits, rounded to 32."""
    r = plan.rotary_dim
    t = positions.double()[:, None, :, None] * plan.freqs
    c, s = torch.cos(t) * plan.scale, torch.sin(t) * plan.scale
    y = x.double().clone()
    a, b = (slice(0, r // 2), slice(r // 2, r)) if plan.layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    x1, x2 = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    return y.float()


def unpack(pages, page, head):
    """(K codes, K scales, V codes, V scales) of a block, read byte by byte: (16, D), (16, D / 32)."""
    D = pages.head_dim
    raw = pages.data[page, head].cpu().tolist()
    G = D // 32
    kc, vc = torch.zeros(16, D), torch.zeros(16, D)

    def nibble(word, e):  # code e of eight: even ones in the low half of the word
        i = (e % 2) * 4 + e // 2
        return ((raw[4 * word + i // 2] >> (4 * (i % 2))) & 15) - 8

    for tok in range(16):
        for d in range(D):
            kc[tok, d] = nibble(tok * D // 8 + d // 8, d % 8)
            tile, c = d // 16, d % 16
            vc[tok, d] = nibble(4 * D + (tok // 4 * 16 + c) * G + tile // 2 - 2 * D, tile % 2 * 4 + tok % 4)
    half = torch.tensor(raw[16 * D:], dtype=torch.uint8).view(torch.float16)
    vs = half[:16 * G].view(4, G, 4).permute(0, 2, 1).reshape(16, G)
    ks = half[16 * G:].view(G, 16).t()
    return kc, ks, vc, vs


def sight(B, Tq, Tk, window, sink, lengths, q_lengths, q_start):
    """(B, Tq, Tk): row i sees key j."""
    see = torch.zeros(B, Tq, Tk, dtype=torch.bool, device="cuda")
    for b in range(B):
        n = max(0, min(Tk, lengths[b]))
        m = max(0, min(Tq, q_lengths[b]))
        base = n - m if q_start is None else q_start[b]
        p, j = base + torch.arange(m, device="cuda")[:, None], torch.arange(Tk, device="cuda")[None]
        ok = (j <= p) & (j < n)
        if window is not None:
            ok &= (j > p - window) | (j < sink)
        see[b, :m] = ok
    return see


def attend(q, k, v, see, scale=None, weights=None):
    """(o, lse, tolerance of o, of lse).  k and v (B, Hkv, N, D) as they are; weights: the type that the softmax's
    weights are rounded to for the second product.

    A logit is off by at most e = (D + 8) 2^-24 of the sum of its terms' magnitudes; a weight by that twice (its own and
    the reference's) and by half a step; fp16 weights below 2^-29 of the largest by up to 2^-40 of it; sums of n
    weights by n / 4 times 2^-24 (the terms of one lane in a row); the result is rounded, fp16 below 2^-14 to 2^-25."""
    B, Hq, T, D = q.shape
    G = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    weights = q.dtype if weights is None else weights
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -INF, dtype=torch.float64, device=q.device)
    tol, tl = torch.zeros_like(o), torch.zeros_like(lse)
    step, out = torch.finfo(weights).eps / 2, torch.finfo(q.dtype).eps / 2
    n = k.shape[2]
    for b in range(B):
        for h in range(Hq):
            if n == 0:
                continue
            x, y, z = q[b, h].double(), k[b, h // G].double(), v[b, h // G].double()
            m = see[b]
            some = m.any(0)
            y, z = (torch.where(some[:, None], w, 0.0) for w in (y, z))  # what no row sees
            s = (x @ y.t() * scale).masked_fill(~m, -INF)
            mag = (x.abs() @ y.abs().t()).masked_fill(~m, 0.0)
            e = torch.nan_to_num(mag).amax(1, keepdim=True) * abs(scale) * (D + 8) * 2.0 ** -24
            l = torch.logsumexp(s, 1)
            w = torch.where(m, torch.exp(s - torch.where(m.any(1), l, 0.0)[:, None]), 0.0)
            bad = ~torch.isfinite(z)
            zz = torch.where(bad, 0.0, z)
            y_o, y_m = w @ zz, w @ zz.abs()
            for j in torch.nonzero(bad.any(1)).flatten().tolist():  # the rows that see it alone
                y_o = torch.where(m[:, j:j + 1] & bad[j], y_o + w[:, j:j + 1] * z[j], y_o)
            o[b, h], lse[b, h] = y_o, l
            tol[b, h] = y_m * (step + 2 * e + 2.0 ** -18 + n / 4 * 2.0 ** -24) + y_o.abs() * out + n * 2.0 ** -40 * zz.abs().max()
            tl[b, h] = 2 * e[:, 0] + n / 4 * 2.0 ** -24 + (torch.nan_to_num(l, neginf=0.0).abs() + 32) * 2.0 ** -22
    if q.dtype == torch.float16:
        tol += 2.0 ** -25
    return o, lse, tol, tl


def check(got, ref):
    o, lse = got
    w_o, w_l, t_o, t_l = ref
    assert torch.equal(torch.isnan(o), torch.isnan(w_o)) and torch.equal(torch.isinf(o), torch.isinf(w_o))
    assert torch.equal(torch.isnan(lse), torch.isnan(w_l)) and torch.equal(torch.isinf(lse), torch.isinf(w_l))
    fine = torch.isfinite(w_o)
    over = ((o.double() - w_o).abs() / t_o.clamp(min=1e-300))[fine]
    assert not over.numel() or float(over.max()) <= 1.0, f"o off by {float(over.max()):.3g} of its tolerance"
    assert torch.equal(o[~fine & ~torch.isnan(w_o)].double(), w_o[~fine & ~torch.isnan(w_o)])
    fine = torch.isfinite(w_l)
    over = ((lse.double() - w_l).abs() / t_l.clamp(min=1e-300))[fine]
    assert not over.numel() or float(over.max()) <= 1.0, f"lse off by {float(over.max()):.3g} of its tolerance"
