"""Operators for serving on pages of 4-bit rows, as timed cases: new tokens are
turned to their positions and written to pages, read back by attention that
may be bounded to a window and a few first tokens, and drafted tokens are
verified against the model's probabilities.

Kinds of case:

* ``append``  k and v of new tokens into a sequence's pages, q and k under
              rotary positions on the way (``append_pages``)
* ``paged``   attention of a sequence's last rows over its pages
              (``paged_attention``)
* ``window``  attention of (ragged) prompts and single tokens over 16-bit rows,
              inside a window and over the first tokens (``window_attention``)
* ``verify``  drafted tokens accepted or replaced (``verify_drafts``)

Where ``own`` is false, ``run`` computes them with elementary torch
operations in 32 bits (rotated heads, which are rounded to 4 bits afterwards,
and sums of probabilities, which are compared with a random number, in 64);
where it is true, it makes a user's calls of ``care_kv``.  ``exact`` evaluates
the definitions in 64 bits.

A page holds 16 tokens of a sequence.  A row of it stands, in groups of 32
values, for half(c s) with s = half(max|x| / 7) and c = clamp(round(half(x /
s)), -8, 7) of the fp16 values x.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_DIR = os.path.join(ROOT, "care-kv-sparse-residual-correction-for-low-bit-kv-cache-quantization_amd")
DEV = "cuda"
F16, F32, F64 = torch.float16, torch.float32, torch.float64
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}
PAGE, GROUP = 16, 32


def _care_kv():
    if PKG_DIR not in sys.path:
        sys.path.insert(1, PKG_DIR)
    import care_kv
    return care_kv


# ---------------------------------------------------------------- cases
def listed():
    return [
        # The next token of one chat on a 1.1B model: a launch's latency counts.
        dict(kind="append", name="append b1 t1 32q/4kv d64", B=1, T=1, Hq=32, Hkv=4, D=64, R=64, layout="half",
             base=10000.0, start=2303, offset=0, ragged=False, dtype="fp16"),
        # Up to four drafted tokens and the one before them, for 64 sequences of a 7B grouped-query model that
        # turns half of each head.
        dict(kind="append", name="append b64 t5 32q/8kv d128 r64", B=64, T=5, Hq=32, Hkv=8, D=128, R=64,
             layout="interleaved", base=10000.0, start=4000, offset=0, ragged=True, dtype="bf16"),
        # Four 8K prompts of a 13B multi-head model behind a text far before them, whose attention runs over the
        # rounded rows.
        dict(kind="append", name="append b4 t8192 40q/40kv d128", B=4, T=8192, Hq=40, Hkv=40, D=128, R=128,
             layout="half", base=500000.0, start=0, offset=100000, ragged=False, dtype="fp16"),
        # The next token of one chat on a 1.1B model.
        dict(kind="paged", name="paged b1 t1 n2303 32q/4kv d64", B=1, T=1, N=2303, Hq=32, Hkv=4, D=64, window=0,
             sink=0, ragged=False, dtype="fp16"),
        # Four drafted tokens and the one before them on 16 ragged contexts, of which a window and the first tokens
        # stay visible.
        dict(kind="paged", name="paged b16 t5 n8191 32q/8kv d128 w4096", B=16, T=5, N=8191, Hq=32, Hkv=8, D=128,
             window=4096, sink=4, ragged=True, dtype="bf16"),
        # A batch of 64 long contexts, one token each, on a 7B grouped-query model.
        dict(kind="paged", name="paged b64 t1 n32768 32q/8kv d128", B=64, T=1, N=32768, Hq=32, Hkv=8, D=128,
             window=0, sink=0, ragged=False, dtype="fp16"),
        # The next 512 tokens of two long prompts of a 13B multi-head model, of which 16K are in the cache.
        dict(kind="paged", name="paged b2 t512 n16896 40q/40kv d128", B=2, T=512, N=16896, Hq=40, Hkv=40, D=128,
             window=0, sink=0, ragged=False, dtype="fp16"),
        # One token of one sequence on the unrounded rows of a long chat, through a window.
        dict(kind="window", name="window b1 q1 n4097 w1024 32q/4kv d64", B=1, Tq=1, Tk=4097, Hq=32, Hkv=4, D=64,
             window=1024, sink=4, ragged=False, dtype="fp16"),
        # Eight ragged prompts just short of 2K on a 7B grouped-query model.
        dict(kind="window", name="window b8 q2047 n2047 w512 32q/8kv d128", B=8, Tq=2047, Tk=2047, Hq=32, Hkv=8,
             D=128, window=512, sink=4, ragged=True, dtype="bf16"),
        # Four 8K prompts on a 13B multi-head model.
        dict(kind="window", name="window b4 q8192 n8192 w4096 40q/40kv d128", B=4, Tq=8192, Tk=8192, Hq=40, Hkv=40,
             D=128, window=4096, sink=4, ragged=False, dtype="fp16"),
        # Four tokens guessed from the text before them, for one chat: a launch's latency counts.
        dict(kind="verify", name="verify b1 t4 v32000 guessed", B=1, T=4, V=32000, guessed=True, ragged=False,
             dtype="fp32"),
        # Eight drafted tokens of 128 sequences over a large vocabulary.
        dict(kind="verify", name="verify b128 t8 v131071", B=128, T=8, V=131071, guessed=False, ragged=True,
             dtype="fp32"),
    ]


HEADS = ((32, 4, 64), (32, 8, 128), (32, 32, 128), (40, 40, 128), (8, 1, 64), (6, 2, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "paged", "paged", "window", "verify"))
    if kind == "verify":
        return dict(kind=kind, B=_log(rng, 1, 128), T=rng.randint(0, 8), V=_log(rng, 100, 131071),
                    guessed=rng.random() < 0.3, ragged=rng.random() < 0.5, dtype=rng.choice(("fp32", "fp32", "bf16")))
    Hq, Hkv, D = rng.choice(HEADS)
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "append":
        B = _log(rng, 1, 64)
        T = rng.choice((1, _log(rng, 2, 8), _log(rng, 9, 8192)))
        T = max(1, min(T, 4 * 8192 * 40 // (B * Hq)))
        return dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, R=rng.choice((D, D, D // 2, D // 4)),
                    layout=rng.choice(("half", "interleaved")), base=float(rng.choice((10000, 500000))),
                    start=_log(rng, 1, 4096) - 1, offset=rng.choice((0, _log(rng, 1, 1 << 20))),
                    ragged=rng.random() < 0.5, dtype=dtype)
    if kind == "paged":
        B = _log(rng, 1, 64)
        N = _log(rng, 1, 32768)
        while B * N * Hkv * D > 64 * 32768 * 8 * 128:
            B //= 2
        T = min(N, rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 9, 512))))
        while T > 1 and B * Hq * T * N * D > 2 * 40 * 512 * 16896 * 128:
            T //= 2
        return dict(kind=kind, B=B, T=T, N=N, Hq=Hq, Hkv=Hkv, D=D, window=rng.choice((0, _log(rng, 1, N))),
                    sink=rng.choice((0, 4, 33)), ragged=rng.random() < 0.5, dtype=dtype)
    B = _log(rng, 1, 16)
    Tk = _log(rng, 1, 8192)
    Tq = min(Tk, rng.choice((1, _log(rng, 2, 64), Tk, Tk)))
    while B > 1 and B * Hq * Tq * Tk * D > 2 * 40 * 8192 * 8192 * 128:
        B //= 2
    return dict(kind=kind, B=B, Tq=Tq, Tk=Tk, Hq=Hq, Hkv=Hkv, D=D, window=rng.choice((0, _log(rng, 1, Tk), 512)),
                sink=rng.choice((0, 4, 33)), ragged=rng.random() < 0.5, dtype=dtype)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _keys(shape, gen, u):
    """Keys as a cache meets them: two strong channels, and one row in 64 that many queries look for (u)."""
    k = torch.randn(*shape, generator=gen, device=DEV)
    k[..., :2] *= 4.0
    hot = torch.rand(*shape[:-1], 1, generator=gen, device=DEV) < 1 / 64
    return k + hot * (0.75 * u)


def _ints(lo, hi, n, gen):
    return torch.randint(lo, hi + 1, (n,), generator=gen, device=DEV, dtype=torch.int32)


def _table(B, pages, gen):
    """Every sequence's pages, anywhere in the pool."""
    return torch.randperm(B * pages, generator=gen, device=DEV).view(B, pages).to(torch.int32)


def _inputs(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    B = case["B"]
    if case["kind"] == "verify":
        T, V = case["T"], case["V"]
        # a peaked target and a draft of the same model made blurred, drafted tokens sampled from the draft
        logits = 2.5 * torch.randn(B, T + 1, V, generator=g, device=DEV)
        near = logits[:, :T] + 0.5 * torch.randn(B, T, V, generator=g, device=DEV)
        p, q = torch.softmax(logits, -1), torch.softmax(near, -1)
        if T:
            pick = torch.rand(B, T, 1, generator=g, device=DEV)
            draft = (torch.cumsum(q, -1) < pick).sum(-1).clamp_(max=V - 1)
        else:
            draft = torch.zeros(B, 0, dtype=torch.int64, device=DEV)
        counts = _ints(0, T, B, g) if case["ragged"] else None
        return dict(draft=draft, p=p.to(dt), q=None if case["guessed"] else q.to(dt), counts=counts,
                    u=torch.rand(B, T, generator=g, device=DEV), u_next=torch.rand(B, generator=g, device=DEV))
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    u = torch.randn(D, generator=g, device=DEV)
    if case["kind"] == "append":
        T = case["T"]
        # projections (B, T, heads, D) seen as heads
        q = torch.randn(B, T, Hq, D, generator=g, device=DEV).to(dt).transpose(1, 2)
        k = _keys((B, T, Hkv, D), g, u).to(dt).transpose(1, 2)
        v = torch.randn(B, T, Hkv, D, generator=g, device=DEV).to(dt).transpose(1, 2)
        start = _ints(case["start"] // 2, case["start"], B, g)
        counts = _ints(1, T, B, g) if case["ragged"] else None
        at = (start.long()[:, None] + torch.arange(T, device=DEV) + case["offset"]) if case["offset"] else None
        return dict(q=q, k=k, v=v, start=start, counts=counts, positions=at,
                    table=_table(B, -(-(case["start"] + T) // PAGE), g))
    if case["kind"] == "paged":
        T, N = case["T"], case["N"]
        q = (torch.randn(B, T, Hq, D, generator=g, device=DEV) + 0.25 * u).to(dt).transpose(1, 2)
        k = torch.empty(B, Hkv, N, D, dtype=F16, device=DEV)
        for b in range(B):
            k[b] = _keys((Hkv, N, D), g, u)
        v = torch.randn(B, Hkv, N, D, generator=g, device=DEV, dtype=F16)
        lengths, rows = torch.full((B,), N, dtype=torch.int32, device=DEV), None
        if case["ragged"]:
            rows = _ints(1, T, B, g)
            lengths = _ints(max(T, N // 3), N, B, g)
            lengths[0] = N
        return dict(q=q, k=k, v=v, lengths=lengths, rows=rows, table=_table(B, -(-N // PAGE), g))
    Tq, Tk = case["Tq"], case["Tk"]
    q = (torch.randn(B, Hq, Tq, D, generator=g, device=DEV) + 0.25 * u).to(dt)
    k = _keys((B, Hkv, Tk, D), g, u).to(dt)
    v = torch.randn(B, Hkv, Tk, D, generator=g, device=DEV).to(dt)
    lengths = None
    if case["ragged"]:  # right-padded: row i of q and of k are one token where Tq = Tk, else q's rows are the last
        lengths = _ints(max(Tq if Tq < Tk else 1, Tk // 3), Tk, B, g)
        lengths[0] = Tk
    return dict(q=q, k=k, v=v, lengths=lengths)


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["kind"] == "append":
        if own:
            state["plan"] = _care_kv().rotary_plan(case["R"], case["base"], layout=case["layout"], device=DEV)
            state["pages"] = _care_kv().int4_pages(state["table"].numel(), case["Hkv"], case["D"], device=DEV)
        else:
            state["plan"] = case["base"] ** (-torch.arange(0, case["R"], 2, dtype=F64, device=DEV) / case["R"])
            n, H, D = state["table"].numel(), case["Hkv"], case["D"]
            state["pages"] = [torch.zeros(n, H, PAGE, w, dtype=t, device=DEV)
                              for t, w in ((torch.uint8, D // 2), (F16, D // GROUP)) for _ in "kv"]
    if case["kind"] == "paged":
        k, v, table, B = state.pop("k"), state.pop("v"), state["table"], case["B"]
        if own:
            care_kv = _care_kv()
            state["pages"] = care_kv.int4_pages(table.numel(), case["Hkv"], case["D"], device=DEV)
            care_kv.append_pages(state["pages"], table, 0, k, v)
        else:
            n, H, D = table.shape[1], case["Hkv"], case["D"]
            state["pages"] = [torch.zeros(B * n, H, PAGE, w, dtype=t, device=DEV)
                              for t, w in ((torch.uint8, D // 2), (F16, D // GROUP)) for _ in "kv"]
            for b in range(B):
                for i, x in enumerate((k, v)):
                    x = torch.nn.functional.pad(x[b], (0, 0, 0, n * PAGE - case["N"]))
                    c, s = _codes(x)
                    for to, part in ((i, c), (2 + i, s)):
                        state["pages"][to][table[b].long()] = part.view(H, n, PAGE, -1).transpose(0, 1)
    return state


# ---------------------------------------------------------------- plain forms
def _codes(x):
    """fp16 rows as bytes of two codes, the lower place in the low bits, and their groups' scales."""
    w = x.to(F32).unflatten(-1, (-1, GROUP))
    s = (w.abs().amax(-1) / 7.0).to(F16)
    c = (w / s.to(F32)[..., None]).to(F16).to(F32).nan_to_num(nan=0.0).round().clamp(-8, 7).flatten(-2)
    c = c.to(torch.int16) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), s


def _values(c, s):
    """What codes and scales stand for, fp16 values in 32 bits."""
    lo, hi = (c & 15).to(torch.int8), (c >> 4).to(torch.int8)
    w = torch.stack((lo, hi), -1).flatten(-2)
    w = torch.where(w > 7, w - 16, w).to(F32).unflatten(-1, (-1, GROUP))
    return (w * s.to(F32)[..., None]).flatten(-2).to(F16).to(F32)


def _turn(x, angles, layout, R):
    """Heads (B, H, T, D) under angles (B, 1, T, R / 2), in 64 bits, rounded to 32."""
    w = x.to(F64)
    c, s = torch.cos(angles), torch.sin(angles)
    if layout == "half":
        x1, x2 = w[..., :R // 2], w[..., R // 2:R]
        y = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s, w[..., R:]), dim=-1)
    else:
        x1, x2 = w[..., 0:R:2], w[..., 1:R:2]
        y = torch.cat((torch.stack((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).flatten(-2), w[..., R:]), dim=-1)
    return y.to(F32)


def _plain_append(state):
    case, q = state["case"], state["q"]
    B, T, H, D = case["B"], case["T"], case["Hkv"], case["D"]
    place = state["start"].long()[:, None] + torch.arange(T, device=DEV)
    at = place if state["positions"] is None else state["positions"]
    angles = at.to(F64)[:, None, :, None] * state["plan"]
    turned = _turn(q, angles, case["layout"], case["R"]).to(q.dtype).contiguous()
    rows = [_turn(state["k"], angles, case["layout"], case["R"]).to(F16), state["v"].to(F16)]
    n = T if state["counts"] is None else state["counts"].long()[:, None]
    new = (torch.arange(T, device=DEV) < n).expand(B, T)
    page = torch.gather(state["table"].long(), 1, place // PAGE)[new]
    hats = []
    for i, x in enumerate(rows):
        c, s = _codes(x)
        state["pages"][i][page, :, (place % PAGE)[new]] = c.transpose(1, 2)[new]
        state["pages"][2 + i][page, :, (place % PAGE)[new]] = s.transpose(1, 2)[new]
        hats.append((_values(c, s) * new[:, None, :, None]).to(F16))
    return [turned, *hats]


def _attend(q, k, v, see):
    """q (B, Hq, T, D), k and v (B, Hkv, N, D) in 32 bits, see (B, T, N): output and log-sum-exp of each row."""
    B, Hq, T, D = q.shape
    H, N = k.shape[1:3]
    s = torch.matmul(q.to(F32).reshape(B, H, -1, D), k.transpose(2, 3).contiguous()) / math.sqrt(D)
    s = s.view(B, H, -1, T, N).masked_fill_(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = torch.exp(s.sub_(m))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, -1, N), v).view(B, H, -1, T, D) / torch.where(z > 0, z, 1.0)
    return o.reshape(q.shape).to(q.dtype), (m + torch.log(z)).reshape(B, Hq, T)


def _see(pos, there, lengths, N, window, sink):
    """(B, T, N): row at pos (B, T) sees key j.  there (B, T): rows that are no padding."""
    j, at = torch.arange(N, device=DEV), pos[..., None]
    see = (j <= at) & (j < lengths[:, None, None]) & there[..., None]
    return see & ((j > at - window) | (j < sink)) if window else see


def _places(state):
    """(positions, rows that are no padding, lengths) of the query rows of an attention case."""
    case = state["case"]
    B = case["B"]
    if case["kind"] == "paged":
        T, n = case["T"], state["lengths"].long()
        rows = torch.full_like(n, T) if state["rows"] is None else state["rows"].long()
    else:
        T, N = case["Tq"], case["Tk"]
        n = torch.full((B,), N, device=DEV) if state["lengths"] is None else state["lengths"].long()
        rows = n if T == N else torch.full_like(n, T)
    t = torch.arange(T, device=DEV)
    return (n - rows)[:, None] + t, t < rows[:, None], n


def _plain_paged(state):
    case = state["case"]
    table = state["table"].long()
    kc, vc, ks, vs = (x[table].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :case["N"]] for x in state["pages"])
    pos, there, n = _places(state)
    see = _see(pos, there, n, case["N"], case["window"], case["sink"])
    return _attend(state["q"], _values(kc, ks), _values(vc, vs), see)


def _plain_window(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    pos, there, n = _places(state)
    step = max(1, (1 << 32) // (case["Hq"] * case["Tq"] * case["Tk"]))  # sequences whose scores fit at once
    parts = []
    for b in range(0, case["B"], step):
        e = slice(b, b + step)
        see = _see(pos[e], there[e], n[e], case["Tk"], case["window"], case["sink"])
        parts.append(_attend(q[e], k[e].to(F32), v[e].to(F32), see))
    return tuple(torch.cat(x) for x in zip(*parts))


def _plain_verify(state):
    draft, p, q = state["draft"], state["p"], state["q"]
    B, T, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    n = torch.full((B,), T, device=DEV) if state["counts"] is None else state["counts"].long()
    px = torch.gather(p[:, :T], 2, draft[..., None])[..., 0].to(F64)
    qx = torch.ones_like(px) if q is None else torch.gather(q, 2, draft[..., None])[..., 0].to(F64)
    good = (state["u"].to(F64) * qx < px) & (torch.arange(T, device=DEV) < n[:, None])
    kept = torch.cumprod(good.long(), 1).sum(1)
    b = torch.arange(B, device=DEV)
    w = p[b, kept].to(F64)
    if T:
        at = kept.clamp(max=T - 1)
        if q is None:
            less = torch.zeros_like(w).scatter_(1, draft[b, at][:, None], float("inf"))
        else:
            less = q[b, at].to(F64)
        rest = (w - less).clamp_(min=0.0)
        w = torch.where(((kept < n) & (rest.sum(1) > 0))[:, None], rest, w)
    run_sum = torch.cumsum(w, 1)
    token = (run_sum <= state["u_next"].to(F64)[:, None] * run_sum[:, -1:]).sum(1)
    t = torch.arange(T + 1, device=DEV)
    out = torch.cat((draft, draft.new_zeros(B, 1)), 1)
    out = torch.where(t < kept[:, None], out, torch.where(t == kept[:, None], token[:, None], -1))
    return out.to(torch.int32), kept.to(torch.int32)


PLAIN = dict(append=_plain_append, paged=_plain_paged, window=_plain_window, verify=_plain_verify)


def run(state):
    case = state["case"]
    if not own:
        return PLAIN[case["kind"]](state)
    care_kv = _care_kv()
    if case["kind"] == "append":
        return list(care_kv.append_pages(state["pages"], state["table"], state["start"], state["k"], state["v"],
                                         q=state["q"], plan=state["plan"], positions=state["positions"],
                                         counts=state["counts"], return_hat=True))
    if case["kind"] == "paged":
        return care_kv.paged_attention(state["q"], state["pages"], state["table"], state["lengths"],
                                       q_lengths=state["rows"], window=case["window"] or None, sink=case["sink"],
                                       return_lse=True)
    if case["kind"] == "window":
        return care_kv.window_attention(state["q"], state["k"], state["v"], window=case["window"] or None,
                                        sink=case["sink"], lengths=state["lengths"], return_lse=True)
    return tuple(care_kv.verify_drafts(state["draft"], state["p"], state["u"], state["u_next"],
                                       draft_probs=state["q"], counts=state["counts"]))


# ---------------------------------------------------------------- what a pass cannot do without
def _pairs(T, N, window, sink):
    """Pairs of the last T of N positions and the keys that they see, and keys that any of them sees."""
    total = sum(min(t + 1, window + min(sink, max(0, t + 1 - window))) if window else t + 1 for t in range(N - T, N))
    seen = min(N, window + T - 1 + min(sink, max(0, N - T + 1 - window))) if window else N
    return total, seen


def work(case):
    e, B = SIZES[case["dtype"]], case["B"]
    if case["kind"] == "verify":
        rows = 1 if case["guessed"] else 2
        return dict(bytes=B * (rows * case["V"] * e + case["T"] * (8 + 4 + 2 * e + 4) + 12), flops=3 * B * case["V"])
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    packed = D // 2 + D // GROUP * 2
    if case["kind"] == "append":
        n = B * (case["T"] if not case["ragged"] else (case["T"] + 1) // 2)
        io = 2 * Hq * D * e * B * case["T"] + n * Hkv * 2 * (D * e + packed)
        io += B * case["T"] * Hkv * 2 * D * 2  # the new rows as the values they stand for
        return dict(bytes=io, flops=3 * n * (Hq + Hkv) * case["R"] + 4 * n * Hkv * D)
    if case["kind"] == "paged":
        T, N = case["T"], case["N"] if not case["ragged"] else max(case["T"], 2 * case["N"] // 3)
        pairs, seen = _pairs(T, N, case["window"], case["sink"])
        return dict(bytes=B * (Hq * case["T"] * (2 * D * e + 4) + seen * Hkv * 2 * packed), flops=4 * B * Hq * D * pairs)
    Tq, Tk = case["Tq"], case["Tk"]
    N = Tk if not case["ragged"] else max(1, 2 * Tk // 3)
    T = N if Tq == Tk else min(Tq, N)
    pairs, seen = _pairs(T, N, case["window"], case["sink"])
    return dict(bytes=B * (Hq * Tq * (2 * D * e + 4) + seen * Hkv * 2 * D * e), flops=4 * B * Hq * D * pairs)


# ---------------------------------------------------------------- 64 bits
def _round4(x):
    """The values that a row of fp16 values is kept as, group by group."""
    g = x.to(F64).reshape(*x.shape[:-1], -1, GROUP)
    scale = (g.abs().max(-1, keepdim=True).values / 7).to(F32).to(F16).to(F64)
    ratio = torch.where(scale > 0, g / torch.where(scale > 0, scale, 1.0), 0.0).to(F32).to(F16).to(F64)
    return (torch.round(ratio).clamp(-8, 7) * scale).to(F32).to(F16).to(F64).reshape(x.shape)


def exact(case, seed):
    d = _inputs(case, seed)
    B = case["B"]
    if case["kind"] == "verify":
        import numpy as np
        T, V = case["T"], case["V"]
        draft, u, un = d["draft"].cpu().numpy(), d["u"].cpu().double().numpy(), d["u_next"].cpu().double().numpy()
        out, took = np.full((B, T + 1), -1, dtype=np.int32), np.zeros(B, dtype=np.int32)
        for b in range(B):
            many = T if d["counts"] is None else int(d["counts"][b])
            n, w = 0, None
            while n < many:
                x = int(draft[b, n])
                p = d["p"][b, n].double().cpu().numpy()
                q = np.eye(1, V, x)[0] if d["q"] is None else d["q"][b, n].double().cpu().numpy()
                if not u[b, n] * q[x] < p[x]:
                    w = np.maximum(p - q, 0.0)
                    if d["q"] is None:
                        w = p.copy()
                        w[x] = 0.0
                    if not w.sum() > 0:
                        w = p
                    break
                out[b, n] = x
                n += 1
            if w is None:
                w = d["p"][b, n].double().cpu().numpy()
            sums = np.cumsum(w)
            out[b, n], took[b] = int(np.searchsorted(sums, un[b] * sums[-1], side="right")), n
        return torch.from_numpy(out).to(DEV), torch.from_numpy(took).to(DEV)
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    if case["kind"] == "append":
        T, r = case["T"], case["R"]
        at = d["start"].to(F64)[:, None] + torch.arange(T, dtype=F64, device=DEV) + case["offset"]
        f = torch.tensor([case["base"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=F64, device=DEV)
        z = torch.polar(torch.ones(B, 1, T, r // 2, dtype=F64, device=DEV), at[:, None, :, None] * f)

        def turn(x):
            y = x.to(F64).clone()
            a, b = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            w = torch.complex(y[..., a].contiguous(), y[..., b].contiguous()) * z
            y[..., a], y[..., b] = w.real, w.imag
            return y
        out = [turn(d["q"])]
        for x in (turn(d["k"]), d["v"].to(F64)):
            x = _round4(x.to(F32).to(F16))
            for b in range(B if d["counts"] is not None else 0):
                x[b, :, int(d["counts"][b]):] = 0
            out.append(x)
        return out
    N = case["N"] if case["kind"] == "paged" else case["Tk"]
    o = torch.zeros(d["q"].shape, dtype=F64, device=DEV)
    lse = torch.full(d["q"].shape[:3], -math.inf, dtype=F64, device=DEV)
    T = d["q"].shape[2]
    for b in range(B):
        n = N if d["lengths"] is None else int(d["lengths"][b])
        if case["kind"] == "paged":
            rows = T if d["rows"] is None else int(d["rows"][b])
        else:
            rows = n if T == N else T
        key, at = torch.arange(n, device=DEV), torch.arange(n - rows, n, device=DEV)[:, None]
        hidden = key > at
        if case["window"]:
            hidden = hidden | ((at - key >= case["window"]) & (key >= case["sink"]))
        for h in range(Hkv):
            k, v = d["k"][b, h, :n], d["v"][b, h, :n]
            k, v = (_round4(k), _round4(v)) if case["kind"] == "paged" else (k.to(F64), v.to(F64))
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                s = torch.mm(d["q"][b, i, :rows].to(F64), k.t()) * D ** -0.5
                s = s.masked_fill(hidden, -math.inf)
                o[b, i, :rows] = torch.mm(torch.softmax(s, 1), v)
                lse[b, i, :rows] = torch.logsumexp(s, 1)
    return o, lse
