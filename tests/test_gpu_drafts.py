"""verify_drafts against its definition, sequence by sequence in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _ref(draft, p, u, un, q=None, counts=None):
    """The definition; and how near the goal each drawn token's borders are, relative to the sum."""
    B, T = draft.shape
    V = p.shape[2]
    tokens, accepted, near = np.full((B, T + 1), -1, np.int64), np.zeros(B, np.int64), 1.0
    x = draft.cpu().numpy()
    P, U, N = p.double().cpu().numpy(), u.double().cpu().numpy(), un.double().cpu().numpy()
    Q = None if q is None else q.double().cpu().numpy()
    for b in range(B):
        count = T if counts is None else max(0, min(T, int(counts[b])))
        n, rest = 0, None
        while n < count:
            t = int(x[b, n])
            inside = 0 <= t < V
            if inside and U[b, n] * (1.0 if Q is None else Q[b, n, t]) < P[b, n, t]:
                tokens[b, n] = t
                n += 1
                continue
            if Q is None:
                rest = P[b, n].copy()
                if inside:
                    rest[t] = 0.0
            else:
                rest = P[b, n] - Q[b, n]
            break
        w = None if rest is None else np.where(rest > 0, rest, 0.0)
        if w is None or not w.sum() > 0:
            w = np.where(P[b, n] > 0, P[b, n], 0.0)
        accepted[b] = n
        s = np.cumsum(w)
        if s[-1] > 0:
            goal = N[b] * s[-1]
            past = np.nonzero(s > goal)[0]
            tokens[b, n] = past[0] if past.size else np.nonzero(w > 0)[0][-1]
            near = min(near, float(np.abs(s - goal).min() / s[-1])) if 0 < N[b] < 1 else near
    return tokens, accepted, near


def _check(got, ref):
    assert got.tokens.dtype == got.accepted.dtype == torch.int32
    np.testing.assert_array_equal(got.accepted.cpu().numpy(), ref[1])
    np.testing.assert_array_equal(got.tokens.cpu().numpy(), ref[0])


def _inputs(seed, B, T, V, dtype, blur=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    logits = 2 * r(B, T + 1, V)
    p, q = torch.softmax(logits, -1), torch.softmax(logits[:, :T] + blur * r(B, T, V), -1)
    draft = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, T) if T else torch.zeros(B, 0, dtype=torch.int64, device="cuda")
    u, un = torch.rand(B, T, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    return draft, p.to(dtype), u, un, q.to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (1, 4, 7), (3, 0, 100), (5, 3, 1000), (2, 8, 2048), (2, 2, 2049), (70, 5, 4097),
                                   (1, 4, 50001), (2, 70, 300), (300, 2, 33)])
def test_against_the_definition(dtype, B, T, V):
    import care_kv
    print(f"verify {dtype} B={B} T={T} V={V}", flush=True)
    draft, p, u, un, q = _inputs(V + T, B, T, V, dtype)
    counts = torch.arange(B, device="cuda") % (T + 2)
    for kw in (dict(draft_probs=q), dict(), dict(draft_probs=q, counts=counts), dict(counts=counts.int())):
        ref = _ref(draft, p, u, un, kw.get("draft_probs"), kw.get("counts"))
        assert ref[2] > 2.0 ** -45  # sums in another order agree on every token
        _check(care_kv.verify_drafts(draft, p, u, un, **kw), ref)
    got = care_kv.verify_drafts(draft.int(), p, u, un, draft_probs=q)
    for a, b in zip(got, care_kv.verify_drafts(draft, p, u, un, draft_probs=q)):
        assert torch.equal(a, b)


def test_borders():
    """Probabilities whose sums are exact: numbers on a border, 0, just below 1, 1 and beyond, NaN."""
    import care_kv
    V = 5000
    p = torch.zeros(1, 2, V, device="cuda")
    p[0, :, [3, 700, 2100, 4999]] = torch.tensor([0.25, 0.25, 0.375, 0.125], device="cuda")
    q = torch.zeros(1, 1, V, device="cuda")
    q[0, 0, [3, 700]] = 0.5
    one = lambda x: torch.tensor([x], device="cuda")  # noqa: E731
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for x, u, un, tokens in [
            (3, 0.5, 0.0, [2100, -1]), (3, 0.49999, 0.0, [3, 3]), (3, 0.49999, 0.25, [3, 700]), (3, 0.49999, 0.5, [3, 2100]),
            (3, 0.49999, 0.875, [3, 4999]), (3, 0.49999, below, [3, 4999]), (3, 0.49999, 1.0, [3, 4999]),
            (3, 0.49999, 7.0, [3, 4999]), (3, 0.49999, math.nan, [3, 3]), (3, 0.49999, -1.0, [3, 3]),
            (700, 0.9, 0.75, [4999, -1]), (700, 0.9, 0.7499, [2100, -1]), (5, 0.0, 0.5, [2100, -1]), (2100, 0.0, 0.1, [2100, 3]),
            (3, math.nan, 0.0, [2100, -1]), (-1, 0.0, 0.0, [2100, -1]), (V, 0.0, 0.8, [4999, -1]), (2 ** 40, 0.0, 0.8, [4999, -1])]:
        got = care_kv.verify_drafts(torch.tensor([[x]], device="cuda"), p, one([u]), one(un), draft_probs=q)
        assert got.tokens[0].tolist() == tokens, (x, u, un)
        assert int(got.accepted) == (tokens[1] != -1)
    guessed = care_kv.verify_drafts(torch.tensor([[2100]], device="cuda"), p, one([0.375]), one(0.5))
    assert guessed.tokens[0].tolist() == [700, -1]  # 0.25, 0.25, 0, 0.125: half of 0.625 is in the second
    guessed = care_kv.verify_drafts(torch.tensor([[2100]], device="cuda"), p, one([0.374]), one(0.5))
    assert guessed.tokens[0].tolist() == [2100, 2100]


def test_rows_without_weight():
    """Nothing left of p - q: p itself.  Rows of zeros and NaN: -1.  NaN and negative values count as 0."""
    import care_kv
    p = torch.zeros(4, 2, 3000, device="cuda")
    p[:, :, 2500] = 1.0
    q = p[:, :1].clone()
    p[1] = 0
    p[2] = math.nan
    p[3, :, :100] = math.nan
    p[3, :, 200:300] = -1.0
    u, un = torch.ones(4, 1, device="cuda"), torch.full((4,), 0.3, device="cuda")
    draft = torch.full((4, 1), 2500, device="cuda")
    got = care_kv.verify_drafts(draft, p, u, un, draft_probs=q)
    assert got.tokens.tolist() == [[2500, -1], [-1, -1], [-1, -1], [2500, -1]] and not got.accepted.any()


def test_strides_and_streams():
    import care_kv
    draft, p, u, un, q = _inputs(3, 4, 3, 900, F32)
    ref = care_kv.verify_drafts(draft, p, u, un, draft_probs=q)
    wide = torch.zeros(4, 4, 1000, device="cuda")
    wide[..., 50:950] = p
    apart = q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    forms = (draft.t().contiguous().t(), wide[..., 50:950], u.t().contiguous().t(), torch.stack((un, un), 1)[:, 0], apart)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = care_kv.verify_drafts(forms[0], forms[1], forms[2], forms[3], draft_probs=forms[4])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    one = p[:1].expand(4, -1, -1)  # one row of probabilities for all
    _check(care_kv.verify_drafts(draft, one, u, un, draft_probs=q), _ref(draft, one, u, un, q))


def test_distribution():
    """What comes out first is distributed as the model's row: of 20000 draws each share is within five deviations."""
    import care_kv
    V, B = 6, 20000
    g = torch.Generator(device="cuda").manual_seed(0)
    p = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.0, 0.3], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.1, 0.05, 0.4, 0.05], device="cuda")
    draft = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1)
    u, un = torch.rand(B, 1, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    got = care_kv.verify_drafts(draft, p.expand(B, 2, V), u, un, draft_probs=q.expand(B, 1, V))
    share = torch.bincount(got.tokens[:, 0].long(), minlength=V).double() / B
    assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt() + 1e-12).all()


def test_a_captured_call():
    import care_kv
    draft, p, u, un, q = _inputs(5, 6, 4, 5000, F32)
    call = lambda: care_kv.verify_drafts(draft, p, u, un, draft_probs=q)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(5):
        new = _inputs(60 + i, 6, 4, 5000, F32)
        for x, y in zip((draft, p, u, un, q), new):
            x.copy_(y)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,V", [(1, 2, 65537), (3, 3, 70001), (2, 1, 131071), (1, 1, 262145)])
def test_more_segments_than_lanes(dtype, B, T, V):
    """Vocabularies of more than 64 segments of 1024."""
    import care_kv
    print(f"verify {dtype} B={B} T={T} V={V}", flush=True)
    draft, p, u, un, q = _inputs(V + T, B, T, V, dtype)
    for kw in (dict(draft_probs=q), dict()):
        for next_at in (un, torch.full_like(un, 0.999), torch.full_like(un, 0.0), torch.full_like(un, 1.0)):
            ref = _ref(draft, p, u, next_at, kw.get("draft_probs"))
            assert ref[2] > 2.0 ** -45  # sums in another order agree on every token
            _check(care_kv.verify_drafts(draft, p, u, next_at, **kw), ref)


def test_borders_of_segments():
    """Weights that are exact, at the first and last places of segments, of lanes' runs and of lanes."""
    import care_kv
    V = 200000
    at = torch.tensor([0, 1023, 1024, 4095, 4096, 65535, 65536, 131071, V - 1], device="cuda")
    p = torch.zeros(1, 1, V, device="cuda")
    p[0, 0, at] = 0.125
    p[0, 0, 1] = math.nan
    p[0, 0, 130000] = -1.0
    none = torch.zeros(1, 0, device="cuda")
    for i, x in enumerate(at.tolist()):
        for share in (i / 9, (i + 0.5) / 9):
            un = torch.tensor([share], device="cuda")
            want = min(8, math.floor(float(un.double()) * 9))
            got = care_kv.verify_drafts(none.long(), p, none, un)
            assert got.tokens.tolist() == [[int(at[want])]], (i, share)


def test_a_captured_call_of_two_launches():
    import care_kv
    draft, p, u, un, q = _inputs(6, 3, 4, 70001, F32)
    call = lambda: care_kv.verify_drafts(draft, p, u, un, draft_probs=q)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        new = _inputs(80 + i, 3, 4, 70001, F32)
        for x, y in zip((draft, p, u, un, q), new):
            x.copy_(y)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        _check(out, _ref(draft, p, u, un, q))
