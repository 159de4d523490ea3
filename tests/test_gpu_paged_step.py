"""CAREKVLayer.paged_step against 64 bits, and a serving loop with drafts on it:
append, attend, verify, lengths that move on the device, eagerly and captured."""
import numpy as np
import pytest
import torch

from pages_ref import attend, check, round4, sight, turn

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _layer(care_kv, Hq, Hkv, D, model, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device="cuda") * model ** -0.5).to(dtype)  # noqa: E731
    cfg = care_kv.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, max_pages=4)
    W = (r(Hq * D, model), r(Hkv * D, model), r(Hkv * D, model), r(model, Hq * D))
    return care_kv.CAREKVLayer(cfg, 0, *W), lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (4, 4, 128)])
def test_steps(dtype, Hq, Hkv, D):
    """A prompt, a chunk and a token, ragged: each step's attention against 64 bits over the layer's own projections."""
    import care_kv
    B, model, P = 3, 96, 9
    layer, r = _layer(care_kv, Hq, Hkv, D, model, dtype)
    plan = care_kv.rotary_plan(D)
    pages = care_kv.int4_pages(B * P, Hkv, D)
    table = torch.randperm(B * P, device="cuda").view(B, P).int()
    held = [0, 0, 0]
    rows = [[None] * B, [None] * B]  # every sequence's turned K and its V, as far as they are held
    window, sink = 50, 3
    for T, counts, fresh in ((60, [60, 41, 1], True), (20, [20, 3, 0], False), (1, [1, 1, 1], False), (4, None, False)):
        h = r(B, T, model)
        lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
        got = layer.paged_step(pages, h, table, lengths, (plan, None), counts=counts, window=window, sink=sink, fresh=fresh)
        assert got.shape == h.shape and got.dtype == dtype
        cnt = [T] * B if counts is None else counts
        Q, K, V = layer._project(h)
        at = lengths.long()[:, None] + torch.arange(T, device="cuda")
        if fresh:
            q, k = care_kv.rotate_heads(Q, K, at, plan)
            ref = attend(q, k, V, sight(B, T, T, window, sink, cnt, cnt, None))
            k16 = k.float().half()
        else:
            q, k16 = turn(Q, at, plan).to(dtype), turn(K, at, plan).half()
        for b in range(B):
            for i, x in enumerate((k16, V.float().half())):
                x = round4(x[b, :, :cnt[b]])[2]
                rows[i][b] = x if rows[i][b] is None else torch.cat((rows[i][b], x), 1)
            held[b] += cnt[b]
        if not fresh:
            N = max(held)
            kk, vv = (torch.stack([torch.nn.functional.pad(x, (0, 0, 0, N - x.shape[1])) for x in w]) for w in rows)
            ref = attend(q, kk, vv, sight(B, T, N, window, sink, held, cnt, None), weights=F16)
        # what the layer's W_O makes of it: half a step for the product's input and output, and the attention's tolerance
        # through the weights' magnitudes
        W = layer.W_O.double()
        flat = lambda x: x.transpose(1, 2).reshape(B, T, -1)  # noqa: E731
        want, tol = flat(ref[0]) @ W.t(), flat(ref[2] + ref[0].abs() * torch.finfo(dtype).eps) @ W.abs().t()
        tol = tol + flat(ref[0].abs()) @ W.abs().t() * Hq * D * 2.0 ** -24 + want.abs() * torch.finfo(dtype).eps + 2.0 ** -24
        for b in range(B):
            assert ((got[b, :cnt[b]].double() - want[b, :cnt[b]]).abs() <= tol[b, :cnt[b]]).all(), (T, b)


def test_refusals():
    import care_kv
    layer, r = _layer(care_kv, 4, 2, 64, 32, F16)
    pages, table = care_kv.int4_pages(4, 2, 64), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    h = r(2, 3, 32)
    tables = torch.ones(1, 3, 64, device="cuda")
    for bad in (dict(hidden=h[0]), dict(position_embeddings=(tables, tables)), dict(lengths=None), dict(window=0), dict(counts=[1])):
        with pytest.raises(ValueError):
            layer.paged_step(**{**dict(pages=pages, hidden=h, table=table, lengths=0), **bad})


def test_serving_with_drafts():
    """Twelve steps of four drafts for three sequences.  What the pages hold at the end is what the tokens that stayed
    leave when they are appended at once: drafts that were rejected have been written over.  Captured, replayed among
    eager steps: the same tokens."""
    import care_kv
    B, T, V, model, Hq, Hkv, D, P, steps = 3, 4, 50, 64, 4, 2, 64, 6, 12
    layer, r = _layer(care_kv, Hq, Hkv, D, model, F16, seed=3)
    emb = r(V, model)
    plan = care_kv.rotary_plan(D)
    g = torch.Generator(device="cuda").manual_seed(9)
    q = torch.softmax(2 * torch.randn(steps, B, T, V, generator=g, device="cuda"), -1)
    draft = torch.multinomial(q.view(-1, V), 1, generator=g).view(steps, B, T)
    u, un = torch.rand(steps, B, T, generator=g, device="cuda"), torch.rand(steps, B, generator=g, device="cuda")
    u *= 0.6  # (drafts of another model: without this hardly one is accepted)

    def begin():
        pages = care_kv.int4_pages(B * P, Hkv, D)
        table = torch.arange(B * P, device="cuda").view(P, B).t().contiguous().int()
        lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        last = torch.tensor([1, 2, 3], device="cuda")
        return pages, table, lengths, last

    def step(state, draft, q, u, un):
        pages, table, lengths, last = state
        tokens = torch.cat((last[:, None], draft), 1)
        h = emb[tokens] + layer.paged_step(pages, emb[tokens], table, lengths, (plan, None), window=20, sink=2)
        p = torch.softmax((h.reshape(-1, model) @ emb.t()).float() * 0.05, -1).view(B, T + 1, V)
        got = care_kv.verify_drafts(draft, p, u, un, draft_probs=q)
        lengths += got.accepted + 1
        last.copy_(got.tokens.gather(1, got.accepted.long()[:, None])[:, 0])
        return got

    state = begin()
    eager, text = [], [[1], [2], [3]]
    for i in range(steps):
        got = step(state, draft[i], q[i], u[i], un[i])
        eager.append([x.clone() for x in got])
        for b in range(B):
            n = int(got.accepted[b])
            text[b] += got.tokens[b, :n + 1].tolist()
            assert got.tokens[b, :n].tolist() == draft[i, b, :n].tolist() and (got.tokens[b, n + 1:] == -1).all()
    taken = sum(int(x[1].sum()) for x in eager)
    assert 0 < taken < steps * B * T, "both are wanted: accepted and rejected drafts"
    pages, table, lengths, _ = state
    assert lengths.tolist() == [len(t) - 1 for t in text]
    # the tokens that stayed, appended at once, behind garbage
    once = care_kv.Int4Pages(torch.full_like(pages.data, 0x77), D)
    n = max(len(t) - 1 for t in text)
    ids = torch.tensor([t[:-1] + [0] * (n + 1 - len(t)) for t in text], device="cuda")
    _, K, W = layer._project(emb[ids])
    care_kv.append_pages(once, table, 0, K, W, plan=plan, counts=lengths)
    probe = r(B, Hq, n, D)
    a, b = (care_kv.paged_attention(probe, x, table, lengths, q_lengths=lengths, return_lse=True) for x in (pages, once))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])

    state = begin()
    ins = [x[0].clone() for x in (draft, q, u, un)]
    step(state, *ins)  # once eagerly: loads the kernels and the products' handles
    fresh = begin()
    for x, y in zip(state[2:], fresh[2:]):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state, *ins)
    for x, y in zip(state[2:], fresh[2:]):
        x.copy_(y)
    for i in range(steps):
        for x, y in zip(ins, (draft, q, u, un)):
            x.copy_(y[i])
        graph.replay()
        step(begin(), draft[i], q[i], u[i], un[i])  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out.tokens, eager[i][0]) and torch.equal(out.accepted, eager[i][1]), f"replay {i}"


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,R,layout", [(8, 2, 64, 64, "half"), (4, 4, 128, 64, "interleaved")])
def test_a_fresh_prompt_is_a_chunk(dtype, Hq, Hkv, D, R, layout):
    """A prompt leaves the same bytes whether it is written fresh or as a chunk of sequences that hold nothing: keys are
    turned and rounded to fp16 once."""
    import care_kv
    B, T, model, P = 3, 90, 64, 6
    layer, r = _layer(care_kv, Hq, Hkv, D, model, dtype, seed=5)
    plan = care_kv.rotary_plan(R, layout=layout)
    table = torch.randperm(B * P, device="cuda").view(B, P).int()
    h = r(B, T, model)
    for pos in (None, torch.arange(T, device="cuda") + 70000, torch.randint(0, 9000, (B, T), device="cuda")):
        for pe in ((plan, pos), None):
            left = []
            for fresh in (True, False):
                pages = care_kv.int4_pages(B * P, Hkv, D)
                layer.paged_step(pages, h, table, 0, pe, counts=[T, 33, 0], fresh=fresh)
                left.append(pages.data)
            assert torch.equal(*left), (pos is None, pe is None)


def test_counts_past_the_step():
    """Counts above T are T and counts below 0 are 0, as the operators take them, also for where the rows stand."""
    import care_kv
    B, T, model, Hq, Hkv, D, P = 4, 5, 64, 8, 2, 64, 4
    layer, r = _layer(care_kv, Hq, Hkv, D, model, F16, seed=6)
    plan = care_kv.rotary_plan(D)
    table = torch.arange(B * P, device="cuda").view(B, P).int()
    before, h = r(B, 30, model), r(B, T, model)
    held, counts, cut = [30, 4, 17, 9], [T + 4, -3, 2, 2 ** 31 - 1], [T, 0, 2, T]
    forms = (cut, counts, torch.tensor(counts, device="cuda"), torch.tensor(counts, device="cuda", dtype=torch.int32))
    want = None
    for fresh in (False, True):
        for i, n in enumerate(forms):
            pages = care_kv.int4_pages(B * P, Hkv, D)
            layer.paged_step(pages, before, table, 0, (plan, None))  # (what is behind held: tokens that did not stay)
            got = layer.paged_step(pages, h, table, held, (plan, None), counts=n, window=20, sink=2, fresh=fresh)
            want = (got, pages.data) if i == 0 else want
            assert torch.equal(pages.data, want[1])
            for b in range(B):
                assert torch.equal(got[b, :cut[b]], want[0][b, :cut[b]]), (fresh, i, b)


@pytest.mark.parametrize("fresh", [False, True])
def test_positions_need_a_plan(fresh):
    import care_kv
    layer, r = _layer(care_kv, 4, 2, 64, 32, F16)
    pages, table = care_kv.int4_pages(4, 2, 64), torch.arange(4, device="cuda").view(2, 2).int()
    with pytest.raises(ValueError):
        layer.paged_step(pages, r(2, 3, 32), table, 0, (None, torch.arange(3, device="cuda")), fresh=fresh)
    assert not pages.data.any()
    got = layer.paged_step(pages, r(2, 3, 32), table, 0, (None, None), fresh=fresh)
    assert got.shape == (2, 3, 32) and pages.data.any()


def test_a_refused_step_writes_nothing():
    import care_kv
    B, T, P = 2, 3, 2
    layer, r = _layer(care_kv, 4, 2, 64, 32, F16)
    pages, table, h = care_kv.int4_pages(B * P, 2, 64), torch.arange(B * P, device="cuda").view(B, P).int(), r(B, T, 32)
    plan = care_kv.rotary_plan(64)
    for fresh in (False, True):
        for bad in (dict(window=0), dict(window=-4), dict(sink=-1), dict(counts=[1]), dict(table=table[:1]),
                    dict(position_embeddings=(care_kv.rotary_plan(128), None)),
                    dict(position_embeddings=(plan, torch.zeros(T + 1, dtype=torch.int64, device="cuda")))):
            kw = {**dict(pages=pages, hidden=h, table=table, lengths=0, position_embeddings=(plan, None)), **bad}
            with pytest.raises(ValueError):
                layer.paged_step(**kw, fresh=fresh)
            assert not pages.data.any(), (fresh, bad)
