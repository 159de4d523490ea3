"""The long-prompt operators as they are used together: a prompt is placed, its
rows weighed and cut, what is left shared by a batch whose own tokens are
cached; and the paths of CAREKVLayer that call them; captured graphs, streams."""
import pytest
import torch

from helpers import PAPER_ENV

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(autouse=True)
def _need_gpu(monkeypatch):
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    for key, val in PAPER_ENV.items():
        monkeypatch.setenv(key, val)


def _rot64(x, pos, plan):
    t = pos.double()[:, None] * plan.freqs
    c, s = torch.cos(t), torch.sin(t)
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def test_together():
    """Prompt -> rotated heads -> attention and its log-sum-exp -> weights -> the
    heaviest rows -> a prefix for four sequences with cached tokens of their own."""
    import care_kv
    Hq, Hkv, D, T, keep, B = 8, 2, 64, 700, 200, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    plan = care_kv.rotary_plan(D, scaling="ntk", factor=4.0)
    pos = torch.arange(T, device="cuda")
    q0, k0, v = r(1, T, Hq, D).transpose(1, 2), r(1, T, Hkv, D).transpose(1, 2), r(1, T, Hkv, D).transpose(1, 2)
    q, k = care_kv.rotate_heads(q0, k0, pos, plan)
    assert float((k.double() - _rot64(k0, pos, plan)).abs().max()) < 4 * 2.0 ** -9  # values below 8: half a step 2^-9
    _, lse = care_kv.prefill_attention(q, k, v, return_lse=True)
    mass = care_kv.attention_mass(q, k, lse=lse)
    s = torch.stack([(q[0, h].double() @ k[0, h // 4].double().t()) * D ** -0.5 for h in range(Hq)])
    p = torch.softmax(s.masked_fill(pos[None, :] > pos[:, None], -float("inf")), -1).view(Hkv, 4, T, T).sum((1, 2))
    assert float((mass[0].double() - p).abs().max()) < 1e-4 * float(p.max())
    kept = care_kv.evict_rows(mass, k, v, keep=keep, sink=4, recent=32)
    order = torch.sort(mass[0, :, 4:T - 32], descending=True, stable=True).indices[:, :keep - 36] + 4
    want = torch.cat((torch.arange(4, device="cuda").expand(2, 4), order.sort(-1).values,
                      torch.arange(T - 32, T, device="cuda").expand(2, 32)), 1)
    assert torch.equal(kept.index[0].long(), want)
    prefix = (kept.k[0], kept.v[0])
    cfg = care_kv.CacheConfig(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, page_size=16, max_pages=8,
                              base_bits=4, group_size=32, packed_base=True, scale_quant="int8")
    cache = care_kv.CAREKVCache(cfg, device="cuda", n_seq=B)
    for step in range(5):
        at = torch.full((B, 1), T + step, device="cuda")
        qs, ks = care_kv.rotate_heads(r(B, Hq, 1, D), r(B, Hkv, 1, D), at, plan)
        cache.append(0, ks[:, :, 0], r(B, Hkv, D))
        out = care_kv.decode_attention(cache, 0, qs[:, :, 0], correction=False, prefix=prefix)
        from care_kv.attention import _base_rows
        for b in range(B):
            for h in range(Hq):
                K, V, _ = _base_rows(cache, 0, h // 4, None, b)
                kk = torch.cat((prefix[0][h // 4], K)).double()
                vv = torch.cat((prefix[1][h // 4], V)).double()
                w = torch.softmax(kk @ qs[b, h, 0].double() * D ** -0.5, 0)
                # fp16 weights (2^-11 each), the cached part and the result rounded to fp16
                tol = 2.0 ** -11 * (w @ vv.abs()) + 2 * 2.0 ** -11 * (w @ vv).abs() + 1e-4
                assert ((out[b, h].double() - w @ vv).abs() <= tol).all()


def _layer(care_kv, Hq=8, Hkv=2, D=64, seed=0, **kw):
    args = dict(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, page_size=16, max_pages=64, base_bits=4,
                group_size=32, k_channel_group=32, v_token_block=4, sketch_dim=32, packed_base=True, scale_quant="int8",
                store_budget_mode="absolute", store_abs_k=1, store_abs_v=1, read_budget_mode="absolute", read_abs_k=4,
                read_abs_v=4, read_budget_ratio=0.0, route_policy="joint")
    args.update(kw)
    cfg = care_kv.CacheConfig(**args)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dim = Hq * D
    w = [torch.randn(o, dim, generator=g, device="cuda").half() * 0.05 for o in (dim, Hkv * D, Hkv * D, dim)]
    return care_kv.CAREKVLayer(cfg, 0, *w), cfg, g


def _tables(plan, pos):
    t = pos.double()[..., None] * plan.freqs
    t = torch.cat((t, t), -1)
    return torch.cos(t).half(), torch.sin(t).half()


def test_layer_takes_positions(monkeypatch):
    """(RotaryPlan, positions) in place of (cos, sin): the heads of rotate_heads,
    near those of the fp16 tables; padded prompts slice the positions alike."""
    import care_kv
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "fp")
    lay, cfg, g = _layer(care_kv)
    B, T = 3, 37
    x = torch.randn(B, T, 512, generator=g, device="cuda").half()
    plan = care_kv.rotary_plan(64)
    pos = torch.arange(T, device="cuda").expand(B, T)
    Q, K, V = lay._project(x)
    q, k, v = lay._heads(x, (plan, pos))
    qr, kr = care_kv.rotate_heads(Q, K, pos, plan)
    assert torch.equal(q, qr) and torch.equal(k, kr) and torch.equal(v, V) and all(t.is_contiguous() for t in (q, k, v))
    tq, tk, _ = lay._heads(x, _tables(plan, pos[:1]))
    # the tables' rounding, two products and a sum in fp16: 4 half steps of |x1| + |x2|
    for a, b, x0 in ((q, tq, Q), (k, tk, K)):
        m = x0.abs().float()
        m = m + torch.cat((m[..., 32:], m[..., :32]), -1)
        assert ((a.float() - b.float()).abs() <= 4 * 2.0 ** -11 * m + 1e-4).all()
    keep = torch.ones(B, T, dtype=torch.int64, device="cuda")
    keep[1, :9] = 0
    caches = [care_kv.CAREKVCache(cfg, n_seq=B) for _ in range(2)]
    o1 = lay.prefill(caches[0], x, attention_mask=keep, position_embeddings=(plan, pos))
    alone = lay.prefill(caches[1], x[1:2, 9:], position_embeddings=(plan, pos[1:2, 9:]), seqs=[1])
    assert torch.equal(o1[1, 9:], alone[0]) and not o1[1, :9].any()
    step = torch.full((B, 1), T, device="cuda")
    assert lay.decode_step(caches[0], x[:, :1], position_embeddings=(plan, step)).shape == (B, 1, 512)


@pytest.mark.parametrize("mode", ["fp", "base_quant", "carekv_eval"])
@pytest.mark.parametrize("window", [0, 16])
def test_layer_keeps_heavy_rows(mode, window, monkeypatch):
    """prefill_keep: the prompt's outputs stay as they are, the pages hold the
    kept rows; prompts that fit keep their pages bit for bit."""
    import care_kv
    monkeypatch.setenv("CAREKV_PREFILL_MODE", mode)
    lay, cfg, g = _layer(care_kv, prefill_keep=64, prefill_keep_sink=4, prefill_keep_recent=16,
                         prefill_keep_window=window)
    whole, wcfg, _ = _layer(care_kv)
    plan = care_kv.rotary_plan(64)
    for T in (150, 64, 10):
        B = 2
        x = torch.randn(B, T, 512, generator=g, device="cuda").half()
        pe = (plan, torch.arange(T, device="cuda"))
        a, b = care_kv.CAREKVCache(cfg, n_seq=B), care_kv.CAREKVCache(wcfg, n_seq=B)
        oa, ob = lay.prefill(a, x, position_embeddings=pe), whole.prefill(b, x, position_embeddings=pe)
        assert torch.equal(oa, ob)
        assert a.total_valid_tokens(0, 0, 1) == min(T, 64)
        if T <= 64:
            assert torch.equal(a.kcodes[:, :, :, :T // 16], b.kcodes[:, :, :, :T // 16])
            continue
        q, k, v = lay._heads(x, pe)
        kh, vh = (care_kv.quant_dequant(t, 4) for t in (k, v))
        ka, va = (k, v) if mode == "fp" else (kh, vh)
        _, lse = care_kv.prefill_attention(q, ka, va, return_lse=True)
        w = window or T
        kept = care_kv.evict_rows(care_kv.attention_mass(q[:, :, T - w:], ka, lse=lse[:, :, T - w:]), k, v, keep=64,
                                  sink=4, recent=16)
        ref = care_kv.CAREKVCache(cfg, n_seq=B)
        ref.write_prefill(0, kept.k, kept.v)
        for nm in ("kcodes", "vcodes", "kscale", "kmaster", "valid", "k_slot", "v_slot"):
            assert torch.equal(getattr(a, nm), getattr(ref, nm)), nm
        y = lay.decode_step(a, x[:, :1], position_embeddings=(plan, torch.full((B, 1), T, device="cuda")))
        assert torch.isfinite(y).all() and a.total_valid_tokens(0, 0, 1) == 65


def test_layer_refuses_what_reads_whole_prompts(monkeypatch):
    import care_kv
    plan = care_kv.rotary_plan(64)
    x = torch.zeros(1, 100, 512, device="cuda").half()
    pe = (plan, torch.arange(100, device="cuda"))
    pre = tuple(torch.zeros(2, 8, 64, device="cuda").half() for _ in range(2))
    lay, cfg, _ = _layer(care_kv, prefill_keep=64)
    cache = care_kv.CAREKVCache(cfg, n_seq=1)
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "carekv_stored")
    with pytest.raises(NotImplementedError):
        lay.prefill(cache, x, position_embeddings=pe)
    for mode in ("carekv_stored", "carekv_eval"):
        monkeypatch.setenv("CAREKV_PREFILL_MODE", mode)
        with pytest.raises(NotImplementedError):
            lay.prefill(cache, x[:, :20], position_embeddings=pe, prefix=pre)
    assert cache.num_pages(0, 0) == 0  # refused before anything was written
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "base_quant")
    lay, cfg, _ = _layer(care_kv, prefill_keep=64, base_quantizer="kivi_style", base_bits=2)
    with pytest.raises(NotImplementedError):
        lay.prefill(care_kv.CAREKVCache(cfg, n_seq=1), x, position_embeddings=pe)


def test_layer_behind_a_prefix(monkeypatch):
    """prefill and decode_step behind a shared prefix: in the fp mode a prompt's
    outputs are those of the whole text's rows, up to the roundings of two fp16
    outputs joined (2^-11 each) and of W_O's product over them."""
    import care_kv
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "fp")
    lay, cfg, g = _layer(care_kv)
    P, T = 333, 21
    plan = care_kv.rotary_plan(64)
    text = torch.randn(1, P + T, 512, generator=g, device="cuda").half()
    q, k, v = lay._heads(text, (plan, torch.arange(P + T, device="cuda")))
    O = care_kv.prefill_attention(q, k, v)[:, :, P:]
    want = lay._out(O, F16)
    prefix = (k[0, :, :P], v[0, :, :P])
    cache = care_kv.CAREKVCache(cfg, n_seq=2)
    x = text[:, P:].expand(2, T, 512)
    got = lay.prefill(cache, x, position_embeddings=(plan, torch.arange(P, P + T, device="cuda")), prefix=prefix)
    tol = (3 * 2.0 ** -11) * (O.abs().double().transpose(1, 2).reshape(1, T, -1) @ lay.W_O.abs().double().t()) + 2e-3
    assert ((got[1].double() - want[0].double()).abs() <= tol[0]).all()
    assert cache.total_valid_tokens(0, 0, 1) == T
    pos = torch.full((2, 1), P + T, device="cuda")
    y = lay.decode_step(cache, x[:, :1], position_embeddings=(plan, pos), prefix=prefix)
    qd, _, _ = lay._heads(x[:, :1], (plan, pos))
    from care_kv.attention import decode_read_mode
    corr, knobs = decode_read_mode(cfg, 0)
    o = care_kv.decode_attention(cache, 0, qd[:, :, 0], correction=corr, knobs=knobs, prefix=prefix)
    assert torch.equal(y, lay._out(o.unsqueeze(2), F16))


def _ops(care_kv, seed):
    """Inputs and one call of each operator over them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    d = dict(q=r(2, 8, 50, 64), k=r(2, 2, 300, 64), v=r(2, 2, 300, 64), pk=r(2, 900, 64), pv=r(2, 900, 64),
             pos=torch.arange(50, device="cuda") + seed, n=torch.tensor([300, 123], device="cuda").int(),
             own=(r(2, 8, 50, 64), torch.randn(2, 8, 50, generator=g, device="cuda")))
    plan = care_kv.rotary_plan(64)

    def call():
        q, _ = care_kv.rotate_heads(d["q"], None, d["pos"], plan)
        mass = care_kv.attention_mass(q, d["k"], lengths=d["n"])
        kept = care_kv.evict_rows(mass, d["k"], d["v"], keep=77, sink=2, recent=9, lengths=d["n"])
        o, lse = care_kv.prefix_attention(q, d["pk"], d["pv"], own=d["own"], return_lse=True)
        return [q, mass, *kept, o, lse]
    return d, call


def test_captured_and_replayed():
    """Each operator in a HIP graph, replayed over new inputs with eager work and
    synchronizations between, two graphs alive at once; eager bits every time."""
    import care_kv
    graphs = []
    for seed in (1, 2):
        d, call = _ops(care_kv, seed)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((d, call, g, out))
    for turn in range(4):
        for i, (d, call, g, out) in enumerate(graphs):
            new, _ = _ops(care_kv, 10 * turn + i)
            for nm in ("q", "k", "v", "pk", "pv", "pos"):
                d[nm].copy_(new[nm])
            for a, b in zip(d["own"], new["own"]):
                a.copy_(b)
        if turn % 2:
            torch.cuda.synchronize()
        for d, call, g, out in graphs:
            g.replay()
        for d, call, g, out in graphs:
            for a, b in zip(out, call()):
                assert torch.equal(a, b)


@pytest.mark.parametrize("correction", [False, True])
def test_decode_behind_a_prefix_captured(correction, monkeypatch):
    """decode_attention(prefix=...) in a graph, replayed over new queries and a
    new prefix with eager calls between."""
    import care_kv
    monkeypatch.setenv("CAREKV_CHECK", "0")  # (the status word's read-back waits for the stream)
    lay, cfg, g = _layer(care_kv)
    cache = care_kv.CAREKVCache(cfg, n_seq=2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    cache.write_prefill(0, r(2, 2, 300, 64), r(2, 2, 300, 64))
    q, k, v = r(2, 8, 64), r(2, 1500, 64), r(2, 1500, 64)

    def call():
        return care_kv.decode_attention(cache, 0, q, correction=correction, prefix=(k, v), return_lse=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn in range(4):
        for x in (q, k, v):
            x.copy_(r(*x.shape))
        if turn % 2:
            torch.cuda.synchronize()
        graph.replay()
        got = [o.clone() for o in out]
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def test_hf_model_keeps_heavy_rows(monkeypatch):
    """A patched model under CacheConfig.prefill_keep: generates from a long and
    a padded prompt, its pages hold the kept rows and the decoded ones; a prompt
    that fits generates the tokens of the unbounded cache."""
    import care_kv
    transformers = pytest.importorskip("transformers")
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "fp")
    hf = transformers.LlamaConfig(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                  num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=512)
    ids = torch.randint(3, 300, (2, 120), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones_like(ids)
    mask[1, :30] = 0
    outs = {}
    for keep in (0, 48, 150):
        torch.manual_seed(0)
        model = transformers.LlamaForCausalLM(hf).half().cuda().eval()
        cfg = care_kv.CacheConfig(num_layers=2, num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, max_pages=16,
                                  base_bits=4, group_size=32, packed_base=True, scale_quant="int8", prefill_keep=keep,
                                  prefill_keep_sink=4, prefill_keep_recent=16)
        model = care_kv.patch_llama_model(model, cfg)
        with torch.no_grad():
            outs[keep] = model.generate(ids, attention_mask=mask, max_new_tokens=6, do_sample=False, pad_token_id=0)
        att = next(m for m in model.modules() if isinstance(m, care_kv.CAREKVLlamaAttention))
        cache = att._shared.cache
        rows = [cache.total_valid_tokens(1, 1, s) for s in range(2)]
        assert rows == [(48 if keep == 48 else 120) + 5, (48 if keep == 48 else 90) + 5]
        assert outs[keep].shape == (2, 126)
    assert torch.equal(outs[0], outs[150])
    assert torch.equal(outs[48][:, :121], outs[0][:, :121])  # the prompt's own attention sees every row


def test_host_lists_are_refused_in_captured_code():
    """A captured call takes lengths on the device (or one int); host lists raise
    and leave the capture to go on."""
    import care_kv
    q, k = torch.randn(2, 4, 40, 64, device="cuda").half(), torch.randn(2, 2, 90, 64, device="cuda").half()
    want = care_kv.attention_mass(q, k, q_start=50)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError):
            care_kv.attention_mass(q, k, lengths=[90, 3])
        with pytest.raises(ValueError):
            care_kv.evict_rows(want, k, k, keep=5, lengths=[90, 3])
        got = care_kv.attention_mass(q, k, q_start=50)
    for _ in range(3):
        got.zero_()
        g.replay()
        assert torch.equal(got, want)


def test_two_streams_at_once():
    import care_kv
    pairs = [_ops(care_kv, s) for s in (3, 4)]
    want = [call() for _, call in pairs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pairs]
    got = [[], []]
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pairs[i][1]())
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            for a, b in zip(outs, want[i]):
                assert torch.equal(a, b)


def test_refusals_leave_the_cache_alone(monkeypatch):
    """A prefix that does not fit is refused before a prompt is written or a
    token appended; an output over the queries or the prefix is refused too."""
    import care_kv
    monkeypatch.setenv("CAREKV_PREFILL_MODE", "fp")
    lay, cfg, g = _layer(care_kv)
    cache = care_kv.CAREKVCache(cfg, n_seq=2)
    x = torch.randn(2, 9, 512, generator=g, device="cuda").half()
    k = torch.randn(2, 33, 64, generator=g, device="cuda").half()
    plan = care_kv.rotary_plan(64)
    pe = (plan, torch.arange(33, 42, device="cuda"))
    for bad in ((k, k[:, :5]), (k.bfloat16(), k.bfloat16()), (k[..., :32], k[..., :32]), (k,)):
        with pytest.raises(ValueError):
            lay.prefill(cache, x, position_embeddings=pe, prefix=bad)
    assert cache.total_valid_tokens(0, 0, 0) == 0
    lay.prefill(cache, x, position_embeddings=pe, prefix=(k, k))
    for bad in ((k, k[:, :5]), (k.float(), k.float())):
        with pytest.raises(ValueError):
            lay.decode_step(cache, x[:, :1], position_embeddings=(plan, pe[1][:1]), prefix=bad)
    assert cache.total_valid_tokens(0, 0, 0) == 9
    q = torch.randn(2, 8, 64, generator=g, device="cuda").half()
    for out in (q, k.view(-1)[:1024].view(2, 8, 64)):
        with pytest.raises(ValueError, match="overlap"):
            care_kv.decode_attention(cache, 0, q, prefix=(k, k), out=out)


def test_layer_rounds_32_bit_heads_after_the_turn():
    """fp32 projections: each head value is off by one fp16 rounding of the
    turned value (half a step, 2^-11 of it; 2^-25 below 2^-14) and the 32-bit turn's own error."""
    import care_kv
    lay, _, g = _layer(care_kv)
    for p in lay.parameters():
        p.data = p.data.float()
    x = torch.randn(2, 37, 512, generator=g, device="cuda")
    plan = care_kv.rotary_plan(64)
    pos = torch.arange(1000, 1037, device="cuda")
    Q, K, _ = lay._project(x)
    q, k, _ = lay._heads(x, (plan, pos))
    for got, x0 in ((q, Q), (k, K)):
        want = _rot64(x0, pos, plan)
        m = x0.abs().double()
        m = m + torch.cat((m[..., 32:], m[..., :32]), -1)
        # angles off by 2^-26 turns (2 pi 2^-26 < 2^-23) and their 32-bit sine, cosine and products
        assert got.dtype == F16 and ((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + 2.0 ** -21 * m).all()


def test_empty_operands_of_any_strides():
    """No query rows, or no prefix: what their views' strides are does not count."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    q, k = r(2, 4, 7, 65)[..., 1:], r(2, 2, 9, 64)
    assert not care_kv.attention_mass(q[:, :, :0], k).any()
    o, lse = r(2, 4, 7, 64), torch.randn(2, 4, 7, generator=g, device="cuda")
    p = r(2, 5, 65)[:, :0, 1:]
    got, l = care_kv.prefix_attention(q, p, p, own=(o, lse), return_lse=True)
    assert torch.equal(got, o) and float((l - lse).abs().max()) < 1e-5


def test_rows_far_apart():
    """Rows 2^22 elements apart and more: copied like any rows that the kernels do not read as they lie."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(4)
    far = lambda n: torch.randn(n * ((1 << 22) + 64), generator=g, device="cuda", dtype=torch.float16).as_strided(  # noqa: E731
        (2, n, 64), (64, (1 << 22) + 64, 1))
    q, k, v = far(3)[None], far(5), far(5)
    assert torch.equal(care_kv.attention_mass(q, k[None]), care_kv.attention_mass(q.contiguous(), k[None].contiguous()))
    got = care_kv.prefix_attention(q, k, v, return_lse=True)
    for a, b in zip(got, care_kv.prefix_attention(q.contiguous(), k.contiguous(), v.contiguous(), return_lse=True)):
        assert torch.equal(a, b)


def test_layer_rounds_bf16_heads_once():
    """bf16 projections past fp16's range in both directions: what a turn brings back into it is rounded once, after
    the turn (half a step, 2^-11 of it; 2^-25 below 2^-14), beside the 32-bit turn's own error."""
    import care_kv
    lay, _, g = _layer(care_kv)
    for p in lay.parameters():
        p.data = p.data.bfloat16()
    lay.W_K.data *= 40000
    lay.W_Q.data *= 2.0 ** -20
    x = torch.randn(2, 37, 512, generator=g, device="cuda").bfloat16()
    plan = care_kv.rotary_plan(64)
    pos = torch.arange(1000, 1037, device="cuda")
    Q, K, _ = lay._project(x)
    q, k, v = lay._heads(x, (plan, pos))
    assert (K.abs() > 65504).any() and (Q.abs() < 2.0 ** -24).any() and q.dtype == k.dtype == v.dtype == F16
    for got, x0 in ((q, Q), (k, K)):
        want = _rot64(x0, pos, plan)
        m = x0.abs().double()
        m = m + torch.cat((m[..., 32:], m[..., :32]), -1)
        fits = want.abs() + 2.0 ** -21 * m < 65504
        assert float(fits.double().mean()) > 0.5
        err = (got.double() - want).abs()
        assert (err[fits] <= (2.0 ** -11 * want.abs() + 2.0 ** -25 + 2.0 ** -21 * m)[fits]).all()


def test_kept_rows_of_a_short_sequence():
    """A ragged batch, one sequence shorter than keep: cut to its kept length, its rows are a prefix of its own rows
    alone, and what the pages store."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    k, v, q, lens = r(2, 2, 200, 64), r(2, 2, 200, 64), r(3, 8, 64), [200, 17]
    kept = care_kv.evict_rows(torch.rand(2, 2, 200, generator=g, device="cuda"), k, v, keep=50, sink=4, recent=8, lengths=lens)
    n = int(kept.lengths[1])
    assert n == 17 and not kept.k[1][:, n:].any()
    for a, b in zip(care_kv.prefix_attention(q, kept.k[1][:, :n], kept.v[1][:, :n], return_lse=True),
                    care_kv.prefix_attention(q, k[1, :, :17], v[1, :, :17], return_lse=True)):
        assert torch.equal(a, b)
    _, cfg, _ = _layer(care_kv)
    a, b = care_kv.CAREKVCache(cfg, n_seq=1), care_kv.CAREKVCache(cfg, n_seq=1)
    a.write_prefill(0, kept.k[1:, :, :n], kept.v[1:, :, :n])
    b.write_prefill(0, k[1:, :, :17], v[1:, :, :17])
    assert a.total_valid_tokens(0, 0, 0) == 17
    for nm in ("kcodes", "vcodes", "kscale", "valid"):
        assert torch.equal(getattr(a, nm), getattr(b, nm)), nm
