"""prefix_attention against a 64-bit softmax over the prefix and the rows' own
tokens, and decode_attention over a cache behind a shared prefix."""
import numpy as np
import pytest
import torch

from helpers import PAPER_ENV

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _ref(q, k, v, own=None, scale=None):
    """(o, lse, tolerance of o) in 64 bits.  The tolerance: each weight is
    rounded to the element type (half a step) and its logit is off by at most
    (D + 8) 2^-24 of the sum of its terms' magnitudes, the result is rounded."""
    B, Hq, T, D = q.shape
    Hkv = k.shape[0]
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -float("inf"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    half = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        for h in range(Hq):
            x, y, z = q[b, h].double(), k[h // (Hq // Hkv)].double(), v[h // (Hq // Hkv)].double()
            s = x @ y.t() * scale
            e = (x.abs() @ y.abs().t()).max() * abs(scale) * (D + 8) * 2.0 ** -24 if s.numel() else 0.0
            if own is not None:
                s = torch.cat((s, own[1][b, h].double()[:, None]), 1)
            if s.shape[1] == 0:
                continue
            l = torch.logsumexp(s, 1)
            w = torch.where(torch.isfinite(l)[:, None], torch.exp(s - l[:, None]), 0.0)
            wp = w[:, :k.shape[1]]
            y_o, mag = wp @ z, wp @ z.abs()
            if own is not None:
                oo = torch.where(w[:, -1:] > 0, own[0][b, h].double(), 0.0)
                y_o, mag = y_o + w[:, -1:] * oo, mag + w[:, -1:] * oo.abs()
            o[b, h], lse[b, h] = y_o, l
            tol[b, h] = mag * (half + 2 * e + 2.0 ** -18) + y_o.abs() * half + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    return o, lse, tol * 1.001


def _check(got, ref):
    (o, lse), (ro, rl, tol) = got, ref
    err = (o.double() - ro).abs()
    assert (err <= tol).all(), float((err - tol).max())
    fin = torch.isfinite(rl)
    assert torch.equal(torch.isinf(lse), ~fin)
    assert ((lse.double() - rl)[fin].abs() <= 2e-5 + 2e-6 * rl[fin].abs()).all()


def _inputs(seed, B, Hq, Hkv, D, T, P, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = r(B, Hq, T, D).to(dtype), r(Hkv, P, D).to(dtype), r(Hkv, P, D).to(dtype)
    return q, k, v, (r(B, Hq, T, D).to(dtype), 3 * r(B, Hq, T) + 2)


SHAPES = [  # B, Hq, Hkv, D, T, P
    (1, 1, 1, 64, 1, 1), (1, 4, 4, 128, 1, 33), (2, 8, 1, 64, 1, 500), (4, 32, 4, 64, 1, 1000), (3, 6, 2, 128, 1, 2049),
    (1, 2, 1, 128, 5, 31), (5, 7, 7, 64, 3, 32), (33, 4, 1, 64, 1, 257), (2, 4, 2, 128, 130, 700), (1, 16, 1, 64, 1, 9000),
    (130, 2, 2, 64, 1, 64), (17, 8, 2, 128, 2, 4097),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,T,P", SHAPES)
def test_against_64_bits(dtype, B, Hq, Hkv, D, T, P):
    import care_kv
    print(f"prefix {dtype} B={B} {Hq}/{Hkv} D={D} T={T} P={P}", flush=True)
    q, k, v, own = _inputs(P + B, B, Hq, Hkv, D, T, P, dtype)
    _check(care_kv.prefix_attention(q, k, v, return_lse=True), _ref(q, k, v))
    got = care_kv.prefix_attention(q, k, v, own=own, return_lse=True)
    _check(got, _ref(q, k, v, own))
    o = own[0].clone()
    again = care_kv.prefix_attention(q, k, v, own=(o, own[1]), out=o)  # in place, and the same bits
    assert again.data_ptr() == o.data_ptr() and torch.equal(o, got[0])
    if T == 1:
        one = care_kv.prefix_attention(q[:, :, 0], k, v, own=(own[0][:, :, 0], own[1][:, :, 0]), return_lse=True)
        assert torch.equal(one[0], got[0][:, :, 0]) and torch.equal(one[1], got[1][:, :, 0])


@pytest.mark.parametrize("P", [0, 40])
def test_rows_without_tokens(P):
    """Rows with no own token (lse -inf, garbage in o), and no prefix at all."""
    import care_kv
    q, k, v, own = _inputs(3, 4, 4, 2, 64, 2, P, torch.float16)
    own[1][1] = -float("inf")
    own[0][1] = float("nan")
    got = care_kv.prefix_attention(q, k, v, own=own, return_lse=True)
    _check(got, _ref(q, k, v, own))
    if P == 0:
        assert not got[0][1].any() and torch.equal(got[0][0], own[0][0])
        alone = care_kv.prefix_attention(q, k, v, return_lse=True)
        assert not alone[0].any() and (alone[1] == -float("inf")).all()


def test_extreme_logits():
    """Logits of some hundreds, rising and falling along the prefix, negative and
    zero scales, one key that outweighs all by more than 32 bits hold."""
    import care_kv
    q, k, v, own = _inputs(7, 3, 4, 2, 64, 1, 900, torch.float16)
    ramp = torch.linspace(0.1, 8, 900, device="cuda")[None, :, None]
    for kk in ((k * ramp).half(), (k * ramp.flip(1)).half()):
        for scale in (None, -0.3, 0.0, 1.0):
            _check(care_kv.prefix_attention(q, kk, v, own=own, sm_scale=scale, return_lse=True),
                   _ref(q, kk, v, own, scale))
    k2 = k.clone()
    k2[:, 500] = 0
    k2[0, 500] = (40 * q[0, 0, 0]).half()
    _check(care_kv.prefix_attention(q, k2, v, own=own, return_lse=True), _ref(q, k2, v, own))


def test_strides():
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    B, T, Hq, Hkv, D, P = 3, 9, 8, 2, 128, 333
    q = r(B, T, Hq, D).transpose(1, 2)
    kv = r(P, 2, Hkv, D)
    k, v = kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1)
    o = r(B, T, Hq, D).transpose(1, 2)
    lse = torch.randn(B, T, Hq, generator=g, device="cuda").transpose(1, 2)
    out = torch.full((B, T, Hq, D + 3), 5.0, device="cuda").bfloat16()
    view = out[..., 3:].transpose(1, 2)
    ref = _ref(q, k, v, (o, lse))
    got = care_kv.prefix_attention(q, k, v, own=(o, lse), out=view, return_lse=True)
    assert got[0].data_ptr() == view.data_ptr() and (out[..., :3] == 5).all()
    _check(got, ref)
    odd = r(Hkv, P, D + 1)[..., 1:]
    apart = r(Hkv, D, P).transpose(1, 2)
    _check(care_kv.prefix_attention(q, odd, apart, own=(o, lse), return_lse=True), _ref(q, odd, apart, (o, lse)))
    same = r(1, P, D).expand(Hkv, P, D)  # one head's rows for every kv head
    _check(care_kv.prefix_attention(q, same, same, return_lse=True), _ref(q, same, same))
    one_row = r(Hkv, 1, D).expand(Hkv, P, D)
    _check(care_kv.prefix_attention(q, one_row, one_row, return_lse=True), _ref(q, one_row, one_row))


def test_offsets_past_32_bits():
    import care_kv
    P, H, D = 900_000, 20, 128
    buf = torch.zeros(P, H, D, dtype=torch.float16, device="cuda")   # 4.6 GB
    k = buf[:, 18:20].transpose(0, 1)
    q = torch.randn(2, 2, 1, D, device="cuda").half()
    for at in (7, 430_000, P - 1):
        k[:, at] = (q[0, :, 0] * 3).half()
    _check(care_kv.prefix_attention(q, k, k, return_lse=True), _ref(q, k, k))


def _cache(care_kv, lens, Hq=8, Hkv=2, D=64, seed=0, **kw):
    args = dict(num_layers=1, num_heads=Hq, num_kv_heads=Hkv, head_dim=D, page_size=16, max_pages=max(lens) // 16 + 4,
                base_bits=3, group_size=32, packed_base=True, scale_quant="int8", store_budget_mode="absolute",
                store_abs_k=1, store_abs_v=1, read_budget_mode="absolute", read_abs_k=6, read_abs_v=6,
                route_policy="joint", read_budget_ratio=0.0)
    args.update(kw)
    cache = care_kv.CAREKVCache(care_kv.CacheConfig(**args), device="cuda", n_seq=len(lens))
    rng = np.random.default_rng(seed)
    for s, T in enumerate(lens):
        if T:
            K, V = (torch.from_numpy(rng.standard_normal((Hkv, T, D)).astype(np.float16)).cuda() for _ in range(2))
            cache.write_prefill(0, K, V, seqs=[s])
    return cache, torch.from_numpy(rng.standard_normal((len(lens), Hq, D)).astype(np.float16)).cuda()


@pytest.mark.parametrize("kw", [dict(), dict(Hq=16, Hkv=1), dict(D=128, base_quantizer="kivi_style", base_bits=2),
                                dict(base_quantizer="kivi_style", base_bits=2, kivi_packed=True)])
def test_decode_lse(kw, monkeypatch):
    """return_lse of the base attention against the dequantised rows, the same
    output bits with and without it."""
    import care_kv
    from care_kv.attention import _base_rows
    for key, val in PAPER_ENV.items():
        monkeypatch.setenv(key, val)
    lens = [0, 5, 16, 333]
    cache, q = _cache(care_kv, lens, **kw)
    cfg = cache.cfg
    out, lse = care_kv.decode_attention(cache, 0, q, correction=False, return_lse=True)
    assert torch.equal(out, care_kv.decode_attention(cache, 0, q, correction=False))
    for b, n in enumerate(lens):
        for h in range(cfg.num_heads):
            if n == 0:
                assert lse[b, h] == -float("inf") and not out[b, h].any()
                continue
            K, _, _ = _base_rows(cache, 0, h // (cfg.num_heads // cfg.num_kv_heads), None, b)
            want = torch.logsumexp(K.double() @ q[b, h].double() * cfg.head_dim ** -0.5, 0)
            assert abs(float(lse[b, h]) - float(want)) < 1e-4
    c_out, c_lse = care_kv.decode_attention(cache, 0, q, correction=True, return_lse=True)
    assert torch.equal(c_out, care_kv.decode_attention(cache, 0, q, correction=True))
    assert torch.isfinite(c_lse[1:]).all() and (c_lse[0] == -float("inf")).all()
    s_out = torch.empty_like(q)
    _, s_lse = care_kv.decode_attention(cache, 0, q, correction=True, return_lse=True, no_alloc=True, out=s_out)
    assert torch.equal(s_out, c_out) and torch.equal(s_lse, c_lse)


def test_corrected_lse_is_the_corrected_scores(monkeypatch):
    """The exact K correction replaces the selected groups' scores by those of
    K_hat + R: with every slot stored and read, the log-sum-exp behind the
    output is that of the rows K_hat + R, up to the weights that the correction
    sums, which are kept in fp16 (2^-11 of each)."""
    import care_kv
    from care_kv.attention import _base_rows
    from care_kv.residual import unpack_4bit
    for key, val in PAPER_ENV.items():
        monkeypatch.setenv(key, val)
    monkeypatch.setenv("CAREKV_K_CORRECTION_MODE", "exact")
    T, D = 64, 64
    cache, q = _cache(care_kv, [T], Hq=2, Hkv=1, D=D, store_abs_k=2, store_abs_v=4, read_abs_k=64, read_abs_v=64)
    out, lse = care_kv.decode_attention(cache, 0, q, correction=True, return_lse=True)
    K, _, _ = _base_rows(cache, 0, 0, None, 0)
    K = K.double()
    for p in range(T // 16):
        for cg in range(D // 32):
            slot = int(cache.k_slot[0, 0, 0, p, cg])
            assert slot >= 0
            R = unpack_4bit(cache.k_res[0, slot], cache.k_res_scale[0, slot:slot + 1], 16 * 32).view(16, 32)
            K[16 * p:16 * p + 16, 32 * cg:32 * cg + 32] += R.double()
    for h in range(2):
        want = torch.logsumexp(K @ q[0, h].double() * D ** -0.5, 0)
        assert abs(float(lse[0, h]) - float(want)) < 2.0 ** -10


@pytest.mark.parametrize("correction", [False, True])
def test_decode_behind_a_prefix(correction, monkeypatch):
    """decode_attention(prefix=...): the softmax over the prefix and the cached
    rows, of which the cached part is decode_attention's own output."""
    import care_kv
    for key, val in PAPER_ENV.items():
        monkeypatch.setenv(key, val)
    cache, q = _cache(care_kv, [0, 40, 500], Hq=8, Hkv=2, D=128)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(2, 777, 128, generator=g, device="cuda").half() for _ in range(2))
    o, l = care_kv.decode_attention(cache, 0, q, correction=correction, return_lse=True)
    got = care_kv.decode_attention(cache, 0, q, correction=correction, prefix=(k, v), return_lse=True)
    ref = _ref(q[:, :, None], k, v, (o[:, :, None], l[:, :, None]))
    _check((got[0][:, :, None], got[1][:, :, None]), ref)
    with_diag = care_kv.decode_attention(cache, 0, q, correction=correction, prefix=(k, v), diag_cap=8)
    assert torch.equal(with_diag[0], got[0]) and with_diag[1].shape == (3, 8, 8)
    with pytest.raises(ValueError):
        care_kv.decode_attention(cache, 0, q, prefix=(k, v), no_alloc=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,T,P", [(40, 4, 2, 64, 1, 5000), (9, 8, 1, 64, 5, 12345), (33, 1, 1, 128, 1, 4096),
                                            (1, 6, 2, 128, 50, 4111), (2, 3, 3, 64, 40, 33000)])
def test_long_prefixes_of_many_rows(dtype, B, Hq, Hkv, D, T, P):
    """Prefixes long enough that the waves of a work-group share the rows as well as the keys."""
    import care_kv
    print(f"prefix {dtype} B={B} {Hq}/{Hkv} D={D} T={T} P={P}", flush=True)
    q, k, v, own = _inputs(P, B, Hq, Hkv, D, T, P, dtype)
    own[1][0] = -torch.inf
    got = care_kv.prefix_attention(q, k, v, own=own, return_lse=True)
    _check(got, _ref(q, k, v, own))
    for a, b in zip(got, care_kv.prefix_attention(q, k, v, own=own, return_lse=True)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nats", [9.0, 17.5, 21.0, 27.0])
@pytest.mark.parametrize("B,D,P", [(1, 64, 1024), (4, 128, 1000), (64, 64, 256), (40, 128, 9000)])
def test_a_long_tail_below_one_key(dtype, nats, B, D, P):
    """One key far above a long flat prefix, and a value of 0 there: the result is the tail's, whose weights keep their
    rounding of half a step each.  fp16 weights that are subnormal even times 2^15 are off by half of 2^-24 of
    2^-15 of the largest."""
    import care_kv
    print(f"prefix {dtype} {nats} nats B={B} D={D} P={P}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(P)
    q = torch.ones(B, 4, 1, D, device="cuda").to(dtype)
    k = (0.1 * torch.randn(2, P, D, generator=g, device="cuda")).to(dtype)
    k[:, P // 3] = nats / D ** 0.5
    v = (200 + 100 * torch.rand(2, P, D, generator=g, device="cuda")).to(dtype)
    v[:, P // 3] = 0
    o, lse, tol = _ref(q, k, v)
    if dtype == torch.float16:
        tol = tol + P * 2.0 ** -40 * float(v.max())
    _check(care_kv.prefix_attention(q, k, v, return_lse=True), (o, lse, tol))
