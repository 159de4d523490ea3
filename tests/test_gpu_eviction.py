"""attention_mass and evict_rows against 64-bit evaluations."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _mass_ref(q, k, causal=True, lse=None, q_start=None, lengths=None, scale=None):
    """(mass, log-sum-exp, bound of a logit's 32-bit error) in 64 bits."""
    B, Hq, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    mass = torch.zeros(B, Hkv, Tk, dtype=torch.float64, device=q.device)
    out_lse = torch.full((B, Hq, Tq), -float("inf"), dtype=torch.float64, device=q.device)
    err = 0.0
    for b in range(B):
        n = Tk if lengths is None else max(0, min(int(lengths[b]), Tk))
        at = (n - Tq if q_start is None else int(q_start[b])) + torch.arange(Tq, device=q.device)
        j = torch.arange(Tk, device=q.device)
        see = (j < n)[None, :] & ((j[None, :] <= at[:, None]) if causal else torch.ones(Tq, Tk, device=q.device).bool())
        for h in range(Hq):
            x, y = q[b, h].double(), k[b, h // (Hq // Hkv)].double()
            x, y = torch.nan_to_num(x) if not see.any() else x, torch.where((j < n)[:, None], y, 0.0)
            s = (x @ y.t()) * scale
            s = torch.where(see, s, -float("inf"))
            l = torch.logsumexp(s, -1)
            out_lse[b, h] = l
            use = l if lse is None else lse[b, h].double()
            p = torch.where(see & torch.isfinite(use)[:, None], torch.exp(s - use[:, None]), 0.0)
            mass[b, h // (Hq // Hkv)] += p.sum(0)
            m = torch.where(see, (x.abs() @ y.abs().t()) * abs(scale), 0.0)
            err = max(err, float(m.max()) if m.numel() else 0.0)
    # a sum of D products in 32 bits, the scale, the exponent's argument and exp2 (2^-22): D + 8 units of 2^-24
    return mass, out_lse, (D + 8) * 2.0 ** -24 * err + 2.0 ** -21


def _check_mass(got, ref, rel, n):
    """A weight is off by its logit's error and its row's log-sum-exp's (the same
    bound), a sum of n weights by n 2^-24 at most."""
    tol = ref * (2 * rel + (n + 4) * 2.0 ** -24) + 1e-30
    err = (got.double() - ref).abs()
    assert got.dtype == torch.float32 and (err <= tol).all(), float((err - tol).max())
    # and far nearer than that bound on the whole: 2-norms within 2e-6
    assert float(err.norm()) <= 2e-6 * float(ref.norm()) + 1e-30


SHAPES = [  # B, Hq, Hkv, D, Tq, Tk
    (1, 4, 4, 64, 1, 1), (2, 8, 1, 64, 1, 300), (3, 6, 2, 128, 1, 129), (1, 32, 4, 64, 5, 5), (2, 4, 2, 128, 31, 200),
    (1, 8, 2, 64, 32, 33), (2, 6, 3, 128, 64, 700), (1, 4, 1, 64, 257, 257), (1, 2, 2, 128, 515, 515),
    (1, 16, 16, 128, 33, 2000), (1, 2, 1, 64, 1100, 1300), (1, 2, 1, 64, 1, 9000), (1, 3, 3, 128, 9, 5000),
    (2, 2, 2, 64, 16, 64), (1, 17, 1, 128, 1, 700),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", SHAPES)
@pytest.mark.parametrize("causal,given", [(True, False), (True, True), (False, False)])
def test_mass(dtype, B, Hq, Hkv, D, Tq, Tk, causal, given):
    import care_kv
    print(f"mass {dtype} B={B} {Hq}/{Hkv} D={D} Tq={Tq} Tk={Tk} causal={causal} lse={given}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(Tq * 7 + Tk)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").to(dtype)
    ref, lse, rel = _mass_ref(q, k, causal)
    got = care_kv.attention_mass(q, k, causal=causal, lse=lse.float() if given else None)
    if given:  # a given log-sum-exp is rounded to 32 bits
        ref, _, _ = _mass_ref(q, k, causal, lse=lse.float())
    _check_mass(got, ref, rel, Hq // Hkv * Tq)
    # each row's weights sum to 1
    assert abs(float(got.double().sum()) / (B * Hq * Tq) - 1) < 1e-5


def test_mass_ragged_starts_and_garbage():
    """Lengths of 0, 1 and inside a block, starts before, inside and behind the
    sequence; NaN and infinities in every masked row of q and k."""
    import care_kv
    B, Hq, Hkv, D, Tq, Tk = 6, 4, 2, 64, 40, 300
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").half()
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").half()
    lengths = [0, 1, 40, 129, 300, 77]
    starts = [0, 0, 0, 89, 290, -10]
    for b, n in enumerate(lengths):
        k[b, :, n:] = float("nan")
        k[b, :, n:, ::2] = float("inf")
    q[0] = float("nan")
    q[5, :, :10] = float("nan")  # positions below 0 see nothing
    for ln, st in ((lengths, starts), (torch.tensor(lengths, device="cuda"), torch.tensor(starts, device="cuda").int())):
        got = care_kv.attention_mass(q, k, lengths=ln, q_start=st)
        qz = torch.nan_to_num(q)
        ref, _, rel = _mass_ref(qz, k, lengths=lengths, q_start=starts)
        assert not torch.isnan(got).any()
        _check_mass(got, ref, rel, 2 * Tq)
        for b, n in enumerate(lengths):
            assert not got[b, :, n:].any()
    got = care_kv.attention_mass(q[4:], k[4:], lengths=lengths[4:], q_start=7, causal=False)
    ref, _, rel = _mass_ref(torch.nan_to_num(q[4:]), k[4:], causal=False, lengths=lengths[4:])
    assert torch.isnan(got[1, :, :77]).all() and not torch.isnan(got[0]).any()  # (not causal: every row counts)
    _check_mass(got[:1], ref[:1], rel, 2 * Tq)


def test_mass_nan_stays_with_the_keys_it_sees():
    import care_kv
    q = torch.randn(1, 1, 200, 64, device="cuda").half()
    k = torch.randn(1, 1, 200, 64, device="cuda").half()
    q[0, 0, 50, 3] = float("nan")
    for lse in (None, torch.zeros(1, 1, 200, device="cuda")):
        got = care_kv.attention_mass(q, k, lse=lse)[0, 0]
        assert torch.isnan(got[:51]).all() and not torch.isnan(got[51:]).any()
    # an infinite lse: the row adds nothing
    lse = torch.zeros(1, 1, 200, device="cuda")
    lse[0, 0, 50] = -float("inf")
    lse[0, 0, 60] = float("inf")
    q[0, 0, 50] = 1.0
    ref, _, rel = _mass_ref(q, k, lse=lse)
    _check_mass(care_kv.attention_mass(q, k, lse=lse), ref, rel, 200)


def test_mass_strides_scale_accumulate():
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(4)
    B, Hq, Hkv, D, T = 2, 6, 2, 128, 150
    q = torch.randn(B, T, Hq, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    k = torch.randn(B, T, 3, Hkv, D, generator=g, device="cuda").bfloat16()[:, :, 1].transpose(1, 2)
    big = torch.full((B, Hkv, T + 60), 3.0, device="cuda")
    out = big[:, :, 10:10 + T]
    for scale in (0.05, -0.11, 0.0):
        out.fill_(3.0)
        got = care_kv.attention_mass(q, k, sm_scale=scale, out=out, accumulate=True)
        assert got.data_ptr() == out.data_ptr()
        ref, _, rel = _mass_ref(q, k, scale=scale)
        tol = (ref + 3) * (2 * rel + 1e-4)
        assert ((got.double() - ref - 3).abs() <= tol).all()
    assert (big[:, :, :10] == 3).all() and (big[:, :, 10 + T:] == 3).all()
    # rows off 16 bytes and values apart are copied first
    odd = torch.randn(B, Hkv, T, D + 1, generator=g, device="cuda").bfloat16()[..., 1:]
    apart = torch.randn(B, Hkv, D, T, generator=g, device="cuda").bfloat16().transpose(2, 3)
    for kk in (odd, apart):
        ref, _, rel = _mass_ref(q, kk)
        _check_mass(care_kv.attention_mass(q, kk), ref, rel, 3 * T)
    one = care_kv.attention_mass(q[0], k[0])
    assert torch.equal(one, care_kv.attention_mass(q, k)[0])


def test_mass_adds_up_over_decode_steps():
    """Single-token calls, each adding to a growing cache's sums, give the mass of
    all rows at once."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(9)
    B, Hq, Hkv, D, T = 2, 8, 2, 64, 45
    q = torch.randn(B, Hq, T, D, generator=g, device="cuda").half()
    k = torch.randn(B, Hkv, T, D, generator=g, device="cuda").half()
    total = torch.zeros(B, Hkv, T, device="cuda")
    for t in range(T):
        care_kv.attention_mass(q[:, :, t:t + 1], k[:, :, :t + 1], out=total[:, :, :t + 1], accumulate=True)
    ref, _, rel = _mass_ref(q, k)
    _check_mass(total, ref, rel, 4 * T)


def test_mass_empty():
    import care_kv
    z = lambda *s: torch.zeros(*s, device="cuda").half()  # noqa: E731
    assert care_kv.attention_mass(z(0, 4, 3, 64), z(0, 2, 9, 64)).shape == (0, 2, 9)
    assert care_kv.attention_mass(z(2, 4, 3, 64), z(2, 2, 0, 64)).shape == (2, 2, 0)
    out = torch.full((2, 2, 9), 5.0, device="cuda")
    assert (care_kv.attention_mass(z(2, 4, 0, 64), z(2, 2, 9, 64), out=out) == 0).all()
    out.fill_(5.0)
    assert (care_kv.attention_mass(z(2, 4, 0, 64), z(2, 2, 9, 64), out=out, accumulate=True) == 5).all()


# ---------------------------------------------------------------- eviction
def _evict_ref(mass, keep, sink, recent, lengths):
    m = mass.detach().cpu().numpy().astype(np.float64)
    B, H, T = m.shape
    keep = min(keep, T)
    index = np.full((B, H, keep), -1, dtype=np.int32)
    for b in range(B):
        n = T if lengths is None else max(0, min(int(lengths[b]), T))
        for h in range(H):
            w = m[b, h, :n].copy()
            low = np.isnan(w)
            w[low] = 0
            sure = np.zeros(n, bool)
            sure[:sink] = True
            sure[max(0, n - recent):] = True
            order = np.lexsort((np.arange(n), -w, low, ~sure))
            sel = np.sort(order[:keep])
            index[b, h, :len(sel)] = sel
    return torch.from_numpy(index)


def _check_evict(care_kv, mass, k, v, keep, sink, recent, lengths):
    got = care_kv.evict_rows(mass, k, v, keep=keep, sink=sink, recent=recent, lengths=lengths)
    ref = _evict_ref(mass, keep, sink, recent, lengths)
    assert torch.equal(got.index.cpu(), ref)
    at, none = got.index.clamp(min=0).long(), got.index < 0
    for x, y in ((k, got.k), (v, got.v)):
        want = torch.take_along_dim(x, at[..., None], 2).masked_fill(none[..., None], 0)
        assert torch.equal(torch.where(torch.isnan(want), 7, want), torch.where(torch.isnan(y), 7, y))
    want = torch.take_along_dim(mass, at, 2).masked_fill(none, 0)
    assert torch.equal(torch.nan_to_num(want, 7), torch.nan_to_num(got.mass, 7))
    T = mass.shape[2]
    n = [T] * mass.shape[0] if lengths is None else [max(0, min(int(x), T)) for x in lengths]
    assert got.lengths.tolist() == [min(x, keep, T) for x in n]
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,T,D,keep,sink,recent", [
    (1, 1, 1, 64, 1, 0, 0), (2, 3, 50, 64, 7, 2, 3), (1, 2, 1024, 128, 128, 4, 32), (2, 2, 1025, 64, 1024, 0, 0),
    (1, 4, 5000, 128, 1300, 4, 0), (2, 1, 8193, 64, 600, 1, 5), (1, 1, 300000, 64, 9000, 4, 100), (1, 1, 600000, 2, 70, 0, 1),
    (3, 1, 333, 6, 332, 100, 232), (1, 1, 20000, 64, 5, 0, 5), (2, 2, 40, 64, 64, 4, 4)])
def test_evict(dtype, B, H, T, D, keep, sink, recent):
    import care_kv
    print(f"evict {dtype} B={B} H={H} T={T} D={D} keep={keep} sink={sink} recent={recent}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + keep)
    mass = torch.exp(3 * torch.randn(B, H, T, generator=g, device="cuda"))
    k, v = (torch.randn(B, H, T, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    _check_evict(care_kv, mass, k, v, keep, sink, recent, None)
    # many equal weights, in every bit range
    for m in (torch.zeros_like(mass), (mass * 2).round() / 2, -mass, mass * 1e-42):
        _check_evict(care_kv, m, k, v, keep, sink, recent, None)


@pytest.mark.parametrize("n_parts", [1, 3, 8])
def test_evict_lengths_and_values(n_parts):
    """Lengths of 0, 1, below, at and above keep; weights of both signs, zeros of
    both signs, infinities and NaN; NaN rows behind a sequence are not read."""
    import care_kv
    B, H, T, D = 6, 2, 2500 * n_parts, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    mass = torch.randn(B, H, T, generator=g, device="cuda")
    mass[:, :, ::3] = 0.0
    mass[:, :, 1::6] = -0.0
    mass[:, :, 5::50] = float("inf")
    mass[:, :, 7::50] = -float("inf")
    mass[:, :, 9::20] = float("nan")
    k, v = (torch.randn(B, H, T, D, generator=g, device="cuda").half() for _ in range(2))
    lengths = [0, 1, 99, 100, 1700, T]
    for b, n in enumerate(lengths):
        mass[b, :, n:] = float("inf")
        k[b, :, n:] = float("nan")
    for keep, sink, recent in ((100, 4, 10), (100, 0, 0), (1600, 0, 800), (100, 50, 50)):
        got = _check_evict(care_kv, mass, k, v, keep, sink, recent, lengths)
        assert not torch.isnan(got.k).any()
        dev = care_kv.evict_rows(mass, k, v, keep=keep, sink=sink, recent=recent,
                                 lengths=torch.tensor(lengths, device="cuda"))
        assert torch.equal(dev.index, got.index)


def test_evict_strides():
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(3)
    B, H, T, D = 2, 3, 700, 64
    mass = torch.rand(B, T, H, generator=g, device="cuda").transpose(1, 2)
    kv = torch.randn(B, T, 2, H, D, generator=g, device="cuda").half()
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    _check_evict(care_kv, mass, k, v, 90, 4, 8, None)
    odd = torch.randn(B, H, T, D + 1, generator=g, device="cuda").half()[..., 1:]      # rows off 4 bytes
    eight = torch.randn(B, H, T, D + 4, generator=g, device="cuda").half()[..., 4:]    # rows on 8 bytes
    _check_evict(care_kv, mass, odd, eight, 90, 4, 8, None)
    one = care_kv.evict_rows(mass[1], k[1], v[1], keep=90, sink=4, recent=8)
    assert torch.equal(one.index.cpu(), _evict_ref(mass[1:], 90, 4, 8, None)[0]) and one.k.shape == (H, 90, D)
    z = torch.zeros(2, 3, 0, 64, device="cuda").half()
    assert care_kv.evict_rows(torch.zeros(2, 3, 0, device="cuda"), z, z, keep=5).lengths.tolist() == [0, 0]


def test_offsets_past_32_bits():
    """Rows of a buffer of 4.6 GB, head 19 of 20: byte offsets past 2^32."""
    import care_kv
    T, H, D = 900_000, 20, 128
    buf = torch.zeros(T, H, D, dtype=torch.float16, device="cuda")
    k = buf[:, 19:20].transpose(0, 1)                        # (1, T, D), rows 5120 bytes apart
    hot = torch.tensor([3, 420_000, 850_001, T - 1], device="cuda")
    q = torch.randn(1, 1, D, device="cuda").half()
    k[0, hot] = 4 * q[0]
    mass = care_kv.attention_mass(q, k)
    ref, _, rel = _mass_ref(q[None], k[None])
    _check_mass(mass[None], ref, rel, 1)
    got = care_kv.evict_rows(mass, k, k, keep=4)
    assert torch.equal(got.index[0].long(), hot) and torch.equal(got.k[0], k[0, hot])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", [(3, 8, 2, 128, 1, 5003), (2, 16, 1, 64, 1, 2500), (2, 3, 3, 128, 5, 4500),
                                              (1, 2, 1, 64, 8, 20000), (70, 8, 8, 64, 1, 8200)])
def test_mass_of_few_rows_on_many_keys(dtype, B, Hq, Hkv, D, Tq, Tk):
    """Decode steps and short windows on long contexts: ragged lengths with NaN behind them, starts of every kind,
    given log-sum-exps, sums added to; the same bits twice."""
    import care_kv
    print(f"mass {dtype} B={B} {Hq}/{Hkv} D={D} Tq={Tq} Tk={Tk}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(Tk)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").to(dtype)
    lengths = ([Tk, 0, 1, Tk - 1, 1025, 64, 65] * 10)[:B]
    starts = [n - Tq if i % 3 < 2 else n // 2 for i, n in enumerate(lengths)]
    for b, n in enumerate(lengths):
        k[b, :, n:] = float("nan")
    ln, st = torch.tensor(lengths, device="cuda"), torch.tensor(starts, device="cuda")
    ref, lse, rel = _mass_ref(q, k, lengths=lengths, q_start=starts)
    n = Hq // Hkv * Tq
    got = care_kv.attention_mass(q, k, lengths=ln, q_start=st)
    _check_mass(got, ref, rel, n)
    assert torch.equal(got, care_kv.attention_mass(q, k, lengths=ln, q_start=st))
    for b, m in enumerate(lengths):
        assert not got[b, :, m:].any()
    out = torch.ones(B, Hkv, Tk + 3, device="cuda")[:, :, 1:Tk + 1]
    care_kv.attention_mass(q, k, lengths=ln, q_start=st, out=out, accumulate=True)
    assert torch.equal(out, got + 1.0)
    with_lse, _, _ = _mass_ref(q, k, lengths=lengths, q_start=starts, lse=lse.float())
    _check_mass(care_kv.attention_mass(q, k, lengths=ln, q_start=st, lse=lse.float()), with_lse, rel, n)
    whole, _, rel = _mass_ref(q[:1], k[:1], causal=False)
    _check_mass(care_kv.attention_mass(q[:1], k[:1], causal=False), whole, rel, n)


@pytest.mark.parametrize("T", [8192, 8193, 12001, 16384, 16385])
@pytest.mark.parametrize("D,keep", [(64, 40), (64, 5000), (6, 300)])
def test_evict_around_one_launch(T, D, keep):
    """The sizes where the keys a thread holds and the launches change; ragged, with equal weights and NaN."""
    import care_kv
    print(f"evict T={T} D={D} keep={keep}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + D)
    mass = torch.randn(4, 3, T, generator=g, device="cuda").mul(4).round()
    mass[:, :, 3::70] = float("nan")
    k, v = (torch.randn(4, 3, T, D, generator=g, device="cuda").half() for _ in range(2))
    for lengths in (None, [T, T - 1, 7, 8200]):
        _check_evict(care_kv, mass, k, v, keep, 4, keep // 4, lengths)
        _check_evict(care_kv, torch.zeros_like(mass), k, v, keep, 0, 0, lengths)


# Each form of the weights' kernels: all scores in LDS, scores to memory, walks over a head's rows, over rows of several
# heads, and 64-row windows whose statistics the walks join.
FORMS = [(2, 4, 2, 64, 3, 300), (1, 8, 2, 128, 2, 5000), (2, 3, 3, 64, 200, 333), (2, 8, 2, 128, 64, 900),
         (3, 12, 3, 64, 9, 700), (1, 2, 1, 128, 700, 700)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", FORMS)
@pytest.mark.parametrize("causal", [True, False])
def test_mass_rows_of_infinite_lse_add_nothing(dtype, B, Hq, Hkv, D, Tq, Tk, causal):
    """Whatever they hold: NaN, infinities, values whose logits are infinite."""
    import care_kv
    print(f"mass {dtype} B={B} {Hq}/{Hkv} D={D} Tq={Tq} Tk={Tk} causal={causal}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(Tq + Tk)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").to(dtype)
    off = torch.rand(B, Hq, Tq, generator=g, device="cuda") < 0.2
    off[0, 0, Tq - 1] = True
    q[off] = 0
    _, lse, _ = _mass_ref(q, k, causal)
    lse = lse.float()
    lse[off] = -float("inf")
    lse[off & (torch.rand(B, Hq, Tq, generator=g, device="cuda") < 0.3)] = float("inf")
    ref, _, rel = _mass_ref(q, k, causal, lse=lse)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).max):
        q[off] = bad
        got = care_kv.attention_mass(q, k, lse=lse, causal=causal)
        _check_mass(got, ref, rel, Hq // Hkv * Tq)


@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", FORMS)
def test_mass_infinite_logits_stay_with_the_keys_they_see(B, Hq, Hkv, D, Tq, Tk):
    """A row without a given lse whose logits pass 32 bits: NaN at every key it sees, as the formula has it, and at no other."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(Tk)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").bfloat16()
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").abs().bfloat16()
    row = Tq // 2
    q[0, 0, row] = torch.finfo(torch.bfloat16).max
    got = care_kv.attention_mass(q, k)
    sees = Tk - Tq + row + 1
    assert torch.isnan(got[0, 0, :sees]).all() and not torch.isnan(got[0, 0, sees:]).any()
    assert not torch.isnan(got[0, 1:]).any() and not torch.isnan(got[1:]).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", [
    (5, 4, 2, 64, 7, 7), (5, 2, 2, 64, 333, 333), (4, 8, 2, 128, 96, 96), (5, 12, 3, 64, 9, 9), (5, 8, 2, 128, 700, 700),
    (5, 4, 2, 64, 3, 300), (4, 8, 2, 128, 4, 5000), (5, 4, 1, 64, 31, 900), (4, 8, 2, 128, 64, 2000), (5, 2, 2, 64, 100, 400)])
@pytest.mark.parametrize("causal,given", [(True, False), (True, True), (False, False), (False, True)])
def test_mass_right_padded_queries(dtype, B, Hq, Hkv, D, Tq, Tk, causal, given):
    """Rows of q behind q_lengths do not vote, and nothing that padded rows of q, k and lse hold is used: each sequence
    is what it is alone.  A prompt (Tq = Tk) takes its lengths for its queries' too."""
    import care_kv
    print(f"mass {dtype} B={B} {Hq}/{Hkv} D={D} Tq={Tq} Tk={Tk} causal={causal} lse={given}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(Tq * 3 + Tk)
    q = torch.randn(B, Hq, Tq, D, generator=g, device="cuda").to(dtype)
    k = torch.randn(B, Hkv, Tk, D, generator=g, device="cuda").to(dtype)
    lengths = [Tk, Tk // 2 + 1, 0, Tk - 1, 1][:B]
    qn = lengths if Tq == Tk else [min(n, m) for n, m in zip([Tq, Tq // 2 + 1, 0, 1, Tq], lengths)]
    ref, lse, rel = torch.zeros(B, Hkv, Tk, dtype=torch.float64, device="cuda"), torch.full((B, Hq, Tq), float("nan")).cuda(), 0.0
    for b, (n, m) in enumerate(zip(lengths, qn)):
        if m:
            x, y = q[b:b + 1, :, :m], k[b:b + 1, :, :n]
            r, l, e = _mass_ref(x, y, causal)
            if given:  # a given log-sum-exp is rounded to 32 bits
                lse[b, :, :m] = l[0].float()
                r, _, _ = _mass_ref(x, y, causal, lse=lse[b:b + 1, :, :m])
            ref[b, :, :n], rel = r[0], max(rel, e)
        q[b, :, m:] = float("nan")
        q[b, :, m:, ::3] = float("inf")
        k[b, :, n:] = float("nan")
    for dev in (False, True):
        ln, ql = (torch.tensor(x, device="cuda") for x in (lengths, qn)) if dev else (lengths, qn)
        kw = dict(lse=lse if given else None, causal=causal, lengths=ln)
        got = care_kv.attention_mass(q, k, q_lengths=ql, **kw)
        _check_mass(got, ref, rel, Hq // Hkv * Tq)
        for b, n in enumerate(lengths):
            assert not got[b, :, n if qn[b] else 0:].any()
        if Tq == Tk:
            assert torch.equal(got, care_kv.attention_mass(q, k, **kw))
        at = [n - m for n, m in zip(lengths, qn)]  # the default start, said
        assert torch.equal(got, care_kv.attention_mass(q, k, q_lengths=ql, q_start=at, **kw))


def test_mass_query_lengths_of_every_kind():
    """Below zero, past the rows, one int for all, with starts of their own."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(3, 4, 40, 64, generator=g, device="cuda").half()
    k = torch.randn(3, 2, 300, 64, generator=g, device="cuda").half()
    got = care_kv.attention_mass(q, k, q_lengths=[-5, 99, 40])
    want = care_kv.attention_mass(q, k)
    assert not got[0].any() and torch.equal(got[1:], want[1:])
    got = care_kv.attention_mass(q, k, q_lengths=17, q_start=[3, 283, -2])
    ref, _, rel = _mass_ref(q[:, :, :17], k, q_start=[3, 283, -2])
    _check_mass(got, ref, rel, 2 * 17)
    assert torch.equal(care_kv.attention_mass(q[0], k[0], q_lengths=17, q_start=3), got[0])


def test_mass_query_lengths_captured():
    """Lengths on the device may change between replays of a captured call, as the tensors may."""
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(12)
    q = torch.randn(3, 4, 200, 64, generator=g, device="cuda").half()
    k = torch.randn(3, 2, 200, 64, generator=g, device="cuda").half()
    n = torch.tensor([200, 50, 120], device="cuda", dtype=torch.int32)
    lse = torch.full((3, 4, 200), 5.0, device="cuda")

    def call():
        return care_kv.attention_mass(q, k, lengths=n), care_kv.attention_mass(q, k, lse=lse, lengths=n, q_lengths=n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn, lens in enumerate(([200, 50, 120], [1, 200, 0], [64, 65, 199], [0, 0, 7])):
        n.copy_(torch.tensor(lens))
        lse[:, :, turn::5] = -float("inf")
        q[:, :, turn::5] = float("nan")
        graph.replay()
        got = [o.clone() for o in out]
        for a, b in zip(got, call()):
            assert torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(b, 7.0))
        assert not torch.isnan(got[1]).any()
