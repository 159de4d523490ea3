"""window_attention against a 64-bit softmax over what each row sees."""
import math

import pytest
import torch

from pages_ref import attend, check, sight

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _inputs(seed, B, Hq, Hkv, D, Tq, Tk, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(B, Hq, Tq, D), r(B, Hkv, Tk, D), r(B, Hkv, Tk, D)


SHAPES = [  # B, Hq, Hkv, D, Tq, Tk
    (1, 1, 1, 64, 1, 1), (2, 4, 4, 128, 1, 33), (1, 8, 1, 64, 1, 5000), (2, 6, 2, 128, 3, 500), (1, 4, 4, 64, 31, 31),
    (2, 4, 2, 128, 130, 130), (1, 3, 1, 64, 333, 333), (1, 2, 2, 128, 70, 900), (1, 7, 1, 64, 40, 4000), (1, 2, 1, 64, 9, 4),
    (3, 5, 5, 64, 64, 65), (1, 2, 2, 128, 1030, 1030),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sink", [(None, 0), (1, 0), (40, 4), (17, 33), (600, 1)])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", SHAPES)
def test_against_64_bits(dtype, window, sink, B, Hq, Hkv, D, Tq, Tk):
    import care_kv
    print(f"window {dtype} w={window} s={sink} B={B} {Hq}/{Hkv} D={D} {Tq} on {Tk}", flush=True)
    q, k, v = _inputs(Tk + Tq, B, Hq, Hkv, D, Tq, Tk, dtype)
    got = care_kv.window_attention(q, k, v, window=window, sink=sink, return_lse=True)
    check(got, attend(q, k, v, sight(B, Tq, Tk, window, sink, [Tk] * B, [Tq] * B, None)))
    assert torch.equal(care_kv.window_attention(q, k, v, window=window, sink=sink), got[0])
    one = care_kv.window_attention(q[0], k[0], v[0], window=window, sink=sink, return_lse=True)
    check((one[0][None], one[1][None]), attend(q[:1], k[:1], v[:1], sight(1, Tq, Tk, window, sink, [Tk], [Tq], None)))
    care_kv.window_attention(q, k, v, window=window, sink=sink, out=q)
    assert torch.equal(q, got[0])


def test_is_the_causal_attention():
    """Without a window, rows alike: prefill_attention's result and log-sum-exp."""
    import care_kv
    q, k, v = _inputs(1, 2, 4, 2, 128, 300, 300, F16)
    a, b = care_kv.window_attention(q, k, v, return_lse=True), care_kv.prefill_attention(q, k, v, return_lse=True)
    ref = attend(q, k, v, sight(2, 300, 300, None, 0, [300] * 2, [300] * 2, None))
    check(a, ref)
    check(b, ref)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sink", [(None, 0), (50, 4), (300, 40)])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (2, 2, 128)])
def test_ragged_prompts(dtype, window, sink, Hq, Hkv, D):
    """Right-padded prompts, NaN and infinities behind them; counts of zero and past the rows."""
    import care_kv
    T = 200
    lengths = [0, 1, 31, 32, 33, 129, T, T + 9]
    B = len(lengths)
    q, k, v = _inputs(5, B, Hq, Hkv, D, T, T, dtype)
    for b, n in enumerate(lengths):
        q[b, :, n:], k[b, :, n:], v[b, :, n:] = math.nan, math.inf, math.nan
    ref = attend(torch.nan_to_num(q), torch.nan_to_num(k, posinf=0), torch.nan_to_num(v),
                 sight(B, T, T, window, sink, lengths, lengths, None))
    for ln in (lengths, torch.tensor(lengths, device="cuda"), torch.tensor(lengths, device="cuda", dtype=torch.int32)):
        check(care_kv.window_attention(q, k, v, window=window, sink=sink, lengths=ln, return_lse=True), ref)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sink", [(None, 0), (20, 2)])
def test_positions(dtype, window, sink):
    """Chunks at their own positions, before the keys, among them and behind them, with counts of their own."""
    import care_kv
    start = [-5, 0, 10, 60, 200, -2 ** 31, 2 ** 31 - 1]
    B, Tq, Tk = len(start), 24, 90
    q, k, v = _inputs(6, B, 6, 2, 64, Tq, Tk, dtype)
    lengths, rows = [90, 90, 30, 90, 90, 90, 90], [24, 24, 24, 7, 24, 24, 24]
    far = [max(-2 ** 29, min(2 ** 29, s)) for s in start]
    got = care_kv.window_attention(q, k, v, window=window, sink=sink, lengths=lengths, q_lengths=rows,
                                   q_start=torch.tensor(start, device="cuda"), return_lse=True)
    check(got, attend(q, k, v, sight(B, Tq, Tk, window, sink, lengths, rows, far)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Tq,Tk,G", [(150, 150, 1), (150, 150, 4), (3, 700, 4), (40, 300, 2)])
def test_not_a_number_where_a_row_does_not_look(dtype, Tq, Tk, G):
    import care_kv
    for which in "kv":
        q, k, v = _inputs(9, 1, 2 * G, 2, 64, Tq, Tk, dtype)
        x = k if which == "k" else v
        x[0, 0, Tk - 2, 7], x[0, 1, Tk // 2, 33], x[0, 1, 2, 0], x[0, 1, Tk // 2 + 1, 33] = math.inf, math.nan, -math.inf, math.inf
        for window, sink in ((None, 0), (20, 0), (20, 3), (130, 0)):
            got = care_kv.window_attention(q, k, v, window=window, sink=sink, return_lse=True)
            see = sight(1, Tq, Tk, window, sink, [Tk], [Tq], None)
            if which == "v":
                check(got, attend(q, k, v, see))
                continue
            ref = attend(q, torch.where(torch.isfinite(k), k, 0.0), v, see)
            for h in range(2):  # rows that do not see such a key
                hit = (see[0] & ~torch.isfinite(k[0, h]).all(-1)).any(-1)
                hs = slice(h * G, (h + 1) * G)
                assert ((got[0].double() - ref[0]).abs() <= ref[2])[0, hs][:, ~hit].all()
                assert ((got[1].double() - ref[1]).abs() <= ref[3])[0, hs][:, ~hit & see[0].any(-1)].all()


def test_nothing_to_see():
    """No sequences, no rows, no keys."""
    import care_kv
    for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 0, 0)):
        q, k, v = _inputs(1, B, 4, 2, 64, Tq, Tk, F16)
        o, lse = care_kv.window_attention(q, k, v, window=4, return_lse=True)
        assert o.shape == q.shape and lse.shape == (B, 4, Tq) and not o.any() and (lse == -math.inf).all()


def test_extreme_logits():
    import care_kv
    q, k, v = _inputs(7, 2, 4, 2, 64, 50, 400, F16)
    see = sight(2, 50, 400, 300, 4, [400] * 2, [50] * 2, None)
    ramp = torch.linspace(0.1, 8, 400, device="cuda")[None, None, :, None]
    for kk in ((k * ramp).half(), (k * ramp.flip(2)).half()):
        for scale in (None, -0.3, 0.0, 1.0):
            check(care_kv.window_attention(q, kk, v, window=300, sink=4, sm_scale=scale, return_lse=True),
                  attend(q, kk, v, see, scale))


def test_strides():
    import care_kv
    g = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    B, T, Hq, Hkv, D = 2, 45, 8, 2, 128
    q = r(B, T, Hq, D).transpose(1, 2)
    kv = r(T, B, 2, Hkv, D)
    k, v = (kv[:, :, i].permute(1, 2, 0, 3) for i in range(2))
    out = torch.full((B, T, Hq, D + 3), 5.0, device="cuda").bfloat16()
    view = out[..., 3:].transpose(1, 2)
    see = sight(B, T, T, 20, 4, [T] * B, [T] * B, None)
    got = care_kv.window_attention(q, k, v, window=20, sink=4, out=view, return_lse=True)
    assert got[0].data_ptr() == view.data_ptr() and (out[..., :3] == 5).all()
    check(got, attend(q, k, v, see))
    odd, apart = r(B, Hkv, T, D + 1)[..., 1:], r(B, Hkv, D, T).transpose(2, 3)
    check(care_kv.window_attention(q, odd, apart, window=20, sink=4, return_lse=True), attend(q, odd, apart, see))
    same = r(B, 1, 1, D).expand(B, Hkv, T, D)
    check(care_kv.window_attention(q, same, same, window=20, sink=4, return_lse=True), attend(q, same, same, see))


def test_offsets_past_32_bits():
    import care_kv
    N, H, D = 900_000, 20, 128
    buf = torch.zeros(1, N, H, D, dtype=F16, device="cuda")   # 4.6 GB
    k = buf[:, :, 18:20].transpose(1, 2)
    q = torch.randn(1, 2, 2, D, device="cuda").half()
    for at in (7, 430_000, N - 3):
        k[0, :, at] = (q[0, :, 0] * 3).half()
    for window in (None, 500_000):
        check(care_kv.window_attention(q, k, k, window=window, sink=8, return_lse=True),
              attend(q, k, k, sight(1, 2, N, window, 8, [N], [2], None)))


def test_takes_part_with_the_others():
    """Its log-sum-exp is what attention_mass and prefix_attention take: a ragged prompt behind a shared prefix."""
    import care_kv
    q, k, v = _inputs(13, 2, 4, 2, 64, 60, 60, BF16)
    g = torch.Generator(device="cuda").manual_seed(2)
    pk, pv = (torch.randn(2, 70, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    lengths = [60, 41]
    own = care_kv.window_attention(q, k, v, lengths=lengths, return_lse=True)
    o, lse = care_kv.prefix_attention(q, pk, pv, own=own, return_lse=True)
    kk, vv = (torch.cat((p.expand(2, -1, -1, -1), x), 2) for p, x in ((pk, k), (pv, v)))
    see = torch.cat((torch.ones(2, 60, 70, dtype=torch.bool, device="cuda"),
                     sight(2, 60, 60, None, 0, lengths, lengths, None)), 2)
    ref = list(attend(q, kk, vv, see))
    ref[2] = 2 * ref[2] + 2.0 ** -8 * ref[0].abs()  # (own's output is rounded before the two are joined)
    check((o[:, :, :41], lse[:, :, :41]), [x[:, :, :41] for x in ref])
    mass = care_kv.attention_mass(q, k, lse=own[1], lengths=lengths)
    total = mass.double().sum(-1)
    want = torch.tensor([60.0, 41.0], device="cuda").double()[:, None] * 2
    assert ((total - want).abs() <= 2.0 ** -8 * want).all()


def test_a_captured_call():
    import care_kv
    q, k, v = _inputs(14, 2, 4, 2, 128, 40, 200, F16)
    lengths = torch.tensor([200, 100], dtype=torch.int32, device="cuda")
    call = lambda: care_kv.window_attention(q, k, v, window=64, sink=4, lengths=lengths, return_lse=True)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in (200, 60, 1, 0, 133):
        lengths[1] = n
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_streams_with_splits():
    """Many rows in a few key splits, values that are not finite in some of them, two streams at once: each call's own."""
    import care_kv
    q, k, v = _inputs(15, 2, 24, 24, 64, 300, 2000, F16)
    v[0, 3, 1990, 5], v[1, 2, 600, 9] = math.inf, math.nan
    lengths, rows = [2000, 1203], [300, 299]
    dev = torch.tensor([lengths, rows], dtype=torch.int32, device="cuda")
    call = lambda x: care_kv.window_attention(x, k, v, window=1500, sink=3, lengths=dev[0], q_lengths=dev[1],  # noqa: E731
                                              return_lse=True)
    check(call(q), attend(q, k, v, sight(2, 300, 2000, 1500, 3, lengths, rows, None)))
    xs = [q * (1 + 0.1 * i) for i in range(6)]
    want = [call(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None] * 6
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = call(x)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(a[0]), torch.nan_to_num(b[0])) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,Hkv,D,Tq,Tk", [(1, 4, 2, 64, 1, 300), (2, 4, 2, 64, 3, 5000), (1, 2, 2, 128, 5, 2000),
                                              (1, 4, 2, 64, 130, 130), (1, 2, 2, 128, 40, 700), (2, 4, 1, 64, 60, 3000),
                                              (1, 8, 1, 128, 30, 9000)])
def test_infinite_values_of_small_weight(dtype, B, Hq, Hkv, D, Tq, Tk):
    """An infinity that a row sees is its result however small its weight: before the key that outweighs it by 2^250 or
    behind it, in its tile, in another wave's keys, in another split."""
    import care_kv
    q, k, v = _inputs(21, B, Hq, Hkv, D, Tq, Tk, dtype)
    u = torch.ones(D, device="cuda")
    u[::3] = -1
    q = (0.5 * q + 2 * u).to(dtype)
    # the strong keys' logits: 2 |u|^2 a / sqrt(D) = 180 with a deviation of 0.5 |u| a / sqrt(D)
    a = 90 / D ** 0.5
    see = sight(B, Tq, Tk, None, 0, [Tk] * B, [Tq] * B, None)
    first = Tk - Tq
    for odd, strong in ((2, 5), (5, 2), (3, 40), (40, 3), (10, 75), (75, 10), (20, Tk // 2), (Tk // 2, 20), (first + 1, 1),
                        (1, first + Tq // 2)):
        if odd == strong or max(odd, strong) >= Tk:
            continue
        kk, vv = k.clone(), v.clone()
        kk[:, :, strong] = (a * u).to(dtype)
        vv[:, :, odd, 7], vv[0, 0, odd, 20], vv[:, :, odd, D - 1] = math.inf, -math.inf, math.nan
        ref = attend(q, kk, vv, see)
        assert float(ref[1].max()) > 150
        print(f"{dtype} {B} {Hq}/{Hkv} D={D} {Tq} on {Tk}: infinite {odd}, strong {strong}", flush=True)
        check(care_kv.window_attention(q, kk, vv, return_lse=True), ref)
    vv = v.clone()  # infinities of both signs: no number
    kk[:, :, Tk // 2] = (a * u).to(dtype)
    vv[:, :, 1, 3], vv[:, :, Tk // 3, 3], vv[:, :, Tk // 3, 4] = math.inf, -math.inf, -math.inf
    check(care_kv.window_attention(q, kk, vv, return_lse=True), attend(q, kk, vv, see))


@pytest.mark.parametrize("Tq", [2, 40])
def test_a_captured_call_with_splits(Tq):
    """Two launches and a workspace in a graph: lengths that move between replays, eager calls among them."""
    import care_kv
    q, k, v = _inputs(16, 2, 4, 2, 64, Tq, 6000, F16)
    lengths = torch.tensor([6000, 100], dtype=torch.int32, device="cuda")
    call = lambda: care_kv.window_attention(q, k, v, window=5000, sink=4, lengths=lengths, return_lse=True)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in (6000, 60, 3001, 0, 133):
        lengths[1] = n
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        check(out, attend(q, k, v, sight(2, Tq, 6000, 5000, 4, [6000, n], [Tq] * 2, None)))
