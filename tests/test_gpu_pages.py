"""append_pages and paged_attention against plain forms in 64 bits: bytes of the
pages, values, masks, what lies where no row looks."""
import math

import pytest
import torch

from pages_ref import attend, check, round4, sight, turn, unpack

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return g, lambda *s: torch.randn(*s, generator=g, device="cuda")


def _table(B, n, g, extra=3):
    """A pool with more pages than the tables name, in any order."""
    return torch.randperm(B * n + extra, generator=g, device="cuda")[:B * n].view(B, n).to(torch.int32), B * n + extra


def _pool(care_kv, n, H, D, seed=None):
    pages = care_kv.int4_pages(n, H, D)
    if seed is None:
        return pages
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages.data.copy_(torch.randint(0, 256, pages.data.shape, generator=g, device="cuda", dtype=torch.uint8))
    return pages


def _fill(care_kv, K, V, table, n_pages):
    pages = _pool(care_kv, n_pages, K.shape[1], K.shape[3], 99)  # (random bytes where nothing is written)
    care_kv.append_pages(pages, table, 0, K, V)
    return pages


def _check_rows(pages, table, start, counts, K, V, before):
    """Every written row's codes and scales, and every other byte as it was."""
    B, H, T, D = K.shape
    (kc, ks, _), (vc, vs, _) = round4(K), round4(V)
    want = _pool_like(pages, before)
    seen = set()
    for b in range(B):
        for slot in range(max(0, start[b]), start[b] + counts[b]):
            at = slot // 16
            page = int(table[b, at]) if at < table.shape[1] else -1
            if 0 <= page < pages.n_pages:
                seen.add((page, b, at))
    touched = torch.zeros_like(pages.data, dtype=torch.bool)
    for page, b, at in seen:
        touched[page] = True
        for h in range(H):
            got, old = unpack(pages, page, h), unpack(want, page, h)
            for i in range(16):
                t = 16 * at + i - start[b]
                new = 0 <= t < counts[b]
                for got_x, old_x, x in zip(got, old, (kc, ks, vc, vs)):
                    w = x[b, h, t].cpu().to(got_x.dtype) if new else old_x[i]
                    same = torch.equal(got_x[i], w) if w.dtype != F16 else torch.equal(
                        torch.nan_to_num(got_x[i].float(), nan=-1.0), torch.nan_to_num(w.float(), nan=-1.0))
                    assert same, f"sequence {b} head {h} place {16 * at + i} (new: {new})"
    assert torch.equal(pages.data[~touched], before[~touched])


def _pool_like(pages, data):
    import care_kv
    return care_kv.Int4Pages(data, pages.head_dim)


APPENDS = [  # B, Hq, Hkv, D, T, R, layout, start, counts
    (1, 1, 1, 64, 1, 64, "half", [0], None), (1, 4, 2, 128, 1, 128, "half", [17], None),
    (2, 8, 1, 64, 5, 32, "interleaved", [3, 30], [5, 2]), (3, 6, 2, 128, 7, 64, "half", [0, 15, 33], [7, 0, 3]),
    (2, 2, 2, 128, 40, 20, "half", [5, 8], [40, 33]), (1, 3, 3, 64, 33, 2, "interleaved", [1], None),
    (2, 5, 1, 64, 9, 12, "half", [7, 16], None), (1, 2, 1, 128, 16, 6, "interleaved", [16], None),
    (4, 4, 4, 64, 3, 64, "half", [0, 1, 2, 3], [3, 2, 1, 0]),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,Hq,Hkv,D,T,R,layout,start,counts", APPENDS)
def test_append(dtype, B, Hq, Hkv, D, T, R, layout, start, counts):
    import care_kv
    print(f"append {dtype} B={B} {Hq}/{Hkv} D={D} T={T} R={R} {layout} {start} {counts}", flush=True)
    g, r = _gen(T + D)
    q, k, v = (r(B, T, h, D).to(dtype).transpose(1, 2) for h in (Hq, Hkv, Hkv))
    plan = care_kv.rotary_plan(R, layout=layout, scale=1.25)
    table, n = _table(B, (max(start) + T + 15) // 16, g)
    pages = _pool(care_kv, n, Hkv, D, 5)
    before = pages.data.clone()
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    out, kh, vh = care_kv.append_pages(pages, table, st, k, v, q=q, plan=plan, counts=counts, return_hat=True)
    at = st.long()[:, None] + torch.arange(T, device="cuda")
    cnt = [T] * B if counts is None else counts
    assert torch.equal(out, turn(q, at, plan).to(dtype)) and out.is_contiguous()
    K, V = turn(k, at, plan).half(), v.float().half()
    _check_rows(pages, table, start, cnt, K, V, before)
    there = (torch.arange(T, device="cuda") < torch.tensor(cnt, device="cuda")[:, None])[:, None, :, None]
    for got, x in ((kh, K), (vh, V)):
        assert torch.equal(got, torch.where(there, round4(x)[2], 0.0))
    # the same again, token by token: the same bytes
    twice = _pool_like(pages, before.clone())
    for t in range(T):
        care_kv.append_pages(twice, table, st + t, k[:, :, t:t + 1], v[:, :, t:t + 1], plan=plan,
                             counts=[int(t < c) for c in cnt])
    assert torch.equal(twice.data, pages.data)


def test_append_values():
    """Zeros, subnormals, the largest, values that are not finite, bf16 beyond fp16."""
    import care_kv
    H, D, T = 2, 64, 6
    for dtype in (F16, BF16):
        g, r = _gen(1)
        k, v = r(1, H, T, D).to(dtype), r(1, H, T, D).to(dtype)
        k[0, 0, 0] = 0
        k[0, 0, 1] *= 2.0 ** -20
        v[0, 0, 2] = 65504 if dtype == F16 else 65280
        k[0, 1, 3, 5] = math.inf
        v[0, 1, 4, 40] = math.nan
        v[0, 0, 5, 0] = -math.inf if dtype == F16 else 1e6
        v[0, 0, 1, :32] = 2.0 ** -24
        pages = _pool(care_kv, 2, H, D, 3)
        before = pages.data.clone()
        table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
        _, kh, vh = care_kv.append_pages(pages, table, 2, k, v, return_hat=True)
        _check_rows(pages, table, [2], [T], k.float().half(), v.float().half(), before)
        for got, x in ((kh, k), (vh, v)):
            want = round4(x.float().half())[2]
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert torch.isnan(kh[0, 1, 3, :32]).all() and not torch.isnan(kh[0, 1, 3, 32:]).any()


def test_append_is_quantize_rows():
    """What the rows stand for is dequantize_rows of quantize_rows."""
    import care_kv
    g, r = _gen(4)
    k, v = (3 * r(2, 4, 50, 128)).half(), r(2, 4, 50, 128).half()
    table, n = _table(2, 4, g)
    _, kh, vh = care_kv.append_pages(care_kv.int4_pages(n, 4, 128), table, 0, k, v, return_hat=True)
    assert torch.equal(kh, care_kv.quant_dequant(k, 4)) and torch.equal(vh, care_kv.quant_dequant(v, 4))


def test_append_positions():
    import care_kv
    g, r = _gen(8)
    B, H, T, D = 3, 2, 5, 64
    q, k, v = (r(B, H, T, D).half() for _ in range(3))
    plan = care_kv.rotary_plan(64, base=500000.0)
    table, n = _table(B, 2, g)
    at = torch.randint(0, 1 << 20, (B, T), generator=g, device="cuda")
    for pos in (at, at.int(), at[:1], at[0], at.t().contiguous().t(), -at, at + (1 << 31)):
        pages = care_kv.int4_pages(n, H, D)
        before = pages.data.clone()
        out = care_kv.append_pages(pages, table, 3, k, v, q=q, plan=plan, positions=pos)
        p = (pos if pos.dim() == 2 else pos[None]).expand(B, T)
        assert torch.equal(out, turn(q, p, plan).half())
        _check_rows(pages, table, [3] * B, [T] * B, turn(k, p, plan).half(), v, before)


def test_append_strides():
    import care_kv
    g, r = _gen(9)
    B, H, T, D = 2, 3, 6, 128
    plan = care_kv.rotary_plan(64)
    qkv = r(B, T, 5, H, D).bfloat16()  # a fused projection, q of twice the heads
    q, k, v = qkv[:, :, :2].flatten(2, 3).transpose(1, 2), qkv[:, :, 3].transpose(1, 2), qkv[:, :, 4].transpose(1, 2)
    table, n = _table(B, 3, g)
    wide = torch.full((B, 7), -9, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = table
    forms = [(q, k, v, table), (q.contiguous(), k.contiguous(), v.contiguous(), wide[:, 2:5])]
    odd = [torch.empty(*x.shape[:3], D + 1, dtype=x.dtype, device="cuda")[..., 1:].copy_(x) for x in (q, k, v)]
    apart = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)]
    forms += [(*odd, table), (*apart, table.t().contiguous().t())]
    ref = None
    for q, k, v, tb in forms:
        pages = care_kv.int4_pages(n, H, D)
        out = care_kv.append_pages(pages, tb, [4, 9], k, v, q=q, plan=plan)
        ref = ref or (out, pages.data)
        assert torch.equal(out, ref[0]) and torch.equal(pages.data, ref[1])


def test_pages_that_are_not_there():
    """Tokens on pages outside the pool, before place 0 and behind the table are dropped."""
    import care_kv
    g, r = _gen(2)
    B, H, T, D = 5, 2, 40, 64
    k, v = r(B, H, T, D).half(), r(B, H, T, D).half()
    pages = _pool(care_kv, 12, H, D, 6)
    before = pages.data.clone()
    table = torch.tensor([[0, 1, 2], [-1, 3, 12], [4, -2 ** 31, 5], [6, 7, 8], [9, 10, 2 ** 31 - 1]], dtype=torch.int32,
                         device="cuda")
    start = [20, 0, 3, -7, 2 ** 31 - 1]
    care_kv.append_pages(pages, table, start, k, v)
    _check_rows(pages, table, [20, 0, 3, -7, 48], [T, T, T, T, 0], k, v, before)
    o, lse = care_kv.paged_attention(r(B, 4, 3, D).half(), pages, table[:, :0], 5, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    none = care_kv.int4_pages(0, H, D)
    care_kv.append_pages(none, table, 0, k, v)
    o = care_kv.paged_attention(r(B, 4, 3, D).half(), none, table, 5)
    assert not o.any()


def test_nothing_to_do():
    """No sequences, no tokens, no heads of q."""
    import care_kv
    pages, h = care_kv.int4_pages(4, 2, 64), lambda *s: torch.zeros(*s, dtype=F16, device="cuda")
    before = pages.data.clone()
    for B, T in ((0, 3), (2, 0), (0, 0)):
        table = torch.zeros(B, 2, dtype=torch.int32, device="cuda")
        out, kh, vh = care_kv.append_pages(pages, table, 0, h(B, 2, T, 64), h(B, 2, T, 64), q=h(B, 4, T, 64), return_hat=True)
        assert out.shape == (B, 4, T, 64) and kh.shape == vh.shape == (B, 2, T, 64)
        o, lse = care_kv.paged_attention(h(B, 4, T, 64), pages, table, 0, return_lse=True)
        assert o.shape == (B, 4, T, 64) and lse.shape == (B, 4, T)
    assert torch.equal(pages.data, before)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    assert care_kv.append_pages(pages, table, 0, h(1, 2, 1, 64), h(1, 2, 1, 64)) is None
    o, lse = care_kv.paged_attention(h(1, 4, 3, 64), pages, table, 0, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()


def _case(seed, B, Hq, Hkv, D, T, N, dtype, mul=1.0):
    import care_kv
    g, r = _gen(seed)
    K, V = (mul * r(B, Hkv, N, D)).half(), r(B, Hkv, N, D).half()
    table, n = _table(B, (N + 15) // 16, g)
    return r(B, Hq, T, D).to(dtype), _fill(care_kv, K, V, table, n), table, round4(K)[2], round4(V)[2]


SHAPES = [  # B, Hq, Hkv, D, T, N
    (1, 1, 1, 64, 1, 1), (1, 4, 4, 128, 1, 33), (2, 8, 1, 64, 1, 500), (4, 32, 4, 64, 1, 1000), (3, 6, 2, 128, 1, 2049),
    (1, 2, 1, 128, 5, 31), (5, 7, 7, 64, 3, 32), (2, 16, 1, 128, 2, 257), (2, 4, 2, 128, 45, 700), (1, 16, 1, 64, 1, 9000),
    (1, 3, 1, 64, 70, 70), (2, 40, 1, 128, 1, 100), (1, 4, 1, 128, 20, 5000),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sink", [(None, 0), (1, 0), (40, 4), (17, 33), (600, 1)])
@pytest.mark.parametrize("B,Hq,Hkv,D,T,N", SHAPES)
def test_paged(dtype, window, sink, B, Hq, Hkv, D, T, N):
    import care_kv
    print(f"paged {dtype} w={window} s={sink} B={B} {Hq}/{Hkv} D={D} T={T} N={N}", flush=True)
    q, pages, table, K, V = _case(N + T, B, Hq, Hkv, D, T, N, dtype)
    got = care_kv.paged_attention(q, pages, table, N, window=window, sink=sink, return_lse=True)
    see = sight(B, T, N, window, sink, [N] * B, [T] * B, None)
    check(got, attend(q, K, V, see, weights=F16))
    again = care_kv.paged_attention(q, pages, table, N, window=window, sink=sink)
    assert torch.equal(again, got[0])
    if T == 1:
        one = care_kv.paged_attention(q[:, :, 0], pages, table, N, window=window, sink=sink, return_lse=True)
        assert torch.equal(one[0], got[0][:, :, 0]) and torch.equal(one[1], got[1][:, :, 0])
    care_kv.paged_attention(q, pages, table, N, window=window, sink=sink, out=q)
    assert torch.equal(q, got[0])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("window,sink", [(None, 0), (50, 4)])
@pytest.mark.parametrize("Hq,Hkv,D,T", [(8, 2, 64, 1), (4, 4, 128, 6), (8, 2, 64, 12), (9, 3, 128, 21), (6, 1, 128, 30)])
def test_ragged(dtype, window, sink, Hq, Hkv, D, T):
    """Lengths of zero and one, before a page's end, past the table; rows of padding; pages that are not there."""
    import care_kv
    N = 333
    lengths = [0, 1, 5, 16, 200, N, 400]
    rows = [T, 1, T, 0, max(1, T // 2), T, T + 4]
    B = len(lengths)
    q, pages, table, K, V = _case(3, B, Hq, Hkv, D, T, 336, dtype)
    table[5, 3], table[6, 0], table[4, 12] = -1, pages.n_pages, -5
    ln, ql = (torch.tensor(x, device="cuda", dtype=t) for x, t in ((lengths, torch.int32), (rows, torch.int64)))
    q[2, :, min(T, 5):] = math.nan if T > 5 else 0
    for b, n in enumerate(rows):
        q[b, :, n:] = math.nan
    see = sight(B, T, 336, window, sink, lengths, rows, None)
    see[5, :, 48:64], see[6, :, :16], see[4, :, 192:208] = False, False, False
    qq = q.clone()
    for b, n in enumerate(rows):
        qq[b, :, n:] = 0
    nan_rows = torch.isnan(qq).any(-1)
    qq = torch.nan_to_num(qq)
    got = care_kv.paged_attention(q, pages, table, ln, q_lengths=ql, window=window, sink=sink, return_lse=True)
    ref = attend(qq, K, V, see, weights=F16)
    # rows that are NaN themselves: NaN where they see anything
    some = see.any(-1)[:, None] & nan_rows
    ref[0][some], ref[1][some] = math.nan, math.nan
    check(got, ref)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(1, 4), (12, 1), (16, 3), (40, 3)])
def test_not_a_number_where_a_row_does_not_look(D, T, G):
    """Values that are not finite at single tokens: the rows that see them are NaN there, the others untouched."""
    import care_kv
    g, r = _gen(21)
    N, H = 150, 2
    for which in "kv":
        K, V = r(1, H, N, D).half(), r(1, H, N, D).half()
        x = K if which == "k" else V
        x[0, 0, N - 3, 7] = math.inf
        x[0, 1, 40, 33] = math.nan
        x[0, 1, 2, 0] = -math.inf
        table, n = _table(1, 10, g)
        pages = _fill(care_kv, K, V, table, n)
        q = r(1, G * H, T, D).half()
        for window, sink in ((None, 0), (20, 0), (20, 3), (130, 0)):
            got = care_kv.paged_attention(q, pages, table, N, window=window, sink=sink, return_lse=True)
            see = sight(1, T, N, window, sink, [N], [T], None)
            if which == "v":
                check(got, attend(q, round4(K)[2], round4(V)[2], see, weights=F16))
                continue
            for h in range(H):  # a key that is no number: every row that sees it
                bad = torch.isnan(round4(K)[2][0, h]).any(-1)
                hit = (see[0] & bad).any(-1)
                hs = slice(h * G, (h + 1) * G)
                assert torch.isnan(got[0][0, hs][:, hit]).all() and torch.isnan(got[1][0, hs][:, hit]).all()
                assert torch.isfinite(got[0][0, hs][:, ~hit]).all()
            fine = ~torch.isnan(got[1])
            ref = attend(q, torch.nan_to_num(round4(K)[2]), round4(V)[2], see, weights=F16)
            assert ((got[0].double() - ref[0]).abs() <= ref[2])[fine].all()


def test_scales_of_q():
    """bf16 queries far beyond fp16 and far below it, negative and zero scales, logits of some hundreds."""
    import care_kv
    q, pages, table, K, V = _case(31, 2, 4, 2, 64, 3, 300, BF16, mul=0.5)
    see = sight(2, 3, 300, None, 0, [300] * 2, [3] * 2, None)
    for mul, scale in ((1.0, -0.3), (1.0, 0.0), (3e5, 2e-6), (2.0 ** -100, 2.0 ** 98), (40.0, 1.0)):
        x = (q * mul).bfloat16()
        x[1, 0, 0] = 0
        check(care_kv.paged_attention(x, pages, table, 300, sm_scale=scale, return_lse=True),
              attend(x, K, V, see, scale, F16))
    x = (q * 30).half()
    check(care_kv.paged_attention(x, pages, table, 300, return_lse=True), attend(x, K, V, see, weights=F16))


@pytest.mark.parametrize("T", [3, 70])
def test_the_smallest_values_of_q(T):
    """bf16 rows of 2^-133 under a small scale: the factor of their logits is below what 32 bits hold, every weight 1."""
    import care_kv
    q, pages, table, K, V = _case(33, 2, 4, 2, 64, T, 150, BF16)
    x = torch.where(q > 0, 2.0 ** -133, -2.0 ** -133).bfloat16()
    lengths, rows = [150, 101], [T, T - 2]
    see = sight(2, T, 150, 40, 3, lengths, rows, None)
    check(care_kv.paged_attention(x, pages, table, lengths, q_lengths=rows, window=40, sink=3, sm_scale=1e-3, return_lse=True),
          attend(x, K, V, see, 1e-3, F16))


def test_strides_of_q():
    import care_kv
    q, pages, table, K, V = _case(32, 2, 6, 2, 128, 5, 90, BF16)
    ref = care_kv.paged_attention(q, pages, table, 90, return_lse=True)
    out = torch.full((2, 5, 6, 131), 3.0, device="cuda").bfloat16()
    view = out[..., 3:].transpose(1, 2)
    a = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(2, 6, 5, 129, device="cuda", dtype=BF16)[..., 1:].copy_(q)
    wide = torch.full((2, 11), 7, device="cuda", dtype=torch.int32)
    wide[:, 5:] = table
    for x, tb, kw in ((a, table, {}), (odd, wide[:, 5:], dict(out=view)), (q.transpose(2, 3).contiguous().transpose(2, 3), table, {})):
        got = care_kv.paged_attention(x, pages, tb, 90, return_lse=True, **kw)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert (out[..., :3] == 3).all()


def test_offsets_past_32_bits():
    """A pool of 5.5 GB, the pages of a sequence at its ends."""
    import care_kv
    H, D, N = 8, 128, 100
    pages = care_kv.int4_pages(300_000, H, D)
    table = torch.tensor([[299_999, 0, 250_000, 1, 299_998, 150_000, 5]], dtype=torch.int32, device="cuda")
    g, r = _gen(40)
    K, V = r(1, H, N, D).half(), r(1, H, N, D).half()
    care_kv.append_pages(pages, table, 0, K, V)
    q = r(1, H, 2, D).half()
    see = sight(1, 2, N, None, 0, [N], [2], None)
    check(care_kv.paged_attention(q, pages, table, N, return_lse=True), attend(q, round4(K)[2], round4(V)[2], see, weights=F16))


def test_streams_and_graphs():
    """A stream of its own; a captured step whose lengths move on the device, replayed among eager work, two graphs at once."""
    import care_kv
    g, r = _gen(50)
    B, Hq, Hkv, D, T, P = 3, 8, 2, 64, 2, 8
    plan = care_kv.rotary_plan(D)
    table, n = _table(B, P, g)
    qs, ks, vs = (r(20, B, h, T, D).half() for h in (Hq, Hkv, Hkv))

    def make():
        return care_kv.int4_pages(n, Hkv, D), torch.tensor([0, 3, 17], dtype=torch.int32, device="cuda")

    def step(pages, length, q, k, v):
        q = care_kv.append_pages(pages, table, length, k, v, q=q, plan=plan)
        length += T
        return care_kv.paged_attention(q, pages, table, length, window=30, sink=2, return_lse=True)
    pages, length = make()
    eager = [step(pages, length, qs[i], ks[i], vs[i]) for i in range(20)]
    side = torch.cuda.Stream()
    other, length2 = make()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(other, length2, qs[i], ks[i], vs[i]) for i in range(20)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for x, y in zip(eager, got) for a, b in zip(x, y))
    assert torch.equal(pages.data, other.data)
    graphs = []
    for _ in range(2):
        pg, ln = make()
        ins = [x[0].clone() for x in (qs, ks, vs)]
        step(pg, ln, *ins)  # once eagerly: loads the kernels
        ln.copy_(torch.tensor([0, 3, 17]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(pg, ln, *ins)
        ln.copy_(torch.tensor([0, 3, 17]))
        graphs.append((graph, ins, out, ln, pg))
    for i in range(20):
        for graph, ins, out, ln, pg in graphs:
            for x, y in zip(ins, (qs, ks, vs)):
                x.copy_(y[i])
            graph.replay()
            step(*make(), qs[i], ks[i], vs[i])  # eager work between the replays
            assert torch.equal(out[0], eager[i][0]) and torch.equal(out[1], eager[i][1]), f"replay {i}"
    torch.cuda.synchronize()
    assert all(torch.equal(pg.data, pages.data) for *_, pg in graphs)


def test_two_streams_with_splits():
    """Many rows in a few key splits, groups that stand for NaN in some of them, two streams at once."""
    import care_kv
    g, r = _gen(60)
    B, H, D, T, N = 2, 24, 64, 150, 3000
    table, n = _table(B, -(-N // 16), g)
    K, V = r(B, H, N, D).half(), r(B, H, N, D).half()
    V[0, 3, 2990, 5], V[1, 2, 600, 9] = math.inf, math.nan
    pages = _fill(care_kv, K, V, table, n)
    q = r(B, H, T, D).half()
    lengths, rows = [N, 1203], [T, T - 1]
    dev = torch.tensor([lengths, rows], dtype=torch.int32, device="cuda")
    call = lambda x: care_kv.paged_attention(x, pages, table, dev[0], q_lengths=dev[1], window=2500, sink=3,  # noqa: E731
                                             return_lse=True)
    see = sight(B, T, N, 2500, 3, lengths, rows, None)
    check(call(q), attend(q, round4(K)[2], round4(V)[2], see, weights=F16))
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
@pytest.mark.parametrize("Hq,Hkv,D,T", [(4, 2, 64, 1), (8, 2, 128, 5), (8, 1, 64, 5), (2, 2, 128, 80)])
def test_captured_attention_with_splits(dtype, Hq, Hkv, D, T):
    """Tables much wider than the text, splits, workspace and join in a graph: lengths that move between replays, eager
    calls among them, two graphs at once."""
    import care_kv
    B, N = 2, 1500
    q, pages, short, K, V = _case(71, B, Hq, Hkv, D, T, N, dtype)
    table = torch.full((B, 700), -1, dtype=torch.int32, device="cuda")
    table[:, :short.shape[1]] = short
    lengths = torch.tensor([N, 100], dtype=torch.int32, device="cuda")
    call = lambda x: care_kv.paged_attention(x, pages, table, lengths, window=1200, sink=4, return_lse=True)  # noqa: E731
    call(q)
    graphs = []
    for i in range(2):
        x = q.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(x)
        graphs.append((graph, x, out))
    for n in (N, T, 777, 0, 1030):
        lengths[1] = n
        for graph, x, out in graphs:
            x.copy_(torch.randn(x.shape, device="cuda"))
            graph.replay()
        for graph, x, out in graphs:
            want = call(x)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
            check(out, attend(x, K, V, sight(B, T, N, 1200, 4, [N, n], [T] * B, None), weights=F16))
