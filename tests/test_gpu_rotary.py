"""rotate_heads against the definition in 64 bits, and its forms: layouts, part
of a head, strides, in place, positions that are far, negative or repeated."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")


def _ref(x, pos, plan, inverse=False):
    """(rotated, sum of magnitudes) in 64 bits: x (B, H, T, D), pos (B, T)."""
    r = plan.rotary_dim
    w = x.double()
    t = pos.double()[:, None, :, None] * plan.freqs * (-1 if inverse else 1)
    c, s = torch.cos(t), torch.sin(t)
    a, b = (w[..., :r // 2], w[..., r // 2:r]) if plan.layout == "half" else (w[..., 0:r:2], w[..., 1:r:2])
    y, mag = w.clone(), torch.zeros_like(w)
    ya, yb, m = plan.scale * (a * c - b * s), plan.scale * (b * c + a * s), plan.scale * (a.abs() + b.abs())
    if plan.layout == "half":
        y[..., :r // 2], y[..., r // 2:r], mag[..., :r // 2], mag[..., r // 2:r] = ya, yb, m, m
    else:
        y[..., 0:r:2], y[..., 1:r:2], mag[..., 0:r:2], mag[..., 1:r:2] = ya, yb, m, m
    return y, mag


def _check(got, x, pos, plan, inverse=False):
    """Half a rounding of the result's type, and 32-bit angles and products: the
    reduced angle 2 pi 2^-26 off, sine and cosine 2 units of 2^-24 (4 units of
    2^-25 at most 1), scale and products 3 more: 8 x 2^-24 of |x1| + |x2|; the
    smallest fp16 step is 2^-24."""
    ref, mag = _ref(x, pos, plan, inverse)
    tol = ref.abs() * torch.finfo(x.dtype).eps / 2 + mag * 8 * 2.0 ** -24 + \
        (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    tol = tol * (1 + 1e-3)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err - tol).max())
    r = plan.rotary_dim
    assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R", [(1, 1, 32, 4, 64, 64), (2, 7, 6, 2, 128, 64), (3, 130, 5, 5, 128, 128),
                                            (1, 9, 4, 1, 64, 16), (2, 5, 3, 1, 80, 20), (1, 3, 2, 2, 6, 2),
                                            (1, 33, 8, 0, 96, 96)])
def test_against_64_bits(dtype, layout, B, T, Hq, Hkv, D, R):
    import care_kv
    print(f"rotary {dtype} {layout} B={B} T={T} {Hq}/{Hkv} D={D} R={R}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + D)
    q = torch.randn(B, T, Hq, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    k = torch.randn(B, Hkv, T, D, generator=g, device="cuda").to(dtype) if Hkv else None
    pos = torch.randint(-5, 5000, (B, T), generator=g, device="cuda")
    plan = care_kv.rotary_plan(R, layout=layout)
    qo, ko = care_kv.rotate_heads(q, k, pos, plan)
    assert qo.is_contiguous() and qo.dtype == dtype
    _check(qo, q, pos, plan)
    if k is None:
        assert ko is None
    else:
        _check(ko, k, pos, plan)
    back, _ = care_kv.rotate_heads(qo, None, pos.to(torch.int32), plan, inverse=True)
    _check(back, qo, pos, plan, inverse=True)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn", "bands"])
def test_far_positions_and_scalings(scaling):
    """Positions up to 2^40: the angle is reduced in 64 bits, off by 2^-53 of the
    turns, 2^40 / 2 pi, that is below the 2^-26 the tolerance counts for base
    angles of 1 down."""
    import care_kv
    plan = care_kv.rotary_plan(64, 500000.0, layout="half", scaling=scaling, factor=1.0 if scaling == "none" else 8.0,
                               original_len=4096)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1, 2, 6, 64, generator=g, device="cuda")
    pos = torch.tensor([[0, 1, 4095, 131072, 2 ** 31 + 5, -2 ** 24 - 1]], device="cuda")
    _check(care_kv.rotate_heads(x, None, pos, plan)[0], x, pos, plan)


def test_plan_formulas():
    """Each scaling at its ends: the fastest pair kept, the slowest divided by
    the factor (ntk, yarn, bands), every pair divided (linear)."""
    import care_kv
    base = care_kv.rotary_plan(128).freqs.cpu()
    assert torch.allclose(base, torch.tensor([10000.0 ** (-i / 64) for i in range(64)], dtype=torch.float64), rtol=1e-14)
    lin = care_kv.rotary_plan(128, scaling="linear", factor=4.0).freqs.cpu()
    assert torch.allclose(lin, base / 4, rtol=1e-14)
    for sc in ("ntk", "yarn", "bands"):
        p = care_kv.rotary_plan(128, scaling=sc, factor=8.0, original_len=4096)
        f = p.freqs.cpu()
        assert math.isclose(f[0], 1.0, rel_tol=1e-12) and math.isclose(f[-1], base[-1] / 8, rel_tol=1e-9), sc
        assert (f <= base * (1 + 1e-12)).all() and (f >= base / 8 * (1 - 1e-12)).all() and (f[1:] < f[:-1]).all()
        assert math.isclose(p.scale, 0.1 * math.log(8.0) + 1.0 if sc == "yarn" else 1.0)


def test_in_place_strided_and_shared_positions():
    import care_kv
    plan = care_kv.rotary_plan(64, layout="interleaved")
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(2, 19, 3, 4, 64, generator=g, device="cuda").half()  # (B, T, q|k|v, heads, D)
    before = qkv.clone()
    q, k = qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2)
    pos = torch.arange(7, 26, device="cuda")
    qo, ko = care_kv.rotate_heads(q, k, pos, plan, out=(q, k))
    assert qo.data_ptr() == q.data_ptr()
    b = before[:, :, 0].transpose(1, 2), before[:, :, 1].transpose(1, 2)
    for got, x in ((q, b[0]), (k, b[1])):
        _check(got, x, pos.expand(2, 19), plan)
    assert torch.equal(qkv[:, :, 2], before[:, :, 2])
    # heads whose values are not next to each other, and rows off 16 bytes, are read as they are
    y = torch.randn(1, 4, 64, 9, generator=g, device="cuda").half().transpose(2, 3)
    _check(care_kv.rotate_heads(y, None, pos[:9], plan)[0], y, pos[None, :9], plan)
    z = torch.randn(1, 4, 9, 65, generator=g, device="cuda").half()[..., 1:]
    _check(care_kv.rotate_heads(z, None, pos[:9], plan)[0], z, pos[None, :9], plan)
    # one sequence without the batch dim, positions of int32
    o, _ = care_kv.rotate_heads(z[0], None, pos[:9].int(), plan)
    _check(o[None], z, pos[None, :9], plan)


def test_empty_and_broadcast():
    import care_kv
    plan = care_kv.rotary_plan(64)
    q = torch.zeros(0, 4, 3, 64, device="cuda").half()
    assert care_kv.rotate_heads(q, None, torch.zeros(1, 3, dtype=torch.int64, device="cuda"), plan)[0].shape == q.shape
    q = torch.zeros(2, 4, 0, 64, device="cuda").half()
    assert care_kv.rotate_heads(q, q, torch.zeros(0, dtype=torch.int64, device="cuda"), plan)[1].shape == q.shape
    x = torch.randn(1, 1, 5, 64, device="cuda").expand(3, 2, 5, 64)
    pos = torch.randint(0, 99, (3, 5), device="cuda")
    _check(care_kv.rotate_heads(x, None, pos, plan)[0], x, pos, plan)


def test_gradient_is_the_inverse():
    """<R x, y> = <x, R^T y>: the inverse call is the gradient, the plan's scale
    kept, against differences of the forward call in 32 bits."""
    import care_kv
    plan = care_kv.rotary_plan(32, scaling="yarn", factor=4.0, original_len=512)
    g = torch.Generator(device="cuda").manual_seed(8)
    x, y = (torch.randn(1, 2, 6, 48, generator=g, device="cuda") for _ in range(2))
    pos = torch.arange(100, 106, device="cuda")
    grad = care_kv.rotate_heads(y, None, pos, plan, inverse=True)[0]
    _check(grad, y, pos[None], plan, inverse=True)
    for at in ((0, 0, 1, 0), (0, 1, 5, 17), (0, 0, 3, 31), (0, 1, 2, 40)):
        e = torch.zeros_like(x)
        e[at] = 1.0  # the forward call is linear: a step of 1 is exact
        d = ((care_kv.rotate_heads(x + e, None, pos, plan)[0] - care_kv.rotate_heads(x, None, pos, plan)[0]).double()
             * y.double()).sum()
        # 32-bit values of about 2: each of the (at most 2) changed outputs is off by a few 2^-23
        assert abs(float(d) - float(grad[at])) < 4e-5
