"""Refusals of the long-prompt operators, on the CPU: Python arguments, C
parameters, configuration."""
import ctypes as C

import pytest
import torch

import care_kv
from care_kv import _lib

CPU = torch.device("cpu")


def _plan(r=64, **kw):
    return care_kv.rotary_plan(r, device=CPU, **kw)


@pytest.mark.parametrize("kw", [dict(rotary_dim=63), dict(rotary_dim=0), dict(layout="pairs"), dict(scaling="cubic"),
                                dict(base=1.0), dict(base=float("inf")), dict(factor=0.5), dict(factor=float("nan")),
                                dict(scaling="yarn", factor=2.0), dict(scaling="bands", factor=2.0),
                                dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                dict(scaling="yarn", original_len=64, fast_turns=1.0, slow_turns=1.0),
                                dict(scaling="bands", original_len=64, low_band=4.0, high_band=4.0)])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        care_kv.rotary_plan(**{"rotary_dim": 64, "device": CPU, **kw})


@pytest.mark.parametrize("r,layout,f", [(64, "pairs", torch.zeros(32).double()), (64, "half", torch.zeros(32)),
                                        (64, "half", torch.zeros(31).double()), (63, "half", torch.zeros(31).double()),
                                        (64, "half", torch.zeros(64).double()[::2])])
def test_plans_made_by_hand(r, layout, f):
    with pytest.raises(ValueError):
        care_kv.RotaryPlan(r, layout, f, 1.0)


def _half(*s):
    return torch.zeros(*s, dtype=torch.float16)


def test_rotate_refusals():
    q, k, pos = _half(2, 4, 3, 64), _half(2, 2, 3, 64), torch.zeros(2, 3, dtype=torch.int64)
    bad = [(q[..., :62], k, pos, _plan()), (q.to(torch.int8), None, pos, _plan()), (q.double(), None, pos, _plan()),
           (q, k.float(), pos, _plan()), (q, k[:, :, :2], pos, _plan()), (q, k[:1], pos, _plan()),
           (q, k, pos.float(), _plan()), (q, k, pos[:, :2], _plan()), (q, k, pos[0, :2], _plan()),
           (q, k, torch.zeros(3, 3, dtype=torch.int64), _plan()), (q[0, 0], None, pos, _plan()),
           (_half(2, 4, 3, 63), None, pos, _plan(62)), (q, k, pos, _plan(128))]
    for a in bad:
        with pytest.raises(ValueError):
            care_kv.rotate_heads(*a)
    buf = _half(2, 4, 4, 64)
    for out in ((q, None), (None, k), (q[:, :2], k), (q.float(), k), (q, k.transpose(0, 1)), (q,),
                (torch.zeros(1, dtype=torch.float16).expand(2, 4, 3, 64), k), (_half(2, 4, 64, 3).transpose(2, 3), k)):
        with pytest.raises(ValueError):
            care_kv.rotate_heads(q, k, pos, _plan(), out=out)
    with pytest.raises(ValueError):  # one token to the side of the input
        care_kv.rotate_heads(buf[:, :, :3], None, pos, _plan(), out=(buf[:, :, 1:], None))
    with pytest.raises(_lib.CarekvError):  # no device tensor
        care_kv.rotate_heads(q, k, pos, _plan())


def test_mass_refusals():
    q, k = _half(2, 4, 3, 64), _half(2, 2, 9, 64)
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    for a, kw in (((q, k[..., :32]), {}), ((q[..., :32], k[..., :32]), {}), ((q.float(), k.float()), {}),
                  ((q, k.bfloat16()), {}), ((q, k[:1]), {}), ((q[:, :3], k), {}), ((q, _half(2, 0, 9, 64)), {}),
                  ((q, k), dict(lse=f(2, 4, 2))), ((q, k), dict(lse=f(2, 4, 3).double())), ((q, k), dict(accumulate=True)),
                  ((q, k), dict(out=f(2, 2, 8))), ((q, k), dict(out=f(2, 2, 9).double())),
                  ((q, k), dict(out=f(2, 2, 1).expand(2, 2, 9))), ((q, k[0]), {})):
        with pytest.raises(ValueError):
            care_kv.attention_mass(*a, **kw)
    with pytest.raises(_lib.CarekvError):
        care_kv.attention_mass(q, k)


def test_row_counts():
    assert _lib.row_counts(None, 3, CPU, "x") is None
    assert _lib.row_counts(5, 3, CPU, "x").tolist() == [5, 5, 5]
    assert _lib.row_counts([1, 2, 3], 3, CPU, "x").tolist() == [1, 2, 3]
    assert _lib.row_counts(torch.tensor([1, 2, 3]), 3, CPU, "x").tolist() == [1, 2, 3]
    with pytest.raises(ValueError):
        _lib.row_counts([1, 2], 3, CPU, "x")
    with pytest.raises(TypeError):
        _lib.row_counts([1.5, 2, 3], 3, CPU, "x")


def test_evict_refusals():
    m, k = torch.zeros(2, 3, 9), _half(2, 3, 9, 64)
    ok = dict(keep=4, sink=1, recent=1)
    for a, kw in (((m, k, k[..., :32]), ok), ((m, k, k.float()), ok), ((m.double(), k, k), ok), ((m[:, :2], k, k), ok),
                  ((m[..., :8], k, k), ok), ((m, k, k), dict(keep=0)), ((m, k, k), dict(keep=4, sink=-1)),
                  ((m, k, k), dict(keep=4, recent=-1)), ((m, k, k), dict(keep=4, sink=3, recent=2)),
                  ((m, k[..., :1], k[..., :1]), ok), ((m, k[..., :0], k[..., :0]), ok)):
        with pytest.raises(ValueError):
            care_kv.evict_rows(*a, **kw)
    with pytest.raises(_lib.CarekvError):
        care_kv.evict_rows(m, k, k, **ok)


def test_prefix_refusals():
    q, k = _half(2, 4, 3, 64), _half(2, 9, 64)
    o, l = _half(2, 4, 3, 64), torch.zeros(2, 4, 3)
    for a, kw in (((q, k, k[:, :8]), {}), ((q, k[..., :32], k[..., :32]), {}), ((q[:, :3], k, k), {}),
                  ((q, k.bfloat16(), k), {}), ((q.float(), k.float(), k.float()), {}), ((q, k[None], k[None]), {}),
                  ((q, k, k), dict(own=(o[:, :, :2], l))), ((q, k, k), dict(own=(o, l[:, :, :2]))),
                  ((q, k, k), dict(own=(o, l.double()))), ((q, k, k), dict(own=(o.float(), l))),
                  ((q, k, k), dict(out=o[:, :2])), ((q, k, k), dict(out=o.float())),
                  ((q, k, k), dict(out=o.transpose(2, 3).contiguous().transpose(2, 3)))):
        with pytest.raises(ValueError):
            care_kv.prefix_attention(*a, **kw)
    buf = _half(3, 4, 3, 64)
    with pytest.raises(ValueError):
        care_kv.prefix_attention(q, k, k, own=(buf[:2], l), out=buf[1:])
    with pytest.raises(_lib.CarekvError):
        care_kv.prefix_attention(q, k, k)


def test_c_entries_refuse_before_any_launch():
    """Null arguments, sizes and alignments are turned into an error and a message."""
    lib = _lib.load()
    err = lambda: lib.carekv_last_error().decode()  # noqa: E731
    p, odd = 4096, 4096 + 2  # addresses that are never read
    rot = dict(batch=1, seq_len=1, n_heads=2, n_kv_heads=1, head_dim=64, rotary_dim=64, dtype=0, pos_bits=64)
    for bad in (dict(head_dim=63), dict(rotary_dim=66), dict(rotary_dim=3), dict(dtype=3), dict(pos_bits=16),
                dict(batch=-1)):
        assert lib.carekv_rotate_heads(_lib.RotaryParams(**{**rot, **bad}), p, p, p, p, p, p, None) == -1 and err()
    assert lib.carekv_rotate_heads(None, p, p, p, p, p, p, None) == -1
    assert lib.carekv_rotate_heads(_lib.RotaryParams(**rot), p, None, p, p, p, p, None) == -1
    assert lib.carekv_rotate_heads(_lib.RotaryParams(**{**rot, "batch": 0}), None, None, None, None, None, None, None) == 0
    mass = dict(batch=1, n_heads=4, n_kv_heads=2, n_queries=1, n_keys=9, head_dim=64, dtype=0, q_sh=64, q_st=64, k_sh=576,
                k_st=64, out_sh=9)
    for bad in (dict(head_dim=32), dict(dtype=2), dict(n_heads=3), dict(n_kv_heads=0), dict(n_keys=-1),
                dict(n_keys=1 << 30), dict(k_st=65)):
        mp = _lib.MassParams(**{**mass, **bad})
        assert lib.carekv_attention_mass(mp, p, p, None, None, None, p, p, 1 << 40, None) == -1 and err(), bad
    assert lib.carekv_attention_mass_workspace_bytes(_lib.MassParams(**{**mass, "head_dim": 32}), 0) == -1
    assert lib.carekv_attention_mass_workspace_bytes(_lib.MassParams(**mass), 0) == 0  # a decode step needs none
    mp = _lib.MassParams(**{**mass, "n_queries": 40})
    need = lib.carekv_attention_mass_workspace_bytes(mp, 0)
    assert lib.carekv_attention_mass_workspace_bytes(mp, 1) < need and lib.carekv_attention_mass(mp, p, p, None, None, None, p, p, need - 1, None) == -3
    assert lib.carekv_attention_mass(mp, odd, p, None, None, None, p, p, need, None) == -1 and "aligned" in err()
    assert lib.carekv_attention_mass(mp, p, None, None, None, None, p, p, need, None) == -1
    ev = dict(batch=1, n_kv_heads=2, n_keys=9, row_bytes=128, keep=4, sink=1, recent=1, k_sh=1152, k_st=128, v_sh=1152,
              v_st=128)
    for bad in (dict(keep=0), dict(sink=4), dict(recent=-1), dict(row_bytes=6), dict(k_st=130), dict(n_keys=1 << 30)):
        assert lib.carekv_evict_rows(_lib.EvictParams(**{**ev, **bad}), p, p, p, None, p, p, p, p, p, p, 1 << 40, None) == -1, bad
    assert lib.carekv_evict_rows(_lib.EvictParams(**ev), None, p, p, None, p, p, p, p, p, p, 1 << 40, None) == -1
    assert lib.carekv_evict_rows_workspace_bytes(_lib.EvictParams(**ev)) == 0
    ep = _lib.EvictParams(**{**ev, "n_keys": 20000})
    need = lib.carekv_evict_rows_workspace_bytes(ep)
    assert need > 0 and lib.carekv_evict_rows(ep, p, p, p, None, p, p, p, p, p, p, need - 1, None) == -3
    assert lib.carekv_evict_rows(ep, p, p, p, None, p, p, p, p, p, None, need, None) == -1
    pre = dict(batch=2, n_heads=4, n_kv_heads=2, seq_len=1, prefix_len=9, head_dim=64, q_sb=256, q_sh=64, k_sh=576,
               k_st=64, v_sh=576, v_st=64, out_sb=256, out_sh=64)
    for bad in (dict(head_dim=96), dict(dtype=2), dict(n_heads=5), dict(prefix_len=-1), dict(k_st=1 << 22), dict(v_st=-64),
                dict(prefix_len=1 << 30), dict(q_sh=60)):
        pp = _lib.PrefixParams(**{**pre, **bad})
        assert lib.carekv_prefix_attn(pp, p, p, p, None, None, p, None, p, 1 << 40, None) == -1 and err(), bad
    assert lib.carekv_prefix_attn_workspace_bytes(_lib.PrefixParams(**pre)) == 0  # one split: nothing to keep
    pp = _lib.PrefixParams(**{**pre, "prefix_len": 4000})
    need = lib.carekv_prefix_attn_workspace_bytes(pp)
    assert need > 0 and lib.carekv_prefix_attn(pp, p, p, p, None, None, p, None, p, need - 1, None) == -3
    assert lib.carekv_prefix_attn(pp, p, p, p, p, None, p, None, p, need, None) == -1  # own without its lse


def test_structs_match_the_header():
    import os
    from test_host import ROOT, _struct_fields
    hdr = open(os.path.join(ROOT, "include", "carekv.h")).read()
    for cname, py in (("carekv_rotary_params", _lib.RotaryParams), ("carekv_mass_params", _lib.MassParams),
                      ("carekv_evict_params", _lib.EvictParams), ("carekv_prefix_params", _lib.PrefixParams)):
        assert [f[0] for f in py._fields_] == _struct_fields(hdr, cname), cname


def test_config(monkeypatch):
    for bad in (dict(prefill_keep=-1), dict(prefill_keep=10, prefill_keep_sink=4, prefill_keep_recent=8),
                dict(prefill_keep_window=-1)):
        with pytest.raises(ValueError):
            care_kv.CacheConfig(**bad)
    monkeypatch.setenv("CAREKV_PREFILL_KEEP", "256")
    monkeypatch.setenv("CAREKV_PREFILL_KEEP_WINDOW", "64")
    c = care_kv.CacheConfig(**care_kv.apply_carekv_env_overrides({}))
    assert (c.prefill_keep, c.prefill_keep_sink, c.prefill_keep_recent, c.prefill_keep_window) == (256, 4, 32, 64)


def test_launches_on_the_tensors_device(monkeypatch):
    """Whatever device is current: the launch and its stream are those of the
    tensors' device (the library and the guard are stand-ins)."""
    entered, launched = [], []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *exc):
            entered.pop()
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 100 + index)
    fn = lambda *a: launched.append((list(entered), a)) or 0  # noqa: E731
    _lib.call(torch.device("cuda", 1), "x", fn, 7)
    _lib.call(torch.device("cuda", 0), "x", fn, 8)
    assert launched == [([torch.device("cuda", 1)], (7, 101)), ([], (8, 100))] and not entered
    with pytest.raises(_lib.CarekvError):
        _lib.call(torch.device("cuda", 0), "x", lambda *a: -1)


def _brute(a, b):
    """Whether two strided views share a byte, by listing both."""
    def cells(t):
        at = {t.data_ptr()}
        for n, st in zip(t.shape, t.stride()):
            at = {x + i * st * t.element_size() for x in at for i in range(n)}
        return {x + j for x in at for j in range(t.element_size())}
    return bool(cells(a) & cells(b))


def test_overlap_of_views():
    """Never missed, and the heads of fused projections in either order are told apart."""
    a = torch.zeros(2, 5, 12, 8, dtype=torch.float16)  # (B, T, heads, D)
    c = torch.zeros(2, 12, 5, 8, dtype=torch.float16)  # (B, heads, T, D)
    split = lambda x: [x[:, :, :6].transpose(1, 2), x[:, :, 6:9].transpose(1, 2), x[:, :, 4:8].transpose(1, 2)]  # noqa: E731
    views = split(a) + [c[:, :6], c[:, 6:9], c[:, 4:8], a[..., :4], a[..., 4:], a[:1], a[1:], a[:, 1:3], a[:, ::2],
                        a[:, 1::2], a.float(), a.view(torch.float32), a[:, :0], a[0, 0, 0], a[:1].expand(3, 5, 12, 8)]
    for x in views:
        for y in views:
            shared = bool(x.numel() and y.numel()) and _brute(x, y)
            assert _lib.overlap(x, y) or not shared
    for x, y in ((views[0], views[1]), (views[3], views[4]), (views[6], views[7]), (a[:, ::2], views[9])):
        assert _lib.overlap(x, y) == _brute(x, y) == _lib.overlap(y, x)


def test_outputs_over_inputs_are_refused():
    q, k, pos = _half(2, 4, 3, 64), _half(2, 4, 3, 64), torch.zeros(2, 3, dtype=torch.int64)
    buf = _half(2, 7, 3, 64)
    for a, b, out in ((q, k, (k, q)), (q, q, (q, q)), (q, k, (_half(2, 4, 3, 64), q)), (q, k, (buf[:, :4], buf[:, 3:])),
                      (buf[:, :4], buf[:, 3:], (buf[:, :4], buf[:, 3:]))):
        with pytest.raises(ValueError, match="overlap"):
            care_kv.rotate_heads(a, b, pos, _plan(), out=out)
    lse = torch.zeros(2, 4, 3)  # of the output's own shape
    with pytest.raises(ValueError, match="overlap"):
        care_kv.attention_mass(q, k, lse=lse, out=lse)


def test_prefix_is_checked_before_the_cache_changes():
    from care_kv.prefix import check_prefix
    k = _half(2, 9, 64)
    check_prefix((k, k), 4, 64, torch.float16, k.device)
    for p, h, d in (((k,), 4, 64), ((k, k[:, :8]), 4, 64), ((k, k), 3, 64), ((k, k), 4, 128), ((k, k.bfloat16()), 4, 64),
                    ((k[..., :32], k[..., :32]), 4, 32), ((k[None], k[None]), 4, 64), ((k[:0], k[:0]), 4, 64)):
        with pytest.raises(ValueError):
            check_prefix(p, h, d, torch.float16, k.device)


def test_launches_that_do_not_fit_are_refused():
    """Grids of 2^32 threads and more: refused with a message, nothing launched."""
    lib = _lib.load()
    p = 4096
    rot = _lib.RotaryParams(batch=1 << 15, seq_len=1 << 20, n_heads=1, n_kv_heads=0, head_dim=64, rotary_dim=64, dtype=0,
                            pos_bits=64)
    assert lib.carekv_rotate_heads(rot, p, None, p, p, p, None, None) == -1
    mass = _lib.MassParams(batch=1 << 20, n_heads=8, n_kv_heads=8, n_queries=1, n_keys=9, head_dim=64, dtype=0)
    assert lib.carekv_attention_mass(mass, p, p, None, None, None, p, p, 1 << 62, None) == -1
    ev = _lib.EvictParams(batch=1 << 20, n_kv_heads=8, n_keys=9, row_bytes=128, keep=4)
    assert lib.carekv_evict_rows(ev, p, p, p, None, p, p, p, p, p, p, 1 << 62, None) == -1
    pre = _lib.PrefixParams(batch=1 << 20, n_heads=64, n_kv_heads=8, seq_len=8, prefix_len=0, head_dim=128)
    assert lib.carekv_prefix_attn(pre, p, p, p, None, None, p, None, p, 1 << 62, None) == -1


def test_prefix_refuses_its_own_lse_as_output():
    lib, p = _lib.load(), 4096
    pp = _lib.PrefixParams(batch=2, n_heads=4, n_kv_heads=2, seq_len=1, prefix_len=9, head_dim=64, q_sb=256, q_sh=64,
                           k_sh=576, k_st=64, v_sh=576, v_st=64, out_sb=256, out_sh=64, own_sb=256, own_sh=64)
    assert lib.carekv_prefix_attn(pp, p, p, p, p, p, p, p, p, 1 << 40, None) == -1
    assert "own_lse" in lib.carekv_last_error().decode()


def test_prefix_output_over_its_own_lse_is_refused():
    q, k = _half(2, 4, 3, 64), _half(2, 9, 64)
    out = _half(2, 4, 3, 64)
    lse = out.view(-1)[:48].view(torch.float32).view(2, 4, 3)
    with pytest.raises(ValueError, match="overlap"):
        care_kv.prefix_attention(q, k, k, own=(_half(2, 4, 3, 64), lse), out=out)


def test_rows_far_apart_are_copied():
    far = torch.empty(0, dtype=torch.float16).set_(torch.zeros(1 << 24, dtype=torch.float16).untyped_storage(), 0, (2, 3, 64),
                                                   (64, _lib.MAX_ROW_STEP, 1))
    assert _lib.aligned_rows(far) is far and _lib.aligned_rows(far[:, :1], near=True).data_ptr() == far.data_ptr()
    assert _lib.aligned_rows(far, near=True).is_contiguous()


@pytest.mark.parametrize("mode,kw,prefix", [("carekv_stored", dict(prefill_keep=40), False),
                                            ("base_quant", dict(prefill_keep=40, base_quantizer="kivi_style", base_bits=2), False),
                                            ("carekv_eval", {}, True), ("carekv_stored", {}, True), ("fp", {}, "short")])
def test_padded_prompts_are_refused_before_any_is_written(mode, kw, prefix, monkeypatch):
    """What a mode does not take of any sequence of a padded batch is refused before the first one is computed."""
    monkeypatch.setenv("CAREKV_PREFILL_MODE", mode)
    cfg = care_kv.CacheConfig(num_layers=1, num_heads=4, num_kv_heads=2, head_dim=64, prefill_keep_sink=4,
                              prefill_keep_recent=8, **kw)
    w = [torch.zeros(o, 256, dtype=torch.float16) for o in (256, 128, 128, 256)]
    lay = care_kv.CAREKVLayer(cfg, 0, *w)
    monkeypatch.setattr(lay, "_heads", lambda *a: pytest.fail("a prompt was computed"))
    mask = torch.ones(3, 60, dtype=torch.int64)
    mask[0, :50] = 0  # 10 rows, 59, 30
    mask[1, 59:] = 0
    mask[2, 30:] = 0
    cache = type("Cache", (), {"hat": "kivi_style" in kw.values()})()
    pre = None if not prefix else (_half(2, 9, 64), _half(2, 8 if prefix == "short" else 9, 64))
    with pytest.raises(ValueError if prefix == "short" else NotImplementedError):
        lay.prefill(cache, _half(3, 60, 256), attention_mask=mask, prefix=pre)


def test_rotate_refusals_of_one_sequence():
    q, k, pos = _half(4, 3, 64), _half(2, 3, 64), torch.zeros(3, dtype=torch.int64)
    for out in ((None, k), (q, None), (q,), (q, k, k), (q[:2], k)):
        with pytest.raises(ValueError):
            care_kv.rotate_heads(q, k, pos, _plan(), out=out)
    with pytest.raises(ValueError):
        care_kv.rotate_heads(q, None, pos, _plan(), out=(q, k))
