"""Refusals of append_pages, paged_attention, window_attention and
verify_drafts, on the CPU: Python arguments and C parameters."""
import ctypes as C

import pytest
import torch

import care_kv
from care_kv import _lib

CPU = torch.device("cpu")


def _half(*s):
    return torch.zeros(*s, dtype=torch.float16)


def _pages(n=4, H=2, D=64):
    return care_kv.int4_pages(n, H, D, device=CPU)


def _table(B=2, n=3):
    return torch.zeros(B, n, dtype=torch.int32)


def test_pool():
    for a in ((-1, 2, 64), (4, 0, 64), (4, 2, 32), (4, 2, 96)):
        with pytest.raises(ValueError):
            care_kv.int4_pages(*a, device=CPU)
    p = _pages(3, 2, 128)
    assert (p.n_pages, p.n_kv_heads, p.data.shape[2]) == (3, 2, 2304)
    for data, D in ((p.data, 64), (p.data.int(), 128), (p.data[0], 128), (p.data[:, :0], 128), (p.data.transpose(0, 1), 128),
                    (torch.zeros(4 * 2304 + 16, dtype=torch.uint8)[3:3 + 4 * 2304].view(2, 2, 2304), 128), (p.data, 32)):
        with pytest.raises(ValueError):
            care_kv.Int4Pages(data, D)
    lib = _lib.load()
    for D in (64, 128, 32, 0):
        assert lib.carekv_page4_bytes(D) == (care_kv.pages.block_bytes(D) if D in (64, 128) else -1)


def test_append_refusals():
    k, v, q, tb, pg = _half(2, 2, 3, 64), _half(2, 2, 3, 64), _half(2, 4, 3, 64), _table(), _pages()
    plan = care_kv.rotary_plan(64, device=CPU)
    pos = torch.zeros(2, 3, dtype=torch.int64)
    bad = [dict(k=k[0], v=v[0]), dict(v=v[:, :1]), dict(v=v.bfloat16()), dict(k=k.float(), v=v.float()), dict(k=_half(2, 3, 3, 64),
           v=_half(2, 3, 3, 64)), dict(k=_half(2, 2, 3, 128), v=_half(2, 2, 3, 128)), dict(q=q[:, :, :2]), dict(q=q[:1]),
           dict(q=q.bfloat16()), dict(q=q[0]), dict(table=tb[0]), dict(table=tb[:1]), dict(table=tb.long()),
           dict(positions=pos), dict(plan=plan, positions=pos.float()), dict(plan=plan, positions=pos[:, :2]),
           dict(plan=plan, positions=torch.zeros(3, 3, dtype=torch.int64)), dict(plan=care_kv.rotary_plan(128, device=CPU))]
    base = dict(pages=pg, table=tb, start=0, k=k, v=v)
    for kw in bad:
        with pytest.raises(ValueError):
            care_kv.append_pages(**{**base, **kw})
    with pytest.raises(_lib.CarekvError):  # no device tensors
        care_kv.append_pages(**base)


def test_paged_refusals():
    q, tb, pg = _half(2, 4, 3, 64), _table(), _pages()
    base = dict(q=q, pages=pg, table=tb, lengths=3)
    for kw in (dict(q=q[0, 0]), dict(q=_half(2, 3, 3, 64)), dict(q=_half(2, 4, 3, 128)), dict(q=q.float()), dict(table=tb.long()),
               dict(table=_table(3)), dict(window=0), dict(window=-1), dict(sink=-1), dict(out=q[:, :2]), dict(out=q.bfloat16()),
               dict(out=_half(2, 4, 64, 3).transpose(2, 3)), dict(q=_half(2, 4, 5, 64), out=pg.data.view(-1)[:5120].view(torch.float16).view(2, 4, 5, 64))):
        with pytest.raises(ValueError):
            care_kv.paged_attention(**{**base, **kw})
    with pytest.raises(_lib.CarekvError):
        care_kv.paged_attention(**base)


def test_window_refusals():
    q, k = _half(2, 4, 3, 64), _half(2, 2, 5, 64)
    base = dict(q=q, k=k, v=k.clone())
    for kw in (dict(q=q[0, 0]), dict(v=k[:, :, :4]), dict(k=k[:1], v=k[:1]), dict(q=_half(2, 3, 3, 64)), dict(q=q.bfloat16()),
               dict(v=k.bfloat16()), dict(q=q.float(), k=k.float(), v=k.float()), dict(window=0), dict(sink=-2),
               dict(out=q[:, :2]), dict(q=_half(2, 4, 3, 96), k=_half(2, 2, 5, 96), v=_half(2, 2, 5, 96))):
        with pytest.raises(ValueError):
            care_kv.window_attention(**{**base, **kw})
    same = _half(2, 4, 5, 64)
    with pytest.raises(ValueError):
        care_kv.window_attention(q=same.clone(), k=same, v=same.clone(), out=same)
    with pytest.raises(_lib.CarekvError):
        care_kv.window_attention(**base)


def test_verify_refusals():
    d, p, u, un = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4, 7), torch.zeros(2, 3), torch.zeros(2)
    base = dict(draft=d, target_probs=p, u=u, u_next=un)
    for kw in (dict(draft=d[0]), dict(draft=d.float()), dict(target_probs=p[:, :3]), dict(target_probs=p[:1]),
               dict(target_probs=p[0]), dict(target_probs=p[..., :0]), dict(target_probs=p.double()), dict(u=u[:, :2]),
               dict(u=u.double()), dict(u_next=un[:1]), dict(u_next=un.half()), dict(draft_probs=p), dict(draft_probs=p[:, :3].half())):
        with pytest.raises(ValueError):
            care_kv.verify_drafts(**{**base, **kw})
    with pytest.raises(_lib.CarekvError):
        care_kv.verify_drafts(**base)


def _last():
    return _lib.load().carekv_last_error().decode()


def test_c_refusals():
    lib = _lib.load()
    none12, none6 = [None] * 12, [None] * 8

    def append(**kw):
        f = dict(batch=1, n_heads=4, n_kv_heads=2, seq_len=1, head_dim=64, rotary_dim=64, dtype=0, pos_bits=64, n_pages=4,
                 max_pages=2, scale=1.0)
        return lib.carekv_append_pages(C.byref(_lib.AppendParams(**{**f, **kw})), *none12, None)
    for kw in (dict(head_dim=96), dict(dtype=2), dict(batch=-1), dict(n_kv_heads=0), dict(rotary_dim=63), dict(rotary_dim=66),
               dict(seq_len=1 << 29), dict(max_pages=1 << 25), dict(n_pages=-1), {}):
        assert append(**kw) == -1 and "carekv_append_pages" in _last()
    assert append(batch=0) == 0 and append(seq_len=0) == 0
    assert lib.carekv_append_pages(None, *none12, None) == -1
    p = _lib.append_params(1, 0, 2, 1, 64, 0, 0, 0, 64, 4, 2, 1.0, 0, 2, 0, 0, 0, 128, 64, 128, 128, 64, 128, 0, 0, 0)
    pool = 1 << 20  # (an address that nothing is read from: the calls are refused first)
    for k, v in ((pool + 4 * 2304 - 16, pool - 4096), (pool - 4096, pool), (pool - 240, pool - 4096), (pool - 4096, pool - 128)):
        assert lib.carekv_append_pages(p, None, k, v, None, None, pool, None, pool, pool, None, None, None, None) == -1
        assert "overlap" in _last()

    def paged(**kw):
        f = dict(batch=1, n_heads=4, n_kv_heads=2, seq_len=1, head_dim=64, dtype=0, n_pages=4, max_pages=200, sm_scale=1.0)
        p = C.byref(_lib.PagedParams(**{**f, **kw}))
        return lib.carekv_paged_attn(p, *none6, 0, None), lib.carekv_paged_attn_workspace_bytes(p)
    for kw in (dict(head_dim=32), dict(dtype=2), dict(batch=-1), dict(n_heads=3), dict(n_kv_heads=0), dict(window=-1), dict(sink=-1),
               dict(max_pages=1 << 25), dict(seq_len=1 << 29), dict(batch=1 << 20, seq_len=1 << 20)):
        assert paged(**kw) == (-1, -1)
    assert paged()[0] == -1 and "null" in _last() and paged()[1] >= 0
    assert paged(batch=0)[0] == 0
    buf = torch.zeros(64, dtype=torch.int64)  # (never read: the calls are refused first)
    at = buf.data_ptr() + -buf.data_ptr() % 16
    big = C.byref(_lib.PagedParams(batch=1, n_heads=4, n_kv_heads=1, seq_len=1, head_dim=64, dtype=0, n_pages=4, max_pages=4000, sm_scale=1.0))
    need = lib.carekv_paged_attn_workspace_bytes(big)
    assert need > 0
    assert lib.carekv_paged_attn(big, at, at, at, at, None, at, None, at, need - 1, None) == -3
    assert lib.carekv_paged_attn(big, at + 2, at, at, at, None, at, None, at, need, None) == -1 and "aligned" in _last()

    def window(**kw):
        f = dict(batch=1, n_heads=4, n_kv_heads=2, seq_len=1, n_keys=5, head_dim=64, dtype=0, sm_scale=1.0)
        p = C.byref(_lib.WindowParams(**{**f, **kw}))
        return lib.carekv_window_attn(p, *([None] * 9), 0, None), lib.carekv_window_attn_workspace_bytes(p)
    for kw in (dict(head_dim=32), dict(dtype=2), dict(n_keys=-1), dict(n_heads=3), dict(window=-1), dict(n_keys=1 << 29),
               dict(k_st=1 << 22), dict(v_st=-1)):
        assert window(**kw) == (-1, -1)
    assert window()[0] == -1 and window(batch=0)[0] == 0

    def verify(**kw):
        p = C.byref(_lib.VerifyParams(**{**dict(batch=1, n_drafts=2, vocab=9, dtype=2), **kw}))
        return lib.carekv_verify_drafts(p, *([None] * 9), 0, None), lib.carekv_verify_drafts_workspace_bytes(p)
    for kw in (dict(dtype=3), dict(vocab=0), dict(batch=-1), dict(n_drafts=-1), dict(batch=1 << 16), dict(vocab=1 << 30)):
        assert verify(**kw) == (-1, -1)
    assert verify()[0] == -1 and verify(batch=0)[0] == 0


def test_structs_match_the_header():
    assert C.sizeof(_lib.AppendParams) == 12 * 4 + 14 * 8
    assert C.sizeof(_lib.PagedParams) == 11 * 4 + 4 + 7 * 8
    assert C.sizeof(_lib.WindowParams) == 10 * 4 + 12 * 8
    assert C.sizeof(_lib.VerifyParams) == 4 * 4 + 6 * 8
    for pack, cls in ((_lib.append_params, _lib.AppendParams), (_lib.paged_params, _lib.PagedParams),
                      (_lib.window_params, _lib.WindowParams), (_lib.verify_params, _lib.VerifyParams)):
        v = list(range(1, len(cls._fields_) + 1))
        assert pack(*v) == bytes(cls(*v))


def test_splits_of_prompts():
    """Prompts whose blocks fill the GPU by themselves have no workspace; few blocks of rows on many keys do."""
    lib = _lib.load()

    def ws(B, T, N, Hq, Hkv, D, window=0):
        p = C.byref(_lib.WindowParams(batch=B, n_heads=Hq, n_kv_heads=Hkv, seq_len=T, n_keys=N, head_dim=D, dtype=0, window=window,
                                      sm_scale=1.0))
        return lib.carekv_window_attn_workspace_bytes(p)
    for B, T, N, Hq, Hkv, D in ((1, 4096, 4096, 32, 8, 128), (1, 8192, 8192, 40, 40, 128), (1, 16384, 16384, 32, 8, 128),
                                (1, 32768, 131072, 32, 8, 128), (4, 8192, 8192, 40, 40, 128), (1, 131072, 131072, 32, 4, 64)):
        assert ws(B, T, N, Hq, Hkv, D) == 0
    row = 4 * (128 + 2)
    assert ws(1, 2048, 16384, 8, 8, 128) >= 4 * 2048 * 8 * row
    assert ws(1, 512, 8192, 32, 8, 128) >= 4 * 512 * 32 * row
