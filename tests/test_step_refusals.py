"""What the speculative step's entries refuse (before any GPU call), and their
host helpers."""
from __future__ import annotations

import ctypes
import math
from ctypes import byref, c_void_p

import pytest
import torch

FAKE = 0x1000  # never dereferenced


def _cfg(tq, H=2, D=128, B=16):
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim, cfg.block_size = H, D, B
    return cfg


def _rope(**kw):
    from turborag_amd.turboquant_wrapper import TQRopeConfig
    r = TQRopeConfig(0, 16, 128, 0, 100, 1e-6)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _call_rope(tq, cfg=None, rope=None, n=4, **ptr):
    p = dict(q=FAKE, qs=2048, k=FAKE, ks=256, qw=None, kw=None, table=FAKE, pos=FAKE, oq=FAKE, oqs=2048,
             ok=FAKE, oks=256)
    p.update(ptr)
    cfg, rope = cfg or _cfg(tq), rope or _rope()
    return tq._fast.tq_launch_qk_norm_rope(
        p["q"], p["qs"], p["k"], p["ks"], p["qw"], p["kw"], p["table"], p["pos"], p["oq"], p["oqs"],
        p["ok"], p["oks"], byref(rope), byref(cfg), n, None)


def _call_append(tq, cfg=None, rope=None, n=4, layout=None, **ptr):
    p = dict(q=FAKE, qs=2048, k=FAKE, ks=256, v=FAKE, vs=256, table=FAKE, pos=FAKE, slots=FAKE,
             pool=FAKE, oq=FAKE, oqs=2048)
    p.update(ptr)
    cfg, rope = cfg or _cfg(tq), rope or _rope()
    layout = layout or tq.make_dense_layout_for(_cfg(tq))
    return tq._fast.tq_launch_dense_rope_append_kv(
        p["q"], p["qs"], p["k"], p["ks"], p["v"], p["vs"], None, None, p["table"], p["pos"], p["slots"],
        p["pool"], p["oq"], p["oqs"], byref(layout), byref(rope), byref(cfg), n, None)


def _call_tree(tq, scheme="dense", cfg=None, layout=None, dtype=0, **a):
    p = dict(q=FAKE, pool=FAKE, tables=FAKE, blocks=8, start=FAKE, prefix=FAKE, mask=FAKE, words=1,
             out=FAKE, hq=16, seqs=1, n=4, kv=100)
    p.update(a)
    cfg = cfg or _cfg(tq)
    if layout is None:
        layout = {"dense": tq.make_dense_layout_for, "turbo_prod": tq.make_layout_for,
                  "turbo_mse": tq.make_mse_layout_for}[scheme](cfg)
    head = [p["q"], p["pool"], p["tables"], p["blocks"], p["start"], p["prefix"], p["mask"], p["words"],
            p["out"], byref(layout), byref(cfg)]
    tail = [p["hq"], p["seqs"], p["n"], p["kv"], None]
    if scheme == "dense":
        head.append(dtype)
    return getattr(tq._fast, f"tq_launch_{scheme}_tree_attention")(*head, *tail)


def _message(tq):
    return tq.lib.tq_last_error().decode()


@pytest.mark.parametrize("name", ["q", "k", "table", "pos", "oq", "ok"])
def test_rope_null_pointers(tq, name):
    assert _call_rope(tq, **{name: None}) == -1


@pytest.mark.parametrize("ptr", [dict(k=None), dict(v=None), dict(table=None), dict(pos=None),
                                 dict(slots=None), dict(pool=None), dict(q=None), dict(oq=None)])
def test_append_null_pointers(tq, ptr):
    assert _call_append(tq, **ptr) == -1


@pytest.mark.parametrize("name", ["q", "pool", "tables", "start", "prefix", "mask", "out"])
@pytest.mark.parametrize("scheme", ["dense", "turbo_prod", "turbo_mse"])
def test_tree_null_pointers(tq, scheme, name):
    assert _call_tree(tq, scheme, **{name: None}) == -1


@pytest.mark.parametrize("rope,word", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(num_q_heads=0), "num_q_heads"),
    (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=130), "rot_dim"),
    (dict(max_position=0), "max_position"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps")])
def test_rope_config_refused(tq, rope, word):
    for call in (_call_rope, _call_append):
        assert call(tq, rope=_rope(**rope)) == -2
        assert word in _message(tq)


def test_rope_shapes_refused(tq):
    for call in (_call_rope, _call_append):
        for D in (0, 3, 96, 256):
            assert call(tq, cfg=_cfg(tq, D=D), rope=_rope(rot_dim=2)) == -2
        assert call(tq, cfg=_cfg(tq, H=0)) == -2
        assert call(tq, n=-1) == -2
        assert call(tq, n=1 << 27) == -2
        for bad in (dict(qs=2047), dict(ks=255), dict(qs=-2048), dict(oqs=0), dict(q=FAKE + 1)):
            assert call(tq, **bad) == -2, bad
    assert _call_rope(tq, oks=255) == -2 and _call_append(tq, vs=255) == -2
    assert _call_append(tq, pool=FAKE + 2) == -2
    assert _call_append(tq, cfg=_cfg(tq, H=4), ks=512, vs=512) == -2  # another cfg's layout
    # nothing to do: no launch
    assert _call_rope(tq, n=0) == 0 and _call_append(tq, n=0) == 0


@pytest.mark.parametrize("scheme", ["dense", "turbo_prod", "turbo_mse"])
@pytest.mark.parametrize("bad,word", [
    (dict(hq=15), "num_q_heads"), (dict(hq=0), "num_q_heads"), (dict(hq=1 << 17), "num_q_heads"),
    (dict(seqs=-1), "num_seqs"), (dict(n=-1), "num_tokens"), (dict(words=0), "mask_words"),
    (dict(blocks=0), "max_blocks"), (dict(kv=129), "max_kv_len"), (dict(kv=-1), "max_kv_len"),
    (dict(n=1 << 23), "2^26"), (dict(q=FAKE + 8), "16-byte"), (dict(out=FAKE + 2), "16-byte")])
def test_tree_refused(tq, scheme, bad, word):
    assert _call_tree(tq, scheme, **bad) == -2
    assert word in _message(tq)


@pytest.mark.parametrize("scheme", ["dense", "turbo_prod", "turbo_mse"])
def test_tree_rows_at_the_limit_refused(tq, scheme):
    """2^26 - 2 rows: the merge's grid would have 2^32 threads."""
    assert _call_tree(tq, scheme, hq=2, n=(1 << 25) - 1) == -2
    assert "2^26 - 4" in _message(tq)


def test_tree_geometry_refused(tq):
    for scheme in ("dense", "turbo_prod", "turbo_mse"):
        for D in (2, 32):
            assert _call_tree(tq, scheme, cfg=_cfg(tq, D=D)) == -2
            assert "head_dim must be 64 or 128" in _message(tq)
        assert _call_tree(tq, scheme, pool=FAKE + 1) == -2
        assert _call_tree(tq, scheme, seqs=0) == 0 and _call_tree(tq, scheme, n=0) == 0
        cfg = _cfg(tq)  # a region that ends past the page
        layout = {"dense": tq.make_dense_layout_for, "turbo_prod": tq.make_layout_for,
                  "turbo_mse": tq.make_mse_layout_for}[scheme](cfg)
        name = {"dense": "v_offset", "turbo_prod": "v4_codes_offset", "turbo_mse": "v_norms_offset"}[scheme]
        setattr(layout, name, int(layout.page_size_bytes) - 16)
        assert _call_tree(tq, scheme, cfg=cfg, layout=layout) == -2
        assert "past the page" in _message(tq)
        if scheme == "dense":
            assert _call_append(tq, layout=layout) == -2
            assert "past the page" in _message(tq)
    assert _call_tree(tq, "dense", pool=FAKE + 8) == -2
    assert _call_tree(tq, "dense", dtype=2) == -2
    cfg = _cfg(tq)
    cfg.page_alignment = 4
    layout = tq.make_dense_layout_for(cfg)
    layout.v_offset += 4
    layout.page_size_bytes += 4
    assert _call_tree(tq, "dense", cfg=cfg, layout=layout) == -2


def test_wrapper_refuses_cpu_tensors(tq):
    cfg = _cfg(tq)
    layout = tq.make_dense_layout_for(cfg)
    q, k = torch.zeros(3, 16, 128).half(), torch.zeros(3, 2, 128).half()
    pos, table = torch.zeros(3, dtype=torch.int32), torch.zeros(8, 128)
    with pytest.raises(ValueError):
        tq.qk_norm_rope(q, k, pos, table, q, k, cfg)
    with pytest.raises(ValueError):
        tq.qk_norm_rope(q.float(), k.float(), pos, table, q, k, cfg)
    pool = torch.zeros(8192, dtype=torch.uint8)
    with pytest.raises(ValueError):
        tq.dense_rope_append(q, k, k, pos, pos, table, q, pool, layout, cfg)
    with pytest.raises(ValueError):
        tq.dense_rope_append(q, k, k, pos, pos, table, None, pool, layout, cfg)
    i2 = torch.zeros(1, 1, dtype=torch.int32)
    for scheme in ("dense", "turbo_prod", "fp8"):
        with pytest.raises(ValueError):
            tq.tree_attn_output(scheme, q, pool, i2, pos, pos, i2, q, layout, cfg, 16)
    with pytest.raises(ValueError):  # compressed pages take fp16 queries
        tq.tree_attn_output("turbo_mse", q.bfloat16(), pool, i2, pos, pos, i2, q, layout, cfg, 16)


def test_rope_table():
    from turborag_amd.turboquant_wrapper import rope_table
    t = rope_table(40000, 64)
    assert t.shape == (40000, 64) and t.dtype is torch.float32
    for p, i in ((0, 0), (1, 0), (39999, 0), (39999, 17), (12345, 31)):
        a = p * 10000.0 ** (-2 * i / 64)
        # one rounding to fp32 of a float64 angle's cosine (the angle itself off by p * 2^-51)
        assert abs(float(t[p, i]) - math.cos(a)) <= 2.0 ** -25 + p * 2.0 ** -51
        assert abs(float(t[p, 32 + i]) - math.sin(a)) <= 2.0 ** -25 + p * 2.0 ** -51
    f = [1.0, 0.25]
    assert torch.equal(rope_table(9, 4, inv_freq=f), rope_table(9, 4, inv_freq=torch.tensor(f)))
    for bad in (lambda: rope_table(4, 3), lambda: rope_table(4, 0),
                lambda: rope_table(4, 8, inv_freq=[1.0])):
        with pytest.raises(ValueError):
            bad()


def test_tree_mask_from_parents():
    from turborag_amd.turboquant_wrapper import tree_mask_from_parents
    m = tree_mask_from_parents([-1, 0, 0, 1, -1])
    assert m.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b10000]]
    n = 70
    m = tree_mask_from_parents(list(range(-1, n - 1)))  # a chain: all before and itself
    assert m.shape == (n, 3) and m.dtype is torch.int32
    bits = (m.long()[:, torch.arange(96) // 32] >> (torch.arange(96) % 32)) & 1
    assert torch.equal(bits, (torch.arange(96)[None] <= torch.arange(n)[:, None]).long())
    assert tree_mask_from_parents([]).shape == (0, 1)
    for bad in ([0], [-2], [-1, 1], [-1, 5]):
        with pytest.raises(ValueError):
            tree_mask_from_parents(bad)
