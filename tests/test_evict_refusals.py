"""What the several-axis and eviction entries refuse (before any GPU call), their
host helpers, and block tables that shrink."""
from __future__ import annotations

import math
from ctypes import byref

import pytest
import torch

from turborag_amd.turboquant_wrapper import BlockTable, PageAllocator, TQRopeAxes, TQRopeConfig, rope_axes

FAKE = 0x1000  # never dereferenced
SCHEMES = ["dense", "turbo_prod", "turbo_mse"]


def _cfg(tq, H=2, D=128, B=16):
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim, cfg.block_size = H, D, B
    return cfg


def _layout(tq, scheme, cfg):
    return {"dense": tq.make_dense_layout_for, "turbo_prod": tq.make_layout_for,
            "turbo_mse": tq.make_mse_layout_for}[scheme](cfg)


def _message(tq):
    return tq.lib.tq_last_error().decode()


def _rope(tq, n=4, axes=None, stride=4, append=False, rot=128, **ptr):
    p = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, pos=FAKE, slots=FAKE, pool=FAKE, oq=FAKE, ok=FAKE)
    p.update(ptr)
    cfg, rope = _cfg(tq), TQRopeConfig(0, 16, rot, 0, 100, 1e-6)
    ax = byref(axes) if axes is not None else None
    if append:
        return tq._fast.tq_launch_dense_rope_axes_append_kv(
            p["q"], 2048, p["k"], 256, p["v"], 256, None, None, p["table"], p["pos"], stride, p["slots"],
            p["pool"], p["oq"], 2048, byref(tq.make_dense_layout_for(cfg)), ax, byref(rope), byref(cfg), n,
            None)
    return tq._fast.tq_launch_qk_norm_rope_axes(p["q"], 2048, p["k"], 256, None, None, p["table"], p["pos"],
                                                stride, p["oq"], 2048, p["ok"], 256, ax, byref(rope),
                                                byref(cfg), n, None)


@pytest.mark.parametrize("append", [False, True])
def test_axes_refused(tq, append):
    good = rope_axes([16, 24, 24])
    assert _rope(tq, append=append) == -1
    for name in ["k", "table", "pos"] + (["v", "slots", "pool"] if append else ["ok"]):
        assert _rope(tq, axes=good, append=append, **{name: None}) == -1
    for num in (0, 5, -1):
        assert _rope(tq, axes=TQRopeAxes(num_axes=num), append=append) == -2
        assert "num_axes" in _message(tq)
    bad = rope_axes([16, 24, 24])
    bad.axis[63] = 3
    assert _rope(tq, axes=bad, append=append) == -2 and "axis" in _message(tq)
    assert _rope(tq, axes=good, stride=3, append=append) == -2 and "axis_stride" in _message(tq)
    assert _rope(tq, axes=good, n=0, append=append) == 0
    # pairs behind the rotated part are not read
    bad.axis[63], bad.axis[40] = 0, 9
    assert _rope(tq, axes=bad, rot=80, n=0, append=append) == 0
    assert _rope(tq, axes=bad, rot=82, n=0, append=append) == -2


def test_rope_axes():
    a = rope_axes([2, 3, 1])
    assert (a.num_axes, list(a.axis[:6])) == (3, [0, 0, 1, 1, 1, 2])
    assert list(rope_axes([4, 2, 1], in_turn=True).axis[:7]) == [0, 1, 2, 0, 1, 0, 0]
    assert list(rope_axes([0, 2], in_turn=True).axis[:2]) == [1, 1]
    for bad in ([], [0], [1] * 5, [65], [-1, 4]):
        with pytest.raises(ValueError):
            rope_axes(bad)


def _weights(tq, scheme="dense", cfg=None, layout=None, dtype=0, **a):
    p = dict(q=FAKE, pool=FAKE, tables=FAKE, blocks=8, start=FAKE, prefix=FAKE, causal=1, inn=FAKE, out=FAKE,
             stride=128, decay=1.0, hq=16, seqs=1, n=4, kv=100)
    p.update(a)
    cfg = cfg or _cfg(tq)
    layout = layout or _layout(tq, scheme, cfg)
    kind = [dtype] if scheme == "dense" else []
    return getattr(tq._fast, f"tq_launch_{scheme}_attention_weights")(
        p["q"], p["pool"], p["tables"], p["blocks"], p["start"], p["prefix"], p["causal"], p["inn"], p["out"],
        p["stride"], p["decay"], byref(layout), byref(cfg), *kind, p["hq"], p["seqs"], p["n"], p["kv"], None)


@pytest.mark.parametrize("scheme", SCHEMES)
def test_weights_refused(tq, scheme):
    for name in ("q", "pool", "tables", "start", "prefix", "out"):
        assert _weights(tq, scheme, **{name: None}) == -1
    for bad, word in [
            (dict(hq=15), "num_q_heads"), (dict(hq=0), "num_q_heads"), (dict(hq=1 << 17), "num_q_heads"),
            (dict(seqs=-1), "num_seqs"), (dict(n=-1), "num_tokens"), (dict(blocks=0), "max_blocks"),
            (dict(kv=129), "max_kv_len"), (dict(kv=-1), "max_kv_len"), (dict(n=(1 << 21) + 1), "2^25"),
            (dict(stride=99), "score_stride"), (dict(decay=-0.5), "decay"), (dict(decay=math.nan), "decay"),
            (dict(decay=1.5), "decay"), (dict(q=FAKE + 8), "16-byte"), (dict(out=FAKE + 2), "4-byte"),
            (dict(inn=FAKE + 1), "4-byte"), (dict(pool=FAKE + 1), "aligned"),
            (dict(kv=1 << 24, blocks=1 << 20, stride=1 << 24, n=1 << 20), "2^30"),
            (dict(kv=1 << 24, blocks=1 << 20, stride=1 << 24, seqs=1 << 14), "2^30")]:
        assert _weights(tq, scheme, **bad) == -2, bad
        assert word in _message(tq), bad
    for D in (2, 32):
        assert _weights(tq, scheme, cfg=_cfg(tq, D=D)) == -2 and "head_dim" in _message(tq)
    # nothing to do: no launch
    assert _weights(tq, scheme, seqs=0) == 0 and _weights(tq, scheme, kv=0) == 0
    # another cfg's layout
    assert _weights(tq, scheme, cfg=_cfg(tq, H=4), layout=_layout(tq, scheme, _cfg(tq))) == -2
    if scheme == "dense":
        assert _weights(tq, dtype=2) == -2 and "dtype" in _message(tq)


def _select(tq, **a):
    p = dict(scores=FAKE, stride=100, lens=FAKE, seqs=1, heads=2, kv=100, budget=10, sink=2, recent=3,
             kept=FAKE, new=None, out=None, ostride=100)
    p.update(a)
    return tq._fast.tq_launch_select_kv(p["scores"], p["stride"], p["lens"], p["seqs"], p["heads"], p["kv"],
                                        p["budget"], p["sink"], p["recent"], p["kept"], p["new"], p["out"],
                                        p["ostride"], None)


def test_select_refused(tq):
    for name in ("scores", "lens", "kept"):
        assert _select(tq, **{name: None}) == -1
    for bad, word in [(dict(seqs=-1), "num_seqs"), (dict(heads=0), "num_kv_heads"), (dict(kv=-1), "max_kv_len"),
                      (dict(budget=0), "budget"), (dict(sink=-1), "sink"), (dict(recent=-1), "recent"),
                      (dict(sink=8), "budget"), (dict(sink=1 << 30, recent=1 << 30), "budget"),
                      (dict(stride=99), "score_stride"), (dict(out=FAKE * 2, ostride=99), "out_stride"),
                      (dict(out=FAKE, ostride=101), "in place"), (dict(scores=FAKE + 2), "4-byte"),
                      (dict(seqs=1 << 21), "2^22")]:
        assert _select(tq, **bad) == -2, bad
        assert word in _message(tq), bad
    assert _select(tq, seqs=0) == 0


def _compact(tq, scheme="dense", cfg=None, layout=None, **a):
    p = dict(pool=FAKE, tables=FAKE, blocks=8, kept=FAKE, budget=10, out=None, oblocks=0, seqs=1)
    p.update(a)
    cfg = cfg or _cfg(tq)
    layout = layout or _layout(tq, scheme, cfg)
    return getattr(tq._fast, f"tq_launch_{scheme}_compact_kv")(
        p["pool"], p["tables"], p["blocks"], p["kept"], p["budget"], p["out"], p["oblocks"], byref(layout),
        byref(cfg), p["seqs"], None)


@pytest.mark.parametrize("scheme", SCHEMES)
def test_compact_refused(tq, scheme):
    for name in ("pool", "tables", "kept"):
        assert _compact(tq, scheme, **{name: None}) == -1
    for bad, word in [(dict(seqs=-1), "num_seqs"), (dict(budget=0), "budget"), (dict(blocks=0), "max_blocks"),
                      (dict(out=FAKE, oblocks=0), "max_blocks"), (dict(blocks=1 << 28), "31 bits"),
                      (dict(budget=(1 << 30) + 1), "31 bits"), (dict(pool=FAKE + 1), "aligned")]:
        assert _compact(tq, scheme, **bad) == -2, bad
        assert word in _message(tq), bad
    for D in (2, 32):
        assert _compact(tq, scheme, cfg=_cfg(tq, D=D)) == -2 and "head_dim" in _message(tq)
    assert _compact(tq, scheme, cfg=_cfg(tq, H=4), layout=_layout(tq, scheme, _cfg(tq))) == -2
    assert _compact(tq, scheme, seqs=0) == 0


def test_wrapper_refuses_cpu_tensors(tq):
    cfg = _cfg(tq)
    i32 = torch.int32
    q, pool = torch.zeros(1, 16, 128, dtype=torch.float16), torch.zeros(1 << 16, dtype=torch.uint8)
    tables, start, prefix = torch.zeros(1, 4, dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32)
    scores, kept = torch.zeros(1, 2, 64), torch.zeros(1, 2, 8, dtype=i32)
    layout = tq.make_dense_layout_for(cfg)
    with pytest.raises(ValueError, match="GPU"):
        tq.attn_weights("dense", q, pool, tables, start, prefix, scores, layout, cfg, 64)
    with pytest.raises(ValueError, match="GPU"):
        tq.select_kv(scores, prefix, kept)
    with pytest.raises(ValueError, match="GPU"):
        tq.compact_kv("dense", pool, tables, kept, layout, cfg)
    with pytest.raises(ValueError, match="scheme"):
        tq.compact_kv("fp8", pool, tables, kept, layout, cfg)
    with pytest.raises(ValueError, match="scheme"):
        tq.attn_weights("fp8", q, pool, tables, start, prefix, scores, layout, cfg, 64)
    with pytest.raises(ValueError, match="scores"):
        tq.attn_weights("dense", q, pool, tables, start, prefix, scores[:, :1], layout, cfg, 64)
    with pytest.raises(ValueError, match="kept"):
        tq.select_kv(scores, prefix, kept[:, :1])
    with pytest.raises(ValueError, match="positions"):
        tq.qk_norm_rope(q, q[:, :2], torch.zeros(2, 1, dtype=i32), torch.zeros(8, 128), q, q[:, :2], cfg,
                        axes=rope_axes([16, 24, 24]))


def test_block_table_truncate(tq):
    alloc = PageAllocator(tq, 64, 10, device_pool=torch.zeros(640, dtype=torch.uint8))
    table = BlockTable(alloc, 4)
    table.build_slot_map(7, 18)
    assert table.blocks(7) == [0, 1, 2, 3, 4] and alloc.num_free() == 5
    table.truncate(7, 18)
    assert table.blocks(7) == [0, 1, 2, 3, 4]
    table.truncate(7, 9)
    assert table.blocks(7) == [0, 1, 2] and table.num_tokens(7) == 9 and alloc.num_free() == 7
    assert table.build_slot_map(7, 4) == [9, 10, 11, 12]  # page 3 again: the last given back first
    table.truncate(7, 0)
    assert table.blocks(7) == [] and alloc.num_free() == 10
    for n in (-1, 1):
        with pytest.raises(ValueError):
            table.truncate(7, n)
    with pytest.raises(KeyError):
        table.truncate(8, 0)
    assert tq.lib.tq_block_table_truncate(None, 0, 0) == -1
    table.close()
    alloc.close()
