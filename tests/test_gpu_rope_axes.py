"""Norm + rotation by positions with several axes (qk_norm_rope and
dense_rope_append with axes) against float64, with tolerances that count
roundings (oracle/evict_oracle.py)."""
from __future__ import annotations

import pytest
import torch

from oracle.evict_oracle import norm_rope_axes
from turborag_amd.turboquant_wrapper import rope_axes, rope_table

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def _cfg(tq, H, D, B=16):
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim, cfg.block_size = H, D, B
    return cfg


def _inputs(N, Hq, H, D, dtype, count, norm, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(N, Hq + 2 * H, D, generator=g).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in range(2)]
    pos = torch.randint(0, 3000, (count, N), generator=g, dtype=torch.int32)
    return qkv, w, pos


def _gpu(t, dev):
    return None if t is None else t.to(dev)


def _close(got, want, what):
    ref, tol = want
    d = (got.cpu().double() - ref).abs()
    assert (d <= tol).all(), f"{what}: worst {float((d / tol).max()):.2f} of the tolerance"


CASES = [
    # N, Hq, H, D, sections, in turn, interleaved, norm
    (1, 16, 2, 128, [16, 24, 24], False, False, True),     # one axis a lane
    (1, 1, 1, 64, [12, 10, 10], True, True, False),        # one a pair
    (37, 16, 2, 128, [24, 20, 20], True, False, True),
    (129, 8, 4, 128, [16, 24, 24], False, True, False),
    (65, 14, 2, 64, [8, 24], False, False, True),
    (33, 4, 4, 64, [3, 29], False, False, True),           # blocks that end inside a lane's pairs
    (50, 12, 4, 128, [16, 16, 16, 16], False, False, True),
    (50, 12, 4, 128, [1, 2, 60, 1], True, True, True),
    (7, 2, 1, 128, [64], False, False, True),              # one axis alone
    (21, 3, 1, 128, [0, 64], False, False, False),         # an axis without pairs
    (21, 4, 2, 128, [8, 12, 12], True, False, True),       # part of a head rotated
    (10, 4, 2, 32, [5, 5, 6], False, False, True),         # other head_dims
    (10, 2, 1, 2, [1], False, True, True),
    (300, 5, 3, 16, [3, 2, 1, 1], True, True, False),
]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("N,Hq,H,D,sections,turn,inter,norm", CASES)
def test_rotation(tq, cuda, N, Hq, H, D, sections, turn, inter, norm, dtype):
    qkv, w, pos = _inputs(N, Hq, H, D, dtype, len(sections), norm, seed=N + D)
    axes = rope_axes(sections, in_turn=turn)
    table = rope_table(3000, 2 * sum(sections))
    axis = list(axes.axis[:sum(sections)])
    dev = qkv.to(cuda)
    q, k, v = dev[:, :Hq], dev[:, Hq:Hq + H], dev[:, Hq + H:]
    oq, ok = torch.full((N, Hq, D), 5.0, dtype=dtype, device=cuda), torch.full((N, H, D), 5.0, dtype=dtype, device=cuda)
    cfg = _cfg(tq, H, D)
    args = dict(q_weight=_gpu(w[0], cuda), k_weight=_gpu(w[1], cuda), interleaved=inter, axes=axes)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, cfg, **args)
    torch.cuda.synchronize()
    want_q = norm_rope_axes(qkv[:, :Hq], w[0], pos, table, axis, inter, 1e-6)
    want_k = norm_rope_axes(qkv[:, Hq:Hq + H], w[1], pos, table, axis, inter, 1e-6)
    _close(oq, want_q, "q")
    _close(ok, want_k, "k")
    # the append: the same keys, bit for bit, and the values in their slots
    g = torch.Generator().manual_seed(1)
    pages = (N + 15) // 16 + 1
    slots = torch.randperm(pages * 16, generator=g)[:N].int()
    slots[N // 2] = -1
    layout = tq.make_dense_layout_for(cfg)
    page = int(layout.page_size_bytes)
    pool = torch.full((pages * page // 2,), 7.0, dtype=dtype, device=cuda).view(torch.uint8)
    oq2 = torch.empty_like(oq)
    tq.dense_rope_append(q, k, v, pos.to(cuda), slots.to(cuda), table.to(cuda), oq2, pool, layout, cfg, **args)
    torch.cuda.synchronize()
    assert torch.equal(oq2, oq)
    got = torch.stack([pool.view(pages, page)[:, int(at):int(at) + 32 * H * D].contiguous().view(dtype)
                       for at in (layout.k_offset, layout.v_offset)]).view(2, pages * 16, H, D).cpu()
    want = torch.full_like(got, 7.0)
    live = slots >= 0
    want[0, slots[live].long()], want[1, slots[live].long()] = ok.cpu()[live], qkv[live, Hq + H:]
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("D,sections,turn", [(128, [16, 24, 24], False), (128, [24, 20, 20], True),
                                             (64, [9, 11, 12], False), (32, [6, 10], True)])
def test_equal_positions_are_one_axis(tq, cuda, D, sections, turn):
    """Text among images: all axes count alike, and nothing differs from one axis."""
    qkv, w, pos = _inputs(77, 6, 2, D, BF16, 1, True, seed=3)
    table, cfg = rope_table(3000, D).to(cuda), _cfg(tq, 2, D)
    q, k = qkv[:, :6].contiguous().to(cuda), qkv[:, 6:8].contiguous().to(cuda)
    outs = []
    for p, axes in ((pos[0], None), (pos.expand(len(sections), -1).contiguous(), rope_axes(sections, turn))):
        oq, ok = torch.empty_like(q), torch.empty_like(k)
        tq.qk_norm_rope(q, k, p.to(cuda), table, oq, ok, cfg, q_weight=w[0].to(cuda), k_weight=w[1].to(cuda),
                        axes=axes)
        outs.append((oq, ok))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("turn", [False, True])
def test_positions_outside_the_table(tq, cuda, D, turn):
    """A position outside on any axis, also one without pairs, leaves the token's outputs as they were."""
    sections = [0, D // 4, D // 4]
    qkv, _, pos = _inputs(9, 4, 2, D, FP16, 3, False, seed=4)
    pos[0, 1], pos[1, 3], pos[2, 5], pos[2, 8] = -1, 3000, -5, 2 ** 31 - 1
    table = rope_table(3000, D)
    q, k = qkv[:, :4].contiguous().to(cuda), qkv[:, 4:6].contiguous().to(cuda)
    oq, ok = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
    axes = rope_axes(sections, turn)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, _cfg(tq, 2, D), axes=axes)
    torch.cuda.synchronize()
    out = torch.tensor([1, 3, 5, 8])
    assert (oq[out.to(cuda)] == 5).all() and (ok[out.to(cuda)] == 5).all()
    inside = [i for i in range(9) if i not in out.tolist()]
    ref, tol = norm_rope_axes(qkv[:, :4], None, pos.clamp(0, 2999), table, list(axes.axis[:D // 2]), False, 0.0)
    _close(oq[inside], (ref[inside], tol[inside]), "q")


def test_in_place_and_graph(tq, cuda):
    """In place on a fused projection's views, captured on a stream; positions are read at every
    replay."""
    qkv, w, pos = _inputs(40, 16, 2, 128, FP16, 3, True, seed=5)
    table, axes, cfg = rope_table(3000, 128), rope_axes([16, 24, 24]), _cfg(tq, 2, 128)
    src = qkv.to(cuda)
    buf, p, tab = src.clone(), pos.to(cuda), table.to(cuda)
    wq, wk = w[0].to(cuda), w[1].to(cuda)

    def call(stream):
        tq.qk_norm_rope(buf[:, :16], buf[:, 16:18], p, tab, buf[:, :16], buf[:, 16:18], cfg, q_weight=wq,
                        k_weight=wk, axes=axes, stream=stream)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(st.cuda_stream)
    for rep in range(3):
        moved = (pos * (rep + 1)) % 3000
        p.copy_(moved)
        buf.copy_(src)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        axis = list(axes.axis[:64])
        _close(buf[:, :16], norm_rope_axes(qkv[:, :16], w[0], moved, table, axis, False, 1e-6), "q")
        _close(buf[:, 16:18], norm_rope_axes(qkv[:, 16:18], w[1], moved, table, axis, False, 1e-6), "k")
        assert torch.equal(buf[:, 18:], src[:, 18:])
