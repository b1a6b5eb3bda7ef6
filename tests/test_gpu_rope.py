"""Per-head norm + rotation (qk_norm_rope) and its append to dense pages
(dense_rope_append) against float64, with tolerances that count roundings
(oracle/step_oracle.py)."""
from __future__ import annotations

import pytest
import torch

from oracle.step_oracle import norm_rope
from turborag_amd.turboquant_wrapper import rope_table

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def _inputs(N, Hq, H, D, dtype, seed, fused=True, norm=True, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(N, Hq + 2 * H, D, generator=g) * scale).to(dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in range(2)]
    pos = torch.randint(0, 5000, (N,), generator=g, dtype=torch.int32)
    parts = [qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]]
    return parts, w, pos


def _cfg(tq, H, D, B=16):
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim, cfg.block_size = H, D, B
    return cfg


def _views(parts, dev, fused):
    """The parts on the GPU: views of one projection, or tensors of their own."""
    if fused:
        whole = torch.cat(parts, 1).to(dev)
        a, b = parts[0].shape[1], parts[0].shape[1] + parts[1].shape[1]
        return whole[:, :a], whole[:, a:b], whole[:, b:]
    return tuple(p.contiguous().to(dev) for p in parts)


def _gpu(t, dev):
    return None if t is None else t.to(dev)


def _close(got, want, what):
    ref, tol = want
    d = (got.cpu().double() - ref).abs()
    bad = ~(d <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((d / tol).max()):.2f} of the tolerance")


CASES = [
    # N, Hq, H, D, rot, interleaved, norm, fused
    (1, 16, 2, 128, 128, False, True, True),
    (1, 1, 1, 64, 64, False, False, False),
    (3, 14, 2, 64, 64, True, True, True),
    (37, 16, 2, 128, 128, True, False, True),
    (129, 8, 4, 128, 128, False, True, False),
    (1000, 16, 2, 128, 128, False, True, True),
    (513, 3, 3, 64, 64, False, True, True),
    (2049, 5, 1, 64, 64, True, False, False),
    (65, 16, 2, 128, 64, False, True, True),    # part of a head
    (65, 7, 1, 128, 32, True, True, True),
    (33, 4, 2, 64, 48, False, False, True),
    (9, 4, 2, 32, 32, False, True, True),       # other head dims
    (9, 4, 2, 16, 10, True, True, True),
    (70, 3, 1, 2, 2, False, True, False),
    (5, 2, 1, 8, 2, False, False, True),
]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("N,Hq,H,D,rot,inter,norm,fused", CASES)
def test_norm_rope(tq, cuda, N, Hq, H, D, rot, inter, norm, fused, dtype):
    print(f"[rope] {N=} {Hq=} {H=} {D=} {rot=} {inter=} {norm=} {fused=} {dtype}", flush=True)
    parts, w, pos = _inputs(N, Hq, H, D, dtype, seed=N + D, norm=norm)
    table = rope_table(5000, rot)
    q, k, _ = _views(parts, cuda, fused)
    # outputs with room around them: what is not a row stays as it was
    oq = torch.full((N, Hq + 1, D), 7.0, dtype=dtype, device=cuda)
    ok = torch.full((N + 1, H, D), 7.0, dtype=dtype, device=cuda)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq[:, :Hq], ok[:N], _cfg(tq, H, D),
                    q_weight=_gpu(w[0], cuda), k_weight=_gpu(w[1], cuda), eps=1e-6,
                    interleaved=inter)
    _close(oq[:, :Hq], norm_rope(parts[0], w[0], pos, table, inter, 1e-6), "query")
    _close(ok[:N], norm_rope(parts[1], w[1], pos, table, inter, 1e-6), "key")
    assert (oq[:, Hq:] == 7).all() and (ok[N:] == 7).all()


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (128, 64), (32, 32)])
def test_in_place(tq, cuda, D, rot, dtype):
    """The outputs are the inputs: views of one projection, changed where they are."""
    parts, w, pos = _inputs(77, 6, 2, D, dtype, seed=5)
    table = rope_table(5000, rot)
    whole = torch.cat(parts, 1).to(cuda)
    q, k = whole[:, :6], whole[:, 6:8]
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), q, k, _cfg(tq, 2, D), _gpu(w[0], cuda),
                    _gpu(w[1], cuda))
    _close(q, norm_rope(parts[0], w[0], pos, table, False, 1e-6), "query")
    _close(k, norm_rope(parts[1], w[1], pos, table, False, 1e-6), "key")
    assert torch.equal(whole[:, 8:].cpu(), parts[2])


def test_only_one_weight(tq, cuda):
    parts, w, pos = _inputs(40, 4, 2, 128, FP16, seed=6)
    table = rope_table(5000, 128)
    q, k, _ = _views(parts, cuda, True)
    oq, ok = torch.empty(40, 4, 128, dtype=FP16, device=cuda), torch.empty(40, 2, 128, dtype=FP16,
                                                                           device=cuda)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, _cfg(tq, 2, 128),
                    k_weight=_gpu(w[1], cuda))
    _close(oq, norm_rope(parts[0], None, pos, table, False, 1e-6), "query")
    _close(ok, norm_rope(parts[1], w[1], pos, table, False, 1e-6), "key")


@pytest.mark.parametrize("D", [64, 128])
def test_unaligned_rows(tq, cuda, D):
    """Pointers and strides that are not multiples of 16 bytes."""
    N, Hq, H = 50, 3, 2
    parts, w, pos = _inputs(N, Hq, H, D, FP16, seed=7)
    table = rope_table(5000, D)
    wide = Hq * D + 3
    room = torch.zeros(1 + N * wide, dtype=FP16, device=cuda)
    q = room[1:].view(N, wide)[:, :Hq * D].unflatten(1, (Hq, D))
    q.copy_(parts[0])
    k = parts[1].contiguous().to(cuda)
    ws = [torch.cat([x[:1], x]).to(cuda)[1:] for x in w]
    oq = torch.zeros(1 + N * Hq * D, dtype=FP16, device=cuda)[1:].view(N, Hq, D)
    ok = torch.empty_like(k)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, _cfg(tq, H, D), ws[0], ws[1])
    _close(oq, norm_rope(parts[0], w[0], pos, table, False, 1e-6), "query")
    _close(ok, norm_rope(parts[1], w[1], pos, table, False, 1e-6), "key")


@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (128, 64)])
def test_positions_outside_the_table(tq, cuda, D, rot):
    """Such tokens are skipped: their outputs and their slots' cells stay as they were."""
    N, Hq, H = 12, 4, 2
    parts, w, pos = _inputs(N, Hq, H, D, FP16, seed=8)
    pos[3], pos[7], pos[11] = -1, 5000, 2 ** 31 - 1
    inside = (pos >= 0) & (pos < 5000)
    table = rope_table(5000, rot)
    q, k, v = _views(parts, cuda, True)
    oq = torch.full((N, Hq, D), 3.0, dtype=FP16, device=cuda)
    ok = torch.full((N, H, D), 3.0, dtype=FP16, device=cuda)
    cfg = _cfg(tq, H, D)
    tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, cfg)
    safe = torch.where(inside, pos, 0)
    for got, x in ((oq, parts[0]), (ok, parts[1])):
        ref, tol = norm_rope(x, None, safe, table, False, 1e-6)
        _close(got[inside.to(cuda)], (ref[inside], tol[inside]), "inside")
        assert (got[~inside.to(cuda)] == 3).all()
    layout = tq.make_dense_layout_for(cfg)
    pool = torch.full((2 * int(layout.page_size_bytes),), 9, dtype=torch.uint8, device=cuda)
    slots = torch.arange(N, dtype=torch.int32, device=cuda) + 10
    oq.fill_(3.0)
    tq.dense_rope_append(q, k, v, pos.to(cuda), slots, table.to(cuda), oq, pool, layout, cfg)
    assert (oq[~inside.to(cuda)] == 3).all()
    cells = pool.view(2, 2, 16, H, D * 2).transpose(0, 1).reshape(2, 32, H, D * 2)[:, 10:10 + N]
    assert (cells[:, ~inside.to(cuda)] == 9).all()
    assert torch.equal(cells[1][inside.to(cuda)].contiguous().view(FP16).cpu(), parts[2][inside])


APPEND = [
    # N, Hq, H, D, rot, block, inter, norm, fused
    (1, 16, 2, 128, 128, 16, False, False, True),
    (33, 16, 2, 128, 128, 16, False, True, True),
    (700, 14, 2, 64, 64, 16, True, True, True),
    (257, 8, 1, 128, 128, 7, False, True, False),
    (64, 4, 4, 64, 64, 1, False, False, True),
    (90, 6, 3, 128, 96, 32, True, True, True),
    (45, 2, 2, 16, 16, 16, False, True, True),
    (20, 2, 1, 2, 2, 5, False, False, False),
]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("N,Hq,H,D,rot,B,inter,norm,fused", APPEND)
def test_append(tq, cuda, N, Hq, H, D, rot, B, inter, norm, fused, dtype):
    print(f"[append] {N=} {Hq=} {H=} {D=} {rot=} {B=} {dtype}", flush=True)
    parts, w, pos = _inputs(N, Hq, H, D, dtype, seed=N + D, norm=norm)
    parts[2][0, 0, 0] = float("nan")  # values are copied as they are
    table = rope_table(5000, rot)
    cfg = _cfg(tq, H, D, B)
    layout = tq.make_dense_layout_for(cfg)
    pages = (N + B - 1) // B + 2
    g = torch.Generator().manual_seed(N)
    slots = torch.randperm(pages * B, generator=g)[:N].int()
    stored = torch.ones(N, dtype=torch.bool)
    if N > 4:
        slots[2] = slots[4] = -1
        stored[2] = stored[4] = False
    pool = torch.randint(0, 255, (pages * int(layout.page_size_bytes),), generator=g,
                         dtype=torch.uint8)
    q, k, v = _views(parts, cuda, fused)
    for with_query in (True, False):
        dpool = pool.to(cuda)
        oq = torch.empty(N, Hq, D, dtype=dtype, device=cuda)
        tq.dense_rope_append(q if with_query else None, k, v, pos.to(cuda), slots.to(cuda),
                             table.to(cuda), oq if with_query else None, dpool, layout, cfg,
                             _gpu(w[0], cuda), _gpu(w[1], cuda), eps=1e-5, interleaved=inter)
        if with_query:  # a token without a slot has its query all the same
            _close(oq, norm_rope(parts[0], w[0], pos, table, inter, 1e-5), "query")
        got = dpool.cpu()
        ref, tol = norm_rope(parts[1], w[1], pos, table, inter, 1e-5)
        size = 2 * D
        untouched = torch.ones(got.numel(), dtype=torch.bool)
        for t in torch.nonzero(stored).flatten().tolist():
            page, tib = divmod(int(slots[t]), B)
            for h in range(H):
                at = page * int(layout.page_size_bytes) + (tib * H + h) * size
                a, b = at + int(layout.k_offset), at + int(layout.v_offset)
                _close(got[a:a + size].view(dtype), (ref[t, h], tol[t, h]), f"key {t} {h}")
                assert torch.equal(got[b:b + size], parts[2][t, h].contiguous().view(torch.uint8))
                untouched[a:a + size] = untouched[b:b + size] = False
        assert torch.equal(got[untouched], pool[untouched])


def test_append_equals_rotation_and_store(tq, cuda):
    """The append's cells are the rotation's output stored by the dense store, bit for bit."""
    N, Hq, H, D = 200, 8, 2, 128
    parts, w, pos = _inputs(N, Hq, H, D, FP16, seed=11)
    cfg = _cfg(tq, H, D)
    layout = tq.make_dense_layout_for(cfg)
    table, pos = rope_table(5000, D, device=cuda), pos.to(cuda)
    q, k, v = _views(parts, cuda, True)
    ws = [_gpu(x, cuda) for x in w]
    slots = torch.randperm(208)[:N].int().to(cuda)
    oq, ok = torch.empty(N, Hq, D, dtype=FP16, device=cuda), torch.empty(N, H, D, dtype=FP16,
                                                                         device=cuda)
    a, b = (tq.alloc_page_pool(208, layout, cfg) for _ in range(2))
    tq.qk_norm_rope(q, k, pos, table, oq, ok, cfg, *ws)
    tq.dense_store(ok, v.contiguous(), slots, a, layout, cfg)
    oq2 = torch.empty_like(oq)
    tq.dense_rope_append(q, k, v, pos, slots, table, oq2, b, layout, cfg, *ws)
    assert torch.equal(a, b) and torch.equal(oq, oq2)


def test_far_position_and_magnitudes(tq, cuda):
    """Angles of positions near 131,072, values near the ends of fp16 and of bf16."""
    for dtype, scale in ((FP16, 3e3), (FP16, 1e-4), (BF16, 1e12), (BF16, 1e-12)):
        parts, w, _ = _inputs(31, 4, 2, 128, dtype, seed=12, scale=scale)
        pos = torch.arange(131041, 131072, dtype=torch.int32)
        table = rope_table(131072, 128, base=1e6)
        q, k, _ = _views(parts, cuda, True)
        oq, ok = torch.empty_like(q, memory_format=torch.contiguous_format), k.clone()
        tq.qk_norm_rope(q, k, pos.to(cuda), table.to(cuda), oq, ok, _cfg(tq, 2, 128),
                        q_weight=_gpu(w[0], cuda), eps=0.0)
        _close(oq, norm_rope(parts[0], w[0], pos, table, False, 0.0), "query")
        _close(ok, norm_rope(parts[1], None, pos, table, False, 0.0), "key")


def test_zero_rows_and_empty_calls(tq, cuda):
    table = rope_table(16, 128, device=cuda)
    cfg = _cfg(tq, 2, 128)
    q = torch.zeros(3, 4, 128, dtype=FP16, device=cuda)
    k = torch.zeros(3, 2, 128, dtype=FP16, device=cuda)
    w = torch.ones(128, dtype=FP16, device=cuda)
    pos = torch.arange(3, dtype=torch.int32, device=cuda)
    oq, ok = torch.ones_like(q), torch.ones_like(k)
    tq.qk_norm_rope(q, k, pos, table, oq, ok, cfg, w, w)
    assert (oq == 0).all() and (ok == 0).all()
    oq.fill_(1.0)
    tq.qk_norm_rope(q[:0], k[:0], pos[:0], table, oq[:0], ok[:0], cfg, w, w)
    assert (oq == 1).all()


def test_more_threads_than_one_grid_line(tq, cuda):
    """71 million rows by the general kernel: 4.6e9 lanes, past the 2^32 of a grid's x."""
    N, n, D = 1 << 22, 100, 128
    table, cfg = rope_table(5000, 64), _cfg(tq, 1, D)
    parts, w, pos = _inputs(n, 16, 1, D, BF16, seed=21)
    q = torch.zeros(N, 16, D, dtype=BF16, device=cuda)
    k = torch.zeros(N, 1, D, dtype=BF16, device=cuda)
    whole = torch.zeros(N, dtype=torch.int32, device=cuda)
    for at in (0, N // 2, N - n):
        q[at:at + n], k[at:at + n], whole[at:at + n] = parts[0].to(cuda), parts[1].to(cuda), pos.to(cuda)
    tq.qk_norm_rope(q, k, whole, table.to(cuda), q, k, cfg, _gpu(w[0], cuda), _gpu(w[1], cuda))
    for at in (0, N // 2, N - n):
        _close(q[at:at + n], norm_rope(parts[0], w[0], pos, table, False, 1e-6), f"query {at}")
        _close(k[at:at + n], norm_rope(parts[1], w[1], pos, table, False, 1e-6), f"key {at}")
    del q, k
    torch.cuda.empty_cache()


@pytest.mark.parametrize("N", [3, 3000])
def test_stream_and_capture(tq, cuda, N):
    """On a stream of its own and in a graph, replayed over changed inputs."""
    parts, w, pos = _inputs(N, 16, 2, 128, BF16, seed=13)
    cfg = _cfg(tq, 2, 128)
    layout = tq.make_dense_layout_for(cfg)
    table, pos = rope_table(5000, 128, device=cuda), pos.to(cuda)
    q, k, v = (x.contiguous() for x in _views(parts, cuda, True))
    ws = [_gpu(x, cuda) for x in w]
    slots = torch.arange(N, dtype=torch.int32, device=cuda)
    oq, pool = torch.empty_like(q), tq.alloc_page_pool(N, layout, cfg)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        tq.dense_rope_append(q, k, v, pos, slots, table, oq, pool, layout, cfg, *ws,
                             stream=st.cuda_stream)
    for i in range(3):
        q.copy_(parts[0].roll(i, 0))
        k.copy_(parts[1].roll(i, 0))
        want_q, want = torch.empty_like(q), torch.zeros_like(pool)
        tq.dense_rope_append(q, k, v, pos, slots, table, want_q, want, layout, cfg, *ws)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oq, want_q) and torch.equal(pool, want)
