"""Selection and compaction (select_kv, compact_kv): equal to plain
restatements, value for value and byte for byte; and the eviction of a batch
with the steps around it."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle.evict_oracle import attention_weights, compact, select
from oracle.step_oracle import agrees, tree_attention
from test_gpu_tree import SCHEMES, Problem
from turborag_amd.batched import PagedBatch
from turborag_amd.turboquant_wrapper import rope_axes, rope_table, tree_mask_from_parents

pytestmark = pytest.mark.gpu

I32 = torch.int32
FP16 = torch.float16
INF, NAN = float("inf"), float("nan")


def _bits(x):
    return x.cpu().contiguous().view(torch.int32)


def _select(tq, cuda, scores, lens, budget, sink, recent, in_place=False, want_new=True):
    x = scores.to(cuda)
    S, H, T = scores.shape
    kept = torch.full((S, H, budget), 77, dtype=I32, device=cuda)
    new = torch.full((S,), 77, dtype=I32, device=cuda) if want_new else None
    out = x if in_place else torch.full_like(x, 5.0)
    tq.select_kv(x, torch.tensor(lens, dtype=I32, device=cuda), kept, new, sink=sink, recent=recent,
                 out_scores=out)
    torch.cuda.synchronize()
    return kept.cpu(), None if new is None else new.cpu(), out.cpu()


def _check_select(tq, cuda, scores, lens, budget, sink, recent):
    want = select(scores, lens, budget, sink, recent)
    for in_place in (False, True):
        kept, new, out = _select(tq, cuda, scores, lens, budget, sink, recent, in_place)
        assert torch.equal(kept, want[0])
        assert torch.equal(new, want[1])
        assert torch.equal(_bits(out), _bits(want[2]))


def _values(kind, shape, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.rand(shape, generator=g)
    if kind == "softmax":
        return torch.exp(3 * torch.randn(shape, generator=g))
    if kind == "equal":
        return torch.full(shape, 0.25)
    if kind == "ties":
        return (x * 6).floor()
    if kind == "signs":
        return torch.randn(shape, generator=g)
    if kind == "close":  # they differ in the last bits alone
        return torch.ones(shape) + (x * 40).floor() * 2.0 ** -23
    special = torch.tensor([0.0, -0.0, INF, -INF, NAN, -NAN, 1e-45, -1e-45, 1.0, 3e38, -3e38])
    return special[(x * len(special)).long()]


@pytest.mark.parametrize("kind", ["softmax", "equal", "ties", "signs", "close", "special"])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([1], 1, 0, 0), ([0, 5], 3, 1, 1), ([64, 65, 63], 64, 4, 32), ([1143], 256, 4, 32),
    ([1000, 999, 2], 1, 0, 0), ([500, 501], 500, 0, 0), ([3000, 40], 1500, 0, 0),
    ([2049, 1024], 100, 40, 60),      # nothing left to the scores
    ([700], 699, 0, 1), ([5000], 4097, 16, 1000)])
def test_select(tq, cuda, kind, lens, budget, sink, recent):
    _check_select(tq, cuda, _values(kind, (len(lens), 2, max(max(lens), 1)), seed=budget), lens, budget, sink,
                  recent)


def test_select_ragged_rows_and_bounds(tq, cuda):
    """Scores wider than any length; lengths past the scores' width or below zero are cut."""
    x = _values("softmax", (4, 3, 900), seed=1)
    _check_select(tq, cuda, x, [300, 2000, -4, 0], 128, 4, 16)
    kept, new, out = _select(tq, cuda, x, [300, 2000, -4, 0], 128, 4, 16, want_new=False)
    assert new is None and torch.equal(kept, select(x, [300, 2000, -4, 0], 128, 4, 16)[0])


@pytest.mark.parametrize("S,H,T,budget", [(2, 2, 100_003, 8192), (1, 1, 300_000, 70_000), (40, 8, 2000, 333)])
def test_select_long(tq, cuda, S, H, T, budget):
    """By a stable sort: rows of hundreds of thousands of tokens, hundreds of rows."""
    x = _values("softmax", (S, H, T), seed=2)
    x[..., ::7] = x[..., :1]  # many ties
    kept, new, out = _select(tq, cuda, x, [T] * S, budget, 4, 100)
    key = x.clone()
    key[..., :4] = key[..., T - 100:] = INF
    want = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget].sort(dim=-1).values
    assert torch.equal(kept.long(), want)
    assert (new == budget).all()
    assert torch.equal(out[..., :budget], x.gather(2, want)) and (out[..., budget:] == 0).all()


@pytest.mark.parametrize("T", [2047, 2048, 2049, 8192, 8193, 32768, 32769, 65537])
@pytest.mark.parametrize("kind", ["softmax", "ties", "special"])
def test_select_widths(tq, cuda, T, kind):
    """Around the tiles that a workgroup holds, with lengths from one to all of it."""
    x = _values(kind, (5, 2, T), seed=T)
    lens, budget, sink, recent = [T, T - 1, T // 2, 1, 700], 600, 3, 50
    for in_place in (False, True):
        kept, new, out = _select(tq, cuda, x, lens, budget, sink, recent, in_place)
        for s, L in enumerate(lens):
            n = min(L, budget)
            key = torch.where(x[s, :, :L].isnan(), -INF, x[s, :, :L].double())
            # (NaN below -infinity: behind every number by a second, stable sort)
            order = key.sort(dim=-1, descending=True, stable=True).indices
            nan = x[s, :, :L].isnan().gather(1, order)
            order = order.gather(1, nan.to(torch.int8).sort(dim=-1, stable=True).indices)
            rank = torch.empty_like(order).scatter_(1, order, torch.arange(L).expand(2, L))
            if L > budget:
                rank[:, :sink] = -1
                rank[:, L - recent:] = -1
                mid = torch.arange(sink, L - recent)
                place = rank[:, mid].argsort(dim=-1, stable=True).argsort(dim=-1, stable=True)
                rank[:, mid] = place
                keep = (rank < budget - sink - recent)
            else:
                keep = torch.ones(2, L, dtype=torch.bool)
            want = torch.stack([k.nonzero()[:, 0] for k in keep]).int()
            assert torch.equal(kept[s, :, :n], want) and (kept[s, :, n:] == -1).all() and new[s] == n
            assert torch.equal(_bits(out[s, :, :n]), _bits(x[s].gather(1, want.long())))
            assert (_bits(out[s, :, n:]) == 0).all()


# ── compaction ───────────────────────────────────────────────────────────── #

def _kept(S, H, lens, budget, how, seed):
    g = torch.Generator().manual_seed(seed)
    kept = torch.full((S, H, budget), -1, dtype=I32)
    for s in range(S):
        for h in range(H):
            L, n = lens[s], min(lens[s], budget)
            if how == "random":
                ids = torch.randperm(L, generator=g)[:n].sort().values
            elif how == "last":
                ids = torch.arange(L - n, L)
            elif how == "hole":  # one token goes: every later place moves by one
                n = min(n, max(L - 1, 0))
                ids = torch.cat([torch.arange(1), torch.arange(2, n + 1)])[:n] if L > 1 else torch.arange(n)
            else:
                ids = torch.arange(n)
            kept[s, h, :len(ids)] = ids.int()
    return kept


def _compact(tq, cuda, p, kept, out_tables=None, pool=None):
    pool = (p.pool if pool is None else pool).to(cuda)
    tq.compact_kv(p.scheme, pool, p.tables.to(cuda), kept.to(cuda), p.layout, p.cfg,
                  out_block_tables=None if out_tables is None else out_tables.to(cuda))
    torch.cuda.synchronize()
    return pool.cpu()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("how", ["random", "last", "hole", "first"])
@pytest.mark.parametrize("lens,budget,H,B", [
    ([1], 1, 1, 16), ([0, 3], 2, 2, 16), ([100, 17, 250], 60, 2, 16), ([700], 650, 4, 16),
    ([2100, 1500], 1400, 2, 16), ([90, 61], 40, 3, 7)])
def test_compact_in_place(tq, cuda, scheme, dtype, D, how, lens, budget, H, B):
    """Chunks of places that other chunks' tokens come from."""
    p = Problem(tq, scheme, dtype, lens, [0] * len(lens), H, H, D, B=B, seed=21)
    kept = _kept(len(lens), H, lens, budget, how, seed=22)
    got = _compact(tq, cuda, p, kept)
    assert torch.equal(got, compact(scheme, p.pool, p.tables, kept, p.layout, p.cfg))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("lens,budget,H,B", [([1], 1, 1, 16), ([100, 17, 250], 60, 2, 16),
                                             ([2100, 1500], 1400, 2, 16), ([90, 61], 40, 3, 7)])
def test_compact_into_other_pages(tq, cuda, scheme, dtype, D, lens, budget, H, B):
    """The originals stay; two sequences may share them."""
    p = Problem(tq, scheme, dtype, lens, [0] * len(lens), H, H, D, B=B, seed=23)
    page = int(p.layout.page_size_bytes)
    P, S = p.pool.numel() // page, len(lens)
    per = (budget + B - 1) // B
    if S > 1:
        p.tables[1] = p.tables[0]
        lens = [lens[0], min(lens[0], lens[1])] + lens[2:]
    out = (P + torch.randperm(S * per, generator=torch.Generator().manual_seed(3))).view(S, per).int()
    pool = torch.cat([p.pool, torch.full((S * per * page,), 0xAB, dtype=torch.uint8)])
    kept = _kept(S, H, lens, budget, "random", seed=24)
    got = _compact(tq, cuda, p, kept, out, pool)
    assert torch.equal(got, compact(scheme, pool, p.tables, kept, p.layout, p.cfg, out))
    assert torch.equal(got[:p.pool.numel()], p.pool)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_compact_skips_what_has_no_place(tq, cuda, scheme, dtype):
    """Unmapped pages on either side, places past the tables' ends, kept that does not rise."""
    p = Problem(tq, scheme, dtype, [200, 100], [0, 0], 2, 2, 128, seed=25)
    p.tables[0, 2], p.tables[0, 7], p.tables[1, 0] = -1, -1, -1
    kept = _kept(2, 2, [200, 100], 90, "random", seed=26)
    kept[0, 0, 5], kept[0, 1, 80], kept[1, 0, 3] = 2 ** 31 - 1, 5, -2 ** 31
    got = _compact(tq, cuda, p, kept)
    assert torch.equal(got, compact(scheme, p.pool, p.tables, kept, p.layout, p.cfg))
    page = int(p.layout.page_size_bytes)
    out = torch.full((2, 3), -1, dtype=I32)  # fewer places than kept tokens
    out[0, :], out[1, 1] = torch.arange(3) + p.pool.numel() // page, 3 + p.pool.numel() // page
    pool = torch.cat([p.pool, torch.zeros(4 * page, dtype=torch.uint8)])
    got = _compact(tq, cuda, p, kept, out, pool)
    assert torch.equal(got, compact(scheme, pool, p.tables, kept, p.layout, p.cfg, out))


@pytest.mark.parametrize("scheme,dtype", [("dense", FP16), ("turbo_prod", FP16)])
def test_compact_many_chunks_in_place(tq, cuda, scheme, dtype):
    """A long sequence: hundreds of chunks in order, by the cells as a plain gather moves them."""
    H, D, B, L, budget = 2, 128, 16, 40_000, 30_000
    p = Problem(tq, scheme, dtype, [L], [0], H, H, D, seed=27)
    for how in ("random", "hole"):
        kept = _kept(1, H, [L], budget, how, seed=28)
        got = _compact(tq, cuda, p, kept)
        page = int(p.layout.page_size_bytes)
        want = p.pool.clone()
        from oracle.evict_oracle import regions
        for h in range(H):
            src = kept[0, h][kept[0, h] >= 0].long()
            dst = torch.arange(src.numel())
            for off, n in regions(scheme, p.layout, p.cfg):
                def at(t):
                    return (p.tables[0, t // B].long() * page + off + (t % B * H + h) * n)[:, None] + torch.arange(n)
                want[at(dst)] = p.pool[at(src)]
        assert torch.equal(got, want)


def test_two_streams_and_graphs(tq, cuda):
    """In-place compactions of two pools at once on two streams, captured and replayed."""
    ps = [Problem(tq, "dense", FP16, [3000, 2000], [0, 0], 2, 2, 128, seed=31 + k) for k in range(2)]
    kept = [_kept(2, 2, [3000, 2000], 1200, "random", seed=33 + k).to(cuda) for k in range(2)]
    want = [compact("dense", p.pool, p.tables, k.cpu(), p.layout, p.cfg) for p, k in zip(ps, kept)]
    pools, tables = [p.pool.to(cuda) for p in ps], [p.tables.to(cuda) for p in ps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def call(k):
        tq.compact_kv("dense", pools[k], tables[k], kept[k], ps[k].layout, ps[k].cfg,
                      stream=streams[k].cuda_stream)

    torch.cuda.synchronize()
    for k in range(2):
        call(k)
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(pools[k].cpu(), want[k])
    graphs = []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k], stream=streams[k]):
            call(k)
    for _ in range(3):
        for k in range(2):
            pools[k].copy_(ps[k].pool)
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(pools[k].cpu(), want[k])
        call(0)  # (eager between replays)
        torch.cuda.synchronize()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_eviction_in_a_graph(tq, cuda, scheme, dtype):
    """Weights, selection and compaction as one graph on a stream: every replay, with lengths that
    change between them, has the results of the calls one by one."""
    p = Problem(tq, scheme, dtype, [900, 400], [4, 4], 16, 2, 128, seed=51)
    pool, tables, q, start = (x.to(cuda) for x in (p.pool, p.tables, p.query, p.row_start))
    prefix, lens = torch.zeros(2, dtype=I32, device=cuda), torch.zeros(2, dtype=I32, device=cuda)
    scores, kept = torch.zeros(2, 2, 904, device=cuda), torch.zeros(2, 2, 128, dtype=I32, device=cuda)

    def step(stream):
        tq.attn_weights(scheme, q, pool, tables, start, prefix, scores, p.layout, p.cfg, 904, scores_in=scores,
                        decay=0.5, stream=stream)
        tq.select_kv(scores, lens, kept, sink=2, recent=10, out_scores=scores, stream=stream)
        tq.compact_kv(scheme, pool, tables, kept, p.layout, p.cfg, stream=stream)

    def reset(k):
        pool.copy_(p.pool)
        scores.copy_(torch.rand(2, 2, 904, generator=torch.Generator().manual_seed(k)))
        prefix.copy_(torch.tensor([900 - 100 * k, 400 - 7 * k], dtype=I32))
        lens.copy_(prefix + 4)
        torch.cuda.synchronize()

    st = torch.cuda.Stream()
    want = []
    for k in range(4):
        reset(k)
        step(st.cuda_stream)
        torch.cuda.synchronize()
        want.append([x.clone() for x in (scores, kept, pool)])
        assert (kept >= 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(st.cuda_stream)
    for k in (2, 0, 3, 1):
        reset(k)
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip((scores, kept, pool), want[k]):
            assert torch.equal(got, ref)


# ── together ─────────────────────────────────────────────────────────────── #

def test_a_document_with_images(tq, cuda):
    """Positions of three axes into dense pages, the last tokens' weights, selection, compaction,
    then a drafted tree over what is left: against the same in float64 from the pages' values."""
    N, Hq, H, D, B, budget, window = 700, 8, 2, 128, 16, 200, 16
    g = torch.Generator().manual_seed(41)
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim, cfg.block_size = H, D, B
    layout, page = tq.make_dense_layout_for(cfg), None
    page = int(layout.page_size_bytes)
    pages = (N + 8 + B - 1) // B
    order = torch.randperm(pages, generator=g).int()
    tables = order[None].to(cuda)
    t = torch.arange(N)
    slots = (order[t // B] * B + t % B).int().to(cuda)
    pos = torch.stack([t // 100, t // 10 % 10, t % 10]).int().to(cuda)
    qkv = torch.randn(N, Hq + 2 * H, D, generator=g).half().to(cuda)
    table, axes = rope_table(1000, D).to(cuda), rope_axes([16, 24, 24])
    pool = torch.zeros(pages * page, dtype=torch.uint8, device=cuda)
    q = torch.empty(N, Hq, D, dtype=FP16, device=cuda)
    tq.dense_rope_append(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], pos, slots, table, q, pool, layout, cfg,
                         axes=axes)
    scores = torch.zeros(1, H, N, device=cuda)
    last = q[N - window:].contiguous()
    start = torch.tensor([0, window], dtype=I32, device=cuda)
    prefix = torch.tensor([N - window], dtype=I32, device=cuda)
    tq.attn_weights("dense", last, pool, tables, start, prefix, scores, layout, cfg, N)
    before = pool.clone()
    kept = torch.empty(1, H, budget, dtype=I32, device=cuda)
    new = torch.empty(1, dtype=I32, device=cuda)
    moved = torch.empty_like(scores)
    tq.select_kv(scores, torch.tensor([N], dtype=I32, device=cuda), kept, new, sink=4, recent=window,
                 out_scores=moved)
    tq.compact_kv("dense", pool, tables, kept, layout, cfg)
    torch.cuda.synchronize()
    ref, tol = attention_weights("dense", last.cpu(), before.cpu(), tables.cpu(), start.cpu(), prefix.cpu(), layout,
                                 cfg, N, True, torch.zeros(1, H, N))
    assert ((scores.cpu().double() - ref).abs() <= tol).all()
    assert torch.equal(kept.cpu(), select(scores.cpu(), [N], budget, 4, window)[0]) and int(new) == budget
    assert torch.equal(pool.cpu(), compact("dense", before.cpu(), tables.cpu(), kept.cpu(), layout, cfg))
    # drafted tokens behind what is left; their positions go on from the document's
    w = 5
    at = torch.arange(w) + budget
    slots = (order[at // B] * B + at % B).int().to(cuda)
    pos = torch.full((3, w), 7, dtype=I32, device=cuda) + torch.arange(w, dtype=I32, device=cuda)
    qkv = torch.randn(w, Hq + 2 * H, D, generator=g).half().to(cuda)
    q = torch.empty(w, Hq, D, dtype=FP16, device=cuda)
    tq.dense_rope_append(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], pos, slots, table, q, pool, layout, cfg,
                         axes=axes)
    mask = tree_mask_from_parents([-1, 0, 0, 1, 2])
    out = torch.empty_like(q)
    rows = torch.tensor([0, w], dtype=I32)
    tq.tree_attn_output("dense", q, pool, tables, rows.to(cuda), new, mask.to(cuda), out, layout, cfg, budget + w)
    torch.cuda.synchronize()
    ref, tol, _ = tree_attention("dense", q.cpu(), pool.cpu(), tables.cpu(), rows, new.cpu(), mask, layout, cfg,
                                 budget + w)
    assert agrees(out.cpu().double(), ref, tol, FP16).all()


@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_batch_under_a_budget(tq, cuda, scheme):
    """Steps of a batch: append, tree attention, weights, eviction; the next step appends to the
    pages that were given back."""
    batch = PagedBatch(tq, scheme, [300, 90, 33], [3, 2, 4], kv_heads=2, q_heads=8, head_dim=128)
    H, D, budget = 2, 128, 64
    g = torch.Generator().manual_seed(42)
    scores = torch.zeros(3, H, 400, device=cuda)
    free = batch.alloc.num_free()
    for step in range(3):
        batch.append_new_tokens(seed=900 + step)
        bt = batch.block_tables()
        start, prefix = batch.tree_rows()
        n = int(start[-1])
        q = torch.randn(n, 8, D, generator=g).half().to(cuda)
        mask = torch.cat([tree_mask_from_parents(list(range(-1, w - 1))) for w in batch.widths]).to(cuda)
        out = torch.empty_like(q)
        batch.tree_attention(q, start, prefix, mask, bt, out)
        old = scores.cpu()
        batch.add_weights(q, start, prefix, bt, scores)
        torch.cuda.synchronize()
        pool = batch.pool.cpu()
        most = max(L + w for L, w in zip(batch.lens, batch.widths))
        ref, tol, _ = tree_attention(scheme, q.cpu(), pool, bt.cpu(), start.cpu(), prefix.cpu(), mask.cpu(),
                                     batch.layout, batch.cfg, most)
        assert agrees(out.cpu().double(), ref, tol, FP16).all()
        ref, tol = attention_weights(scheme, q.cpu(), pool, bt.cpu(), start.cpu(), prefix.cpu(), batch.layout,
                                     batch.cfg, most, True, old, old)
        assert ((scores.cpu().double() - ref).abs() <= tol).all()
        full = scores.cpu()
        held = [L + w for L, w in zip(batch.lens, batch.widths)]
        lens = batch.evict(scores, budget, bt, sink=2, recent=8, new_widths=[2, 2, 2])
        torch.cuda.synchronize()
        kept, new, moved = select(full, held, budget, 2, 8)
        assert lens == new.tolist() == [min(x, budget) for x in held]
        assert torch.equal(scores.cpu(), moved)
        assert torch.equal(batch.pool.cpu(), compact(scheme, pool, bt.cpu(), kept, batch.layout, batch.cfg))
        assert [batch.table.num_tokens(s) for s in range(3)] == lens
    assert batch.alloc.num_free() > free
    batch.close()


def test_batch_evicts_on_another_stream(tq, cuda):
    """What evict allocates belongs to the stream that it runs on, not to the caller's; it refuses
    scores and tables that hold fewer tokens than the batch."""
    batch = PagedBatch(tq, "turbo_mse", [300, 90], [3, 2], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=7)
    bt = batch.block_tables()
    held = [303, 92]
    full = torch.rand(2, 2, 320, generator=torch.Generator().manual_seed(43))
    scores = full.to(cuda)
    with pytest.raises(ValueError, match="303 tokens"):
        batch.evict(scores[:, :, :302].contiguous(), 64, bt)
    with pytest.raises(ValueError, match="303 tokens"):
        batch.evict(scores, 64, bt[:, :18].contiguous())
    assert [batch.table.num_tokens(s) for s in range(2)] == held
    torch.cuda.synchronize()
    pool = batch.pool.cpu()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy = torch.randn(2048, 2048, device=cuda)
        for _ in range(20):  # evict's kernels wait behind these
            busy = (busy @ busy).clamp(-1.0, 1.0)
    lens = batch.evict(scores, 64, bt, sink=2, recent=8, stream=side.cuda_stream)
    other = [torch.full((2, 2, 64), -1, dtype=torch.int32, device=cuda) for _ in range(4)]
    torch.cuda.synchronize()
    kept, new, moved = select(full, held, 64, 2, 8)
    assert lens == new.tolist()
    assert torch.equal(scores.cpu(), moved)
    assert torch.equal(batch.pool.cpu(), compact("turbo_mse", pool, bt.cpu(), kept, batch.layout, batch.cfg))
    assert all(int(x.max()) == -1 for x in other)
    batch.close()


def test_host_threads_on_one_stream(tq, cuda):
    """In-place compactions from four threads on one stream: each call's flags are its
    own until its last launch."""
    ps = [Problem(tq, "dense", torch.float16, [1500 + 64 * k, 700], [0, 0], 2, 2, 128, seed=70 + k) for k in range(4)]
    keeps = [_kept(2, 2, [1500 + 64 * k, 700], 900 + k, "random", seed=80 + k) for k in range(4)]
    want = [compact("dense", p.pool, p.tables, kept, p.layout, p.cfg) for p, kept in zip(ps, keeps)]
    pools = [[p.pool.to(cuda) for _ in range(6)] for p in ps]
    tables, kepts = [p.tables.to(cuda) for p in ps], [k.to(cuda) for k in keeps]
    stream, errors = torch.cuda.Stream(), []
    torch.cuda.synchronize()

    def work(k):
        try:
            torch.cuda.set_device(cuda)
            for pool in pools[k]:
                tq.compact_kv("dense", pool, tables[k], kepts[k], ps[k].layout, ps[k].cfg,
                              stream=stream.cuda_stream)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for k in range(4):
        for pool in pools[k]:
            assert torch.equal(pool.cpu(), want[k])
