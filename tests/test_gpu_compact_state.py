"""In-place compaction over a workspace that another call's kernels write over, as two
graphs of one stream do that are replayed at once against the rule: the state is forced
from the host (tq_test_compact).  Nothing out of bounds is touched, no cell that is still
to be read is written over, and the next call says that cells were not moved."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle.evict_oracle import compact
from test_gpu_evict import _compact, _kept, _select
from test_gpu_tree import SCHEMES, Problem
from turborag_amd.batched import PagedBatch

pytestmark = pytest.mark.gpu


@pytest.fixture
def state(tq):
    f = tq.lib.tq_test_compact
    f.argtypes, f.restype = [ctypes.c_uint32, ctypes.c_int], ctypes.c_int
    yield f
    f(0, -1)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("first", [0x7FFFFFFF, 0x80000000, 0xFF800000, 0xFFFFF000, 100])
def test_tickets_out_of_range(tq, cuda, state, scheme, dtype, first):
    """Any bits (those of -infinity among them) where a row's tickets lie: a workgroup whose ticket
    names no chunk, above them all or below 0 as a signed number, moves nothing."""
    p = Problem(tq, scheme, dtype, [900, 700], [0, 0], 2, 2, 128, seed=61)
    kept = _kept(2, 2, [900, 700], 600, "random", seed=62)
    state(first, -1)
    assert torch.equal(_compact(tq, cuda, p, kept), p.pool)
    state(0, -1)
    with pytest.raises(RuntimeError, match="left cells unmoved"):
        _compact(tq, cuda, p, kept)
    assert torch.equal(_compact(tq, cuda, p, kept), compact(scheme, p.pool, p.tables, kept, p.layout, p.cfg))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_waits_given_up(tq, cuda, state, scheme, dtype, D):
    """Without a poll every wait is given up: the chunks that overlap one before them stay as they
    were, the others are moved.  The next call refuses, once."""
    lens, budget = [2100, 1500], 1400
    p = Problem(tq, scheme, dtype, lens, [0, 0], 2, 2, D, seed=63)
    kept = _kept(2, 2, lens, budget, "random", seed=64)
    T = 256 * 8 // (2 * (D // 8 if scheme == "dense" else D // 32))  # tokens of a chunk
    written = kept.clone()
    for s in range(2):
        for h in range(2):
            for c in range(1, -(-budget // T)):
                if any(kept[s, h, k * T + T - 1] >= c * T and kept[s, h, k * T] < (c + 1) * T for k in range(c)):
                    written[s, h, c * T:(c + 1) * T] = -1
    assert (written >= 0).any() and (written != kept).any()
    state(0, 0)
    got = _compact(tq, cuda, p, kept)
    state(0, -1)
    assert torch.equal(got, compact(scheme, p.pool, p.tables, written, p.layout, p.cfg))
    scores = torch.rand(1, 1, 100)
    with pytest.raises(RuntimeError, match="left cells unmoved"):
        _select(tq, cuda, scores, [100], 10, 0, 0)
    _select(tq, cuda, scores, [100], 10, 0, 0)
    assert torch.equal(_compact(tq, cuda, p, kept), compact(scheme, p.pool, p.tables, kept, p.layout, p.cfg))


def test_a_batch_hears_of_it(tq, cuda, state):
    """evict refuses before it changes anything."""
    batch = PagedBatch(tq, "turbo_mse", [700, 90], [3, 2], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=7)
    bt = batch.block_tables()
    scores = torch.rand(2, 2, 720, device=cuda)
    old, pool = scores.clone(), batch.pool.clone()
    p = Problem(tq, "dense", torch.float16, [500], [0], 1, 1, 64, seed=65)
    state(100, -1)
    _compact(tq, cuda, p, _kept(1, 1, [500], 400, "hole", seed=66))
    state(0, -1)
    with pytest.raises(RuntimeError, match="left cells unmoved"):
        batch.evict(scores, 64, bt, sink=2, recent=8)
    assert torch.equal(scores, old) and torch.equal(batch.pool, pool)
    assert [batch.table.num_tokens(s) for s in range(2)] == [703, 92]
    assert batch.evict(scores, 64, bt, sink=2, recent=8) == [64, 64]
    batch.close()


def test_replays_say_so(tq, cuda, state):
    """What a graph's replays leave unmoved is reported too."""
    p = Problem(tq, "dense", torch.float16, [500], [0], 1, 1, 128, seed=67)
    kept = _kept(1, 1, [500], 400, "hole", seed=68)
    want = compact("dense", p.pool, p.tables, kept, p.layout, p.cfg)
    pool, tables, on_gpu = p.pool.to(cuda), p.tables.to(cuda), kept.to(cuda)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        tq.compact_kv("dense", pool.clone(), tables, on_gpu, p.layout, p.cfg, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    graphs = []
    for polls in (-1, 0):
        state(0, polls)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            tq.compact_kv("dense", pool, tables, on_gpu, p.layout, p.cfg, stream=stream.cuda_stream)
    state(0, -1)
    for _ in range(3):
        pool.copy_(p.pool)
        graphs[1].replay()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="left cells unmoved"):
            tq.compact_kv("dense", pool, tables, on_gpu, p.layout, p.cfg)
        pool.copy_(p.pool)
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(pool.cpu(), want)
