"""Batches whose sequences grow over many steps: pages for them, block tables as wide as
they are, and refusals before anything is changed."""
from __future__ import annotations

import pytest
import torch

from oracle.evict_oracle import attention_weights, compact, select
from oracle.step_oracle import agrees, tree_attention
from turborag_amd.batched import PagedBatch
from turborag_amd.turboquant_wrapper import tree_mask_from_parents

pytestmark = pytest.mark.gpu

FP16 = torch.float16


def _state(batch, scores):
    torch.cuda.synchronize()
    return (scores.cpu(), batch.pool.cpu(), [batch.table.blocks(s) for s in range(batch.S)],
            [batch.table.num_tokens(s) for s in range(batch.S)], batch.lens, batch.widths, batch.alloc.num_free())


def _same(a, b):
    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[2:] == b[2:]


def _step(tq, cuda, batch, scheme, scores, step, budget, new_widths, g):
    """Append, tree attention, weights, eviction, each against float64 of what the pages hold."""
    batch.append_new_tokens(seed=900 + step)
    bt = batch.block_tables()
    start, prefix = batch.tree_rows()
    held = [L + w for L, w in zip(batch.lens, batch.widths)]
    assert [batch.table.num_tokens(s) for s in range(batch.S)] == held
    assert bt.shape[1] * batch.B >= max(held)
    q = torch.randn(int(start[-1]), 8, batch.D, generator=g).half().to(cuda)
    mask = torch.cat([tree_mask_from_parents(list(range(-1, w - 1))) for w in batch.widths]).to(cuda)
    out = torch.empty_like(q)
    batch.tree_attention(q, start, prefix, mask, bt, out)
    old = scores.cpu()
    batch.add_weights(q, start, prefix, bt, scores)
    full, pool = scores.cpu(), batch.pool.cpu()
    host = [x.cpu() for x in (q, bt, start, prefix, mask)]
    ref, tol, _ = tree_attention(scheme, host[0], pool, *host[1:], batch.layout, batch.cfg, max(held))
    assert agrees(out.cpu().double(), ref, tol, FP16).all()
    ref, tol = attention_weights(scheme, host[0], pool, *host[1:4], batch.layout, batch.cfg, max(held), True, old, old)
    assert ((full.double() - ref).abs() <= tol).all()
    lens = batch.evict(scores, budget, bt, sink=2, recent=8, new_widths=new_widths)
    kept, new, moved = select(full, held, budget, 2, 8)
    torch.cuda.synchronize()
    assert lens == new.tolist() == [min(n, budget) for n in held]
    assert torch.equal(scores.cpu(), moved)
    assert torch.equal(batch.pool.cpu(), compact(scheme, pool, host[1], kept, batch.layout, batch.cfg))
    return lens


@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_sequences_below_the_budget_grow(tq, cuda, scheme):
    """From 10 and 3 tokens over page after page up to the budget, and on at it."""
    batch = PagedBatch(tq, scheme, [10, 3], [8, 2], kv_heads=2, q_heads=8, head_dim=128, capacity=64 + 11)
    g = torch.Generator().manual_seed(44)
    scores = torch.zeros(2, 2, 80, device=cuda)
    widths = [[8, 2], [8, 11], [8, 1], [5, 11], [11, 11], [11, 11], [3, 11], [11, 8], [1, 1]]
    for step, w in enumerate(widths):
        lens = _step(tq, cuda, batch, scheme, scores, step, 64, w, g)
    assert lens == [64, 64]
    assert batch.block_tables().shape[1] == 5
    batch.close()


def test_as_built_it_grows_into_the_spare_pages(tq, cuda):
    """Without a capacity: 18, 26, 34 and 42 tokens in the three pages that there are; then the
    append refuses and changes nothing."""
    batch = PagedBatch(tq, "turbo_mse", [10], [8], kv_heads=2, q_heads=8, head_dim=64)
    g = torch.Generator().manual_seed(45)
    scores = torch.zeros(1, 2, 64, device=cuda)
    for step in range(4):
        _step(tq, cuda, batch, "turbo_mse", scores, step, 64, None, g)
    assert batch.lens == [42]
    before = _state(batch, scores)
    with pytest.raises(RuntimeError, match="1 pages are needed, 0 are free"):
        batch.append_new_tokens(seed=950)
    assert _same(_state(batch, scores), before)
    batch.close()


def test_append_refuses_before_any_sequence_has_pages(tq, cuda):
    """The first sequence's pages would be there, the second's not."""
    batch = PagedBatch(tq, "turbo_prod", [16, 30], [1, 1], kv_heads=2, q_heads=8, head_dim=128)
    scores = torch.zeros(2, 2, 64, device=cuda)
    batch.widths = [1, 60]
    before = _state(batch, scores)
    with pytest.raises(RuntimeError, match="append_new_tokens"):
        batch.append_new_tokens(seed=951)
    assert _same(_state(batch, scores), before)
    batch.close()


@pytest.mark.parametrize("new_widths,match", [([200, 1], "pages"), ([1], "2 widths"), ([1, -1], "2 widths")])
def test_new_widths_refused(tq, cuda, new_widths, match):
    """Widths that the pool has no pages for, and such as are none: nothing is selected or moved."""
    batch = PagedBatch(tq, "turbo_mse", [90, 40], [2, 3], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=952)
    bt = batch.block_tables()
    scores = torch.rand(2, 2, 100, device=cuda)
    before = _state(batch, scores)
    with pytest.raises(ValueError, match=match):
        batch.evict(scores, 32, bt, sink=2, recent=8, new_widths=new_widths)
    assert _same(_state(batch, scores), before)
    assert batch.evict(scores, 32, bt, sink=2, recent=8, new_widths=[30, 20]) == [32, 32]
    batch.append_new_tokens(seed=953)
    assert [batch.table.num_tokens(s) for s in range(2)] == [62, 52]
    batch.close()


def test_repack_after_an_eviction(tq, cuda):
    """The last append's slots hold other tokens by then, or another sequence's pages: repack refuses
    until the next append, whose tokens it stores again."""
    batch = PagedBatch(tq, "turbo_prod", [90, 40], [2, 3], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=954)
    batch.repack()
    scores = torch.rand(2, 2, 100, device=cuda)
    before = _state(batch, scores)
    assert batch.evict(scores, 92, batch.block_tables(), sink=2, recent=8) == [92, 43]
    batch.repack()  # (nothing was evicted)
    assert torch.equal(_state(batch, scores)[1], before[1])
    batch.evict(scores, 32, batch.block_tables(), sink=2, recent=8)
    before = _state(batch, scores)
    with pytest.raises(RuntimeError, match="repack"):
        batch.repack()
    assert _same(_state(batch, scores), before)
    batch.append_new_tokens(seed=955)
    after = _state(batch, scores)
    batch.repack()
    assert _same(_state(batch, scores), after)
    batch.close()


def test_repack_after_a_refused_eviction(tq, cuda):
    batch = PagedBatch(tq, "turbo_prod", [90, 40], [2, 3], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=956)
    scores = torch.rand(2, 2, 100, device=cuda)
    before = _state(batch, scores)
    with pytest.raises(RuntimeError):
        batch.evict(scores, 8, batch.block_tables(), sink=4, recent=8)
    batch.repack()
    assert _same(_state(batch, scores), before)
    batch.close()


@pytest.mark.parametrize("change,match", [
    (lambda bt: bt.long(), "int32"), (lambda bt: bt.cpu(), "GPU tensor"), (lambda bt: bt[:1], "kept must be"),
    (lambda bt: bt.repeat_interleave(2, 1)[:, ::2], "contiguous"), (lambda bt: bt[None], "2 dimensions")])
def test_tables_refused_before_scores_move(tq, cuda, change, match):
    """What the move would refuse is refused before the selection moves the scores."""
    batch = PagedBatch(tq, "turbo_mse", [90, 40], [2, 3], kv_heads=2, q_heads=8, head_dim=64)
    batch.append_new_tokens(seed=957)
    bt = batch.block_tables()
    scores = torch.rand(2, 2, 100, device=cuda)
    before = _state(batch, scores)
    with pytest.raises(ValueError, match=match):
        batch.evict(scores, 32, change(bt), sink=2, recent=8)
    assert _same(_state(batch, scores), before)
    assert batch.evict(scores, 32, bt, sink=2, recent=8) == [32, 32]
    batch.close()
