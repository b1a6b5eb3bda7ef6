"""Infinite and NaN values of dense pages in chunks that every row sees whole: the
rows of their sequence hold them, with their sign, the other rows do not."""
from __future__ import annotations

import pytest
import torch

from test_gpu_tree import Problem

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
FAR = 300_000
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("widths,Hq,H,room", [
    ([4, 3], 2, 1, 0), ([6, 30], 6, 2, 0), ([8, 8], 6, 2, FAR), ([12, 10], 8, 2, FAR), ([14, 14], 16, 2, FAR),
    ([30, 30], 32, 2, FAR)])
@pytest.mark.parametrize("L", [700, 5000])
def test_values_of_the_prefix(tq, cuda, monkeypatch, widths, Hq, H, room, dtype, D, L):
    monkeypatch.setattr(Problem, "room", room)
    p = Problem(tq, "dense", dtype, [L, 450], widths, Hq, H, D, seed=81)
    want = p.run(cuda)
    clean = p.pool.clone()
    w = widths[0]
    for values, expect in (({200: INF}, INF), ({3: -INF, 640: -INF}, -INF), ({7: INF, L - 300: -INF}, NAN),
                           ({L // 2: NAN}, NAN)):
        p.pool = clean.clone()
        for t, value in values.items():
            p.fill_token(0, t, value, "v")
        got = p.run(cuda)
        mine, rest = got[:w], got[w:]
        assert (torch.isnan(mine) if expect != expect else mine == expect).all(), values
        # the other sequence's: the same bits as before
        assert torch.equal(rest, want[w:])


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("widths,Hq,H,room", [([4, 3], 2, 1, 0), ([8, 8], 6, 2, FAR), ([12, 10], 8, 2, FAR),
                                              ([14, 14], 16, 2, FAR), ([30, 30], 32, 2, FAR)])
def test_one_value(tq, cuda, monkeypatch, widths, Hq, H, room, dtype):
    """A single infinite element: its dimension of the heads that read it, and nothing else."""
    monkeypatch.setattr(Problem, "room", room)
    p = Problem(tq, "dense", dtype, [900, 300], widths, Hq, H, 128, seed=82)
    want = p.run(cuda)
    _, v, _ = p.cell_bytes(0, 333)
    p.pool[v + 2 * 77:v + 2 * 78] = torch.tensor([-INF], dtype=dtype).view(torch.uint8)  # kv head 0
    got = p.run(cuda)
    w, G = widths[0], Hq // H
    assert (got[:w, :G, 77] == -INF).all()
    got[:w, :G, 77] = want[:w, :G, 77]
    # (the other dimensions' sums are added up in the same order)
    assert torch.equal(got, want)


def test_not_finite_queries(tq, cuda):
    """A NaN in one row's query: that row alone."""
    p = Problem(tq, "dense", FP16, [900], [20], 16, 2, 128, seed=83)
    want = p.run(cuda)
    p.query[7, 3, 50] = NAN
    got = p.run(cuda)
    assert torch.isnan(got[7, 3]).all()
    got[7, 3] = want[7, 3]
    assert torch.equal(got, want)
