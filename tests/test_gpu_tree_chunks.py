"""Tree attention where a workgroup works through several chunks of tokens and
goes from one item (kv head, sequence, row tile) to the next, on every tile: the
alternating buffers, the page ids read ahead, sums rescaled when a later chunk
holds larger logits.  The tile and a workgroup's share of chunks are restated here
from the launch's rules and asserted, so that a change of those rules cannot take
the cases to other kernels unseen.  And: a row does not depend on the batch."""
from __future__ import annotations

from dataclasses import dataclass

import pytest
import torch

from oracle.step_oracle import tree_attention
from test_gpu_tree import SCHEMES, Problem

pytestmark = pytest.mark.gpu

LEAD = 2  # chunks without tokens that begin an item


@dataclass
class Plan:
    rows: int      # of a tile
    tokens: int    # of a chunk
    groups: int    # workgroups
    per: int       # chunks of a workgroup
    most: int      # chunks of tokens of the longest piece
    crossing: int  # workgroups that go from one item to another


def plan(p: Problem) -> Plan:
    """What tq_tree.hip's launch makes of a call."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    H, D = p.cfg.num_kv_heads, p.cfg.head_dim
    N, Hq, _ = p.query.shape
    G, S, turned = Hq // H, len(p.lens), p.scheme != "dense"
    rows = -(-N * G // S)
    tiles = -(-rows // 16)
    most = 1024 if not turned or D == 64 or tiles == 1 else 0 if tiles == 2 else 640
    if (D == 64 and tiles == 1) or tiles * S * p.max_kv * H <= most * cus:
        RT, WR, NW = 1, 1, 4
    elif rows <= 32:
        RT, WR, NW = 1, 2, 4
    elif rows <= 64:
        RT, WR, NW = (1, 4, 4) if turned else (2, 2, 4)
    else:
        RT, WR, NW = (2, 4, 4) if rows <= 128 else (2, 8, 8)
    C, M = (64 if WR >= 4 else 32) * (NW // WR), 16 * RT * WR
    per_cu = 3 if turned and RT == 1 and WR == 4 else 1 if WR == 1 and D == 128 else 8 // NW
    bound = (N * G // M + min(S, N)) * H * (max(1, -(-p.max_kv // C)) + LEAD)
    groups = max(1, min(cus * per_cu, bound))
    line = []  # (first chunk, chunks) of every item, by head, sequence, tile
    at = 0
    for _ in range(H):
        for n, w in zip(p.lens, p.widths):
            c = max(-(-min(n + w, p.max_kv) // C), 1) + LEAD
            for _ in range(-(-w * G // M)):
                line.append((at, c))
                at += c
    per = max(-(-at // groups), 1)
    longest, items = 0, {}
    for first, c in line:
        lo = first + LEAD
        for g in range(lo // per, (first + c - 1) // per + 1):
            longest = max(longest, min(first + c, (g + 1) * per) - max(lo, g * per))
            items[g] = items.get(g, 0) + 1
    return Plan(M, C, groups, per, longest, sum(n > 1 for n in items.values()))


def grow_keys(p, top):
    """Keys times 1 .. top from a sequence's first page to its last: later chunks have larger logits."""
    page, B = int(p.layout.page_size_bytes), p.cfg.block_size
    name, size = {"dense": ("k_offset", 2 * p.cfg.head_dim), "turbo_prod": ("k_scales_offset", 2),
                  "turbo_mse": ("k_norms_offset", 2)}[p.scheme]
    at = int(getattr(p.layout, name))
    n = B * p.cfg.num_kv_heads * size
    pages = p.pool.view(-1, page)
    x = pages[:, at:at + n].contiguous().view(p.dtype if p.scheme == "dense" else torch.float16)
    for s, (L, w) in enumerate(zip(p.lens, p.widths)):
        count = -(-(L + w) // B)
        ids = p.tables[s, :count].long()
        f = 1 + (top - 1) * torch.arange(count) / max(count - 1, 1)
        x[ids] = (x[ids].float() * f[:, None]).to(x.dtype)
    pages[:, at:at + n] = x.view(torch.uint8)


# rows of a tile, sequences, prefix lengths between, drafted tokens around, query and kv heads
SHAPES = [(16, 64, 150, 500, 2, 16, 8), (32, 24, 500, 1200, 6, 32, 8), (64, 32, 600, 1300, 6, 64, 8),
          (128, 24, 500, 1200, 12, 64, 8), (256, 8, 500, 1100, 40, 64, 8)]


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,S,lo,hi,width,Hq,H", SHAPES)
def test_several_chunks_and_items(tq, cuda, scheme, dtype, D, M, S, lo, hi, width, Hq, H):
    lens = [lo + (hi - lo) * (7 * s % S) // S - s % 5 for s in range(S)]
    widths = [width + (s % 3 - 1) * (width > 2) for s in range(S)]
    p = Problem(tq, scheme, dtype, lens, widths, Hq, H, D, seed=101)
    grow_keys(p, 8.0)
    pl = plan(p)
    print(f"[tree chunks] {scheme} {dtype} {D=} {pl}", flush=True)
    assert pl.rows == M and pl.per >= 6 and pl.most >= 4 and pl.crossing > 0
    p.check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("D", [64, 128])
def test_a_wide_tree_over_a_long_prefix(tq, cuda, scheme, dtype, D):
    """Pieces of many chunks of one item, merged; keys that grow to the end."""
    p = Problem(tq, scheme, dtype, [20011], [64], 16, 1, D, seed=102)
    grow_keys(p, 8.0)
    pl = plan(p)
    print(f"[tree chunks] {scheme} {dtype} {D=} {pl}", flush=True)
    assert pl.rows == 256 and pl.most >= 4
    p.check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("room", [0, 300_000])
def test_rows_do_not_depend_on_the_batch(tq, cuda, monkeypatch, scheme, dtype, room):
    """Each sequence alone, and all of them in another order: within the tolerance of either."""
    monkeypatch.setattr(Problem, "room", room)
    p = Problem(tq, scheme, dtype, [5000, 40, 900, 0], [6, 2, 20, 1], 16, 2, 128, seed=103)
    both, tol, _ = tree_attention(scheme, p.query, p.pool, p.tables, p.row_start, p.prefix, p.mask,
                                  p.layout, p.cfg, p.max_kv)
    whole = p.run(cuda)
    for order in ([0], [1], [2], [3], [2, 0, 3, 1], [3, 1, 1, 0]):
        rows = [torch.arange(int(p.row_start[s]), int(p.row_start[s + 1])) for s in order]
        at = torch.cat(rows)
        start = torch.tensor([0] + [len(r) for r in rows]).cumsum(0).int()
        out = torch.full((len(at), 16, 128), 5.0, dtype=dtype, device=cuda)
        tq.tree_attn_output(scheme, p.query[at].to(cuda), p.gpu[1], p.tables[order].contiguous().to(cuda),
                            start.to(cuda), p.prefix[order].to(cuda), p.mask[at].to(cuda), out, p.layout,
                            p.cfg, p.max_kv)
        got = out.cpu().double()
        assert ((got - both[at]).abs() <= tol[at]).all(), order
        assert ((got - whole[at]).abs() <= 2 * tol[at]).all(), order
