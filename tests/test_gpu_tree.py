"""Attention of drafted token trees over paged caches (tree_attn_output)
against float64, with tolerances that count roundings
(oracle/step_oracle.py)."""
from __future__ import annotations

import pytest
import torch

from oracle.step_oracle import agrees, tree_attention
from turborag_amd.turboquant_wrapper import tree_mask_from_parents

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
SCHEMES = [("dense", FP16), ("dense", BF16), ("turbo_prod", FP16), ("turbo_mse", FP16)]


class Problem:
    """Sequences with prefixes `lens` and `widths` drafted tokens in shuffled pages, on the CPU."""

    room = 0  # tokens that max_kv_len and the block tables hold beyond the longest sequence

    def __init__(self, tq, scheme, dtype, lens, widths, Hq, H, D, B=16, seed=0, words=None,
                 kv_scale=1.0, q_scale=1.0, extra_rows=0, extra_blocks=0):
        g = torch.Generator().manual_seed(seed)
        self.tq, self.scheme, self.dtype = tq, scheme, dtype
        self.cfg = tq.default_config()
        self.cfg.num_kv_heads, self.cfg.head_dim, self.cfg.block_size = H, D, B
        self.layout = {"dense": tq.make_dense_layout_for, "turbo_prod": tq.make_layout_for,
                       "turbo_mse": tq.make_mse_layout_for}[scheme](self.cfg)
        page = int(self.layout.page_size_bytes)
        total = [n + w for n, w in zip(lens, widths)]
        counts = [(n + B - 1) // B for n in total]
        S, P = len(lens), sum(counts) + 1
        extra_blocks += min(self.room // B, 4_000_000 // max(S, 1))
        order = torch.randperm(P, generator=g).int()
        self.tables = torch.full((S, max(max(counts, default=0), 1) + extra_blocks), -1,
                                 dtype=torch.int32)
        at = 0
        for s, n in enumerate(counts):
            self.tables[s, :n] = order[at:at + n]
            at += n
        if scheme == "dense":
            self.pool = (torch.randn(P * page // 2, generator=g) * kv_scale).to(dtype).view(torch.uint8)
        else:  # random codes; scales around kv_scale
            self.pool = torch.randint(0, 256, (P * page,), generator=g, dtype=torch.uint8)
            lay, cells = self.layout, B * H
            names = (("k_residual_scales_offset", "k_scales_offset", "v_scales_offset")
                     if scheme == "turbo_prod" else ("k_norms_offset", "v_norms_offset"))
            v = self.pool.view(P, page)
            for i, nm in enumerate(names):
                mean = 0.2 if "residual" in nm else 1.3 * kv_scale
                sc = (mean * torch.exp(0.2 * torch.randn(P, cells, generator=g))).half()
                off = int(getattr(lay, nm))
                v[:, off:off + 2 * cells] = sc.view(torch.uint8)
        self.row_start = torch.tensor([sum(widths[:s]) for s in range(S + 1)], dtype=torch.int32)
        self.prefix = torch.tensor(lens, dtype=torch.int32)
        N = sum(widths) + extra_rows
        words = words or max(1, (max(widths, default=1) + 31) // 32)
        self.mask = torch.zeros(N, words, dtype=torch.int32)
        for s, w in enumerate(widths):
            par = [-1 if j == 0 else int(torch.randint(-1, j, (1,), generator=g)) for j in range(w)]
            m = tree_mask_from_parents(par)
            r = int(self.row_start[s])
            self.mask[r:r + w, :m.shape[1]] = m[:, :words]
        self.query = (torch.randn(N, Hq, D, generator=g) * q_scale).to(dtype)
        self.max_kv = self.tables.shape[1] * B if self.room else max(total, default=0)
        self.lens, self.widths = lens, widths

    def cell_bytes(self, s, t):
        """(start of K's row, of V's row, bytes) of token t, head 0, of a dense page."""
        B, H, D = self.cfg.block_size, self.cfg.num_kv_heads, self.cfg.head_dim
        at = int(self.tables[s, t // B]) * int(self.layout.page_size_bytes) + t % B * H * 2 * D
        return at + int(self.layout.k_offset), at + int(self.layout.v_offset), H * 2 * D

    def fill_token(self, s, t, value, what="kv"):
        """Every K and / or V value of token t to `value` (compressed pages: its scales)."""
        B, H = self.cfg.block_size, self.cfg.num_kv_heads
        if self.scheme == "dense":
            k, v, n = self.cell_bytes(s, t)
            bits = torch.tensor([value], dtype=self.dtype).view(torch.uint8).repeat(n // 2)
            if "k" in what:
                self.pool[k:k + n] = bits
            if "v" in what:
                self.pool[v:v + n] = bits
            return
        names = {"turbo_prod": ("k_scales_offset", "v_scales_offset"),
                 "turbo_mse": ("k_norms_offset", "v_norms_offset")}[self.scheme]
        bits = torch.tensor([value], dtype=FP16).view(torch.uint8).repeat(H)
        for c, nm in zip("kv", names):
            if c in what:
                at = (int(self.tables[s, t // B]) * int(self.layout.page_size_bytes)
                      + int(getattr(self.layout, nm)) + t % B * H * 2)
                self.pool[at:at + 2 * H] = bits

    def run(self, dev, stream=0, out=None):
        self.out = torch.full(self.query.shape, 5.0, dtype=self.dtype, device=dev) if out is None else out
        self.gpu = [x.to(dev) for x in (self.query, self.pool, self.tables, self.row_start, self.prefix,
                                        self.mask)]
        self.call(stream)
        torch.cuda.synchronize()
        return self.out.cpu().double()

    def call(self, stream=0):
        self.tq.tree_attn_output(self.scheme, *self.gpu, self.out, self.layout, self.cfg, self.max_kv,
                                 stream=stream)

    def expect(self):
        return tree_attention(self.scheme, self.query, self.pool, self.tables, self.row_start,
                              self.prefix, self.mask, self.layout, self.cfg, self.max_kv)

    def check(self, dev):
        got = self.run(dev)
        ref, tol, written = self.expect()
        bad = ~agrees(got, ref, tol, self.dtype)[written]
        d = (got - ref).abs()[written]
        worst = float((d / tol[written]).nan_to_num(posinf=0.0).max()) if d.numel() else 0.0
        print(f"    worst {worst:.2f} of the tolerance", flush=True)
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {worst:.2f}"
        assert (got[~written] == 5).all()
        return got


@pytest.fixture(params=[0, 300_000], ids=["", "room"], autouse=True)
def room(request, monkeypatch):
    """Tiles are chosen by max_kv_len: small trees run in the large ones too where it says that the
    cache may hold far more."""
    monkeypatch.setattr(Problem, "room", request.param)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("lens,widths,Hq,H,B", [
    ([0], [1], 2, 1, 16),                       # a token that sees itself alone
    ([1], [1], 16, 2, 16),
    ([1143], [5], 16, 2, 16),
    ([63, 64, 65], [1, 1, 1], 14, 2, 16),
    ([127, 0, 128, 15, 16, 17], [3, 4, 1, 2, 0, 8], 8, 4, 16),
    ([300, 5], [33, 70], 4, 2, 16),             # more than one mask word
    ([250], [64], 6, 1, 16),
    ([100, 333, 1], [7, 9, 2], 12, 4, 7),       # pages that end inside a tile
    ([40, 50], [3, 3], 3, 3, 1),
    ([500], [2], 32, 1, 64),
    ([700, 30], [17, 4], 7, 1, 32),
])
def test_against_float64(tq, cuda, scheme, dtype, lens, widths, Hq, H, B, D):
    print(f"[tree] {scheme} {dtype} {lens=} {widths=} {Hq=} {H=} {B=} {D=}", flush=True)
    Problem(tq, scheme, dtype, lens, widths, Hq, H, D, B, seed=len(lens) + D).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("D,lens,widths,Hq,H", [
    (128, [20000], [3], 16, 2),
    (64, [9001, 17, 4000], [1, 8, 2], 14, 2),
    (128, [6000, 1], [40, 1], 8, 1),
    (128, [3000] * 9, [4] * 9, 4, 4),
])
def test_long_prefixes(tq, cuda, scheme, dtype, D, lens, widths, Hq, H):
    """Sequences split over workgroups and merged."""
    print(f"[tree long] {scheme} {dtype} {lens=} {widths=} {D=}", flush=True)
    Problem(tq, scheme, dtype, lens, widths, Hq, H, D, seed=3).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("D,lens,widths", [(128, [33000], [3]), (128, [17000, 16000], [3, 4]),
                                           (64, [45000], [3]), (64, [34000], [7])])
def test_few_rows_of_many_pieces(tq, cuda, scheme, dtype, D, lens, widths):
    """Rows whose sums come from more than a hundred workgroups."""
    Problem(tq, scheme, dtype, lens, widths, 16, 2, D, seed=43).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_many_sequences(tq, cuda, scheme, dtype):
    """More sequences than a wave has lanes, empty ones among them, at both ends too."""
    lens = [(37 * s) % 101 for s in range(150)]
    widths = [0] + [s % 3 for s in range(148)] + [0]
    Problem(tq, scheme, dtype, lens, widths, 4, 2, 64, seed=4, extra_rows=3).check(cuda)


@pytest.mark.parametrize("seqs,H,longest", [(65, 3, 400), (700, 1, 300), (4300, 1, 40), (9000, 2, 9)])
def test_very_many_sequences(tq, cuda, seqs, H, longest):
    """From one sequence more than a wave has lanes to more than 64 blocks of 64, whole runs of them
    empty."""
    lens = [(37 * s + s * s // 7) % longest for s in range(seqs)]
    widths = [0 if s // 100 % 4 == 2 else (s * 5 // 3) % 3 for s in range(seqs)]
    Problem(tq, "dense", FP16, lens, widths, H * 2, H, 64, B=32, seed=4, extra_rows=2).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_rows_that_attend_nothing(tq, cuda, scheme, dtype):
    p = Problem(tq, scheme, dtype, [0, 0, 40], [3, 2, 2], 8, 2, 128, seed=5, extra_rows=5)
    p.mask[1] = 0
    p.mask[3:5] = 0
    got = p.check(cuda)
    assert (got[1] == 0).all() and (got[3:5] == 0).all()
    # and with nothing to read at all
    p.max_kv = 0
    assert (p.check(cuda)[:7] == 0).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_bits_past_the_drafted_tokens(tq, cuda, scheme, dtype):
    """Set bits of tokens that a sequence has not drafted, and drafted tokens without bits."""
    p = Problem(tq, scheme, dtype, [70, 10], [5, 3], 4, 2, 128, seed=6, words=3)
    p.mask[:] |= -(1 << 20)
    p.check(cuda)
    p = Problem(tq, scheme, dtype, [70, 100], [50, 40], 4, 2, 128, seed=6, words=1)
    p.check(cuda)


# Heads and widths for every number of rows per tile: 7, 18, 54, 72 and 288 rows a sequence.
TILES = [([6, 8], 2, 2), ([6, 30], 2, 2), ([6, 30], 6, 2), ([6, 30], 8, 2), ([6, 30], 32, 2)]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("widths,Hq,H", TILES)
@pytest.mark.parametrize("D", [64, 128])
def test_non_finite_values_that_a_row_does_not_see(tq, cuda, scheme, dtype, value, widths, Hq, H, D):
    """Behind the last token, in another branch of the tree, and on pages of other sequences."""
    p = Problem(tq, scheme, dtype, [90, 200], widths, Hq, H, D, seed=7)
    for s in (0, 1):
        n = p.lens[s] + p.widths[s]
        for t in range(n, -(-n // 16) * 16):
            p.fill_token(s, t, value)
        r = int(p.row_start[s])
        p.mask[r:r + p.widths[s], 0] &= ~(1 << 2)  # nobody sees drafted tokens 2
        p.fill_token(s, p.lens[s] + 2, value)
    p.check(cuda)
    # Drafted token 4 of the second sequence: rows that see it are not finite, the others right.
    r, w = int(p.row_start[1]), widths[1]
    sees = (p.mask[r:r + w, 0] >> 4 & 1).bool()
    sees[3], p.mask[r + 3, 0] = False, p.mask[r + 3, 0] & ~(1 << 4)
    clean, tol, _ = p.expect()
    p.fill_token(1, p.lens[1] + 4, value, "v")
    got = p.run(cuda)
    assert not torch.isfinite(got[r:r + w][sees]).any()
    rest = torch.ones(got.shape[0], dtype=torch.bool)
    rest[r:r + w] = ~sees
    assert ((got - clean).abs()[rest] <= tol[rest]).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("widths,Hq,H", TILES)
@pytest.mark.parametrize("L", [65, 97, 129, 230])
def test_non_finite_values_of_the_prefix(tq, cuda, scheme, dtype, widths, Hq, H, L):
    """In a chunk whose other half holds the drafted tokens or ends the sequence: every row of the
    sequence sees them, no other's does."""
    p = Problem(tq, scheme, dtype, [L, 50], widths, Hq, H, 128, seed=17)
    clean, tol, _ = p.expect()
    for t in (L - 60, L - 2):
        q = Problem(tq, scheme, dtype, [L, 50], widths, Hq, H, 128, seed=17)
        q.fill_token(0, t, float("inf"), "v")
        got = q.run(cuda)
        w = widths[0]
        if scheme == "dense":  # one token of +infinity, all others finite: the sum is +infinity
            assert (got[:w] == float("inf")).all()
        else:
            assert not torch.isfinite(got[:w]).any()
        assert ((got - clean).abs()[w:] <= tol[w:]).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_nan_key_reaches_its_rows_alone(tq, cuda, scheme, dtype):
    p = Problem(tq, scheme, dtype, [130], [20], 8, 2, 128, seed=8)
    sees = (p.mask[:, 0] >> 7 & 1).bool()
    clean, tol, _ = p.expect()
    p.fill_token(0, 137, float("nan"), "k")
    got = p.run(cuda)
    assert torch.isnan(got[sees]).all()
    assert ((got - clean).abs()[~sees] <= tol[~sees]).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_unmapped_pages_and_capped_lengths(tq, cuda, scheme, dtype):
    p = Problem(tq, scheme, dtype, [300, 90], [6, 3], 8, 2, 128, seed=9, extra_blocks=5)
    p.tables[0, 3] = -1
    p.tables[0, 7:9] = -5
    p.tables[1, 0] = -1
    p.check(cuda)
    p.max_kv = 200
    p.check(cuda)
    p.tables[1, :] = -1
    got = p.check(cuda)
    assert (got[6:9] == 0).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("q_scale,kv_scale", [(20.0, 1.0), (1.0, 30.0), (1e-3, 1e-2), (60.0, 1e3),
                                              (1.0, 1e4), (1e-2, 1e-4)])
def test_magnitudes(tq, cuda, scheme, dtype, q_scale, kv_scale):
    """From flat weights to a single one; pages' values near the ends of fp16."""
    p = Problem(tq, scheme, dtype, [1000, 3], [9, 4], 8, 2, 128, seed=10, q_scale=q_scale,
                kv_scale=kv_scale)
    p.check(cuda)


@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_value_scales_of_all_sizes(tq, cuda, scheme):
    """Cells whose V scales span fp16, zero included: the sum is the large ones', and rows that do
    not see those are as exact."""
    p = Problem(tq, scheme, FP16, [64, 30], [12, 12], 8, 2, 128, seed=11)
    for t in range(64):
        p.fill_token(0, t, 2.0 ** ((t % 31) - 20) if t % 7 else 0.0, "v")
    p.check(cuda)
    for t in range(30):
        p.fill_token(1, t, 1e-5, "v")
    p.fill_token(1, 30 + 5, 3e4, "v")
    p.check(cuda)
    p = Problem(tq, scheme, FP16, [200], [4], 8, 2, 128, seed=12)
    for t in range(204):
        p.fill_token(0, t, 0.0, "v")
    assert (p.check(cuda) == 0).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_results_repeat_and_do_not_depend_on_the_batch(tq, cuda, scheme, dtype):
    """The same bits again; and within tolerance when other sequences share the call."""
    p = Problem(tq, scheme, dtype, [5000, 40, 900], [6, 2, 20], 16, 2, 128, seed=13)
    a = p.check(cuda)
    assert torch.equal(a, p.run(cuda))


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_stream_and_graph(tq, cuda, scheme, dtype):
    """On a stream of its own; captured after one eager call, replayed over changed lengths and
    masks, with eager work in between."""
    p = Problem(tq, scheme, dtype, [4000, 300], [7, 12], 16, 2, 128, seed=14)
    want = p.run(cuda)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    p.out.fill_(5.0)
    st.wait_stream(torch.cuda.current_stream())
    p.call(st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(p.out.cpu().double(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        p.call(st.cuda_stream)
    for new in (4000, 17, 2500, 0):
        p.prefix[0] = new
        p.gpu[4].copy_(p.prefix)
        p.out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = p.out.cpu()
        p.out.fill_(5.0)
        p.call()
        torch.cuda.synchronize()
        assert torch.equal(got, p.out.cpu())
    tq.release_workspaces()


def test_offsets_past_32_bits(tq, cuda):
    """A page whose first byte is more than 4 GiB into the pool."""
    p = Problem(tq, "dense", FP16, [100], [3], 4, 2, 128, seed=15)
    page = int(p.layout.page_size_bytes)
    first = (1 << 32) // page + 3
    pool = torch.zeros((first + 8) * page, dtype=torch.uint8, device=cuda)
    pool[first * page:first * page + p.pool.numel()] = p.pool.to(cuda)[:8 * page]
    want = p.run(cuda)
    p.gpu[1] = pool
    p.gpu[2] = torch.where(p.gpu[2] >= 0, p.gpu[2] + first, p.gpu[2]).int()
    p.out.zero_()
    p.call()
    assert torch.equal(p.out.cpu().double(), want)


def test_host_threads_on_one_stream(tq, cuda):
    """Two trees and a slot-mapped attention from three threads on one stream, whose workspace they
    share: every call gives what it gives alone."""
    from concurrent.futures import ThreadPoolExecutor
    trees = [Problem(tq, "dense", FP16, [3000, 900], [5, 9], 16, 2, 128, seed=31),
             Problem(tq, "turbo_prod", FP16, [2500], [40], 16, 2, 128, seed=32)]
    for p in trees:
        p.run(cuda)
    p = trees[1]
    N = 2000
    slots = (p.tables[0, torch.arange(N) // 16] * 16 + torch.arange(N) % 16).int().to(cuda)
    query = torch.randn(8, 2, 128, generator=torch.Generator().manual_seed(33)).half().to(cuda)

    def tree(p, out):
        tq.tree_attn_output(p.scheme, *p.gpu, out, p.layout, p.cfg, p.max_kv)

    def slot_mapped(_, out):
        tq.fused_attn_output(query, p.gpu[1], slots, out, p.layout, p.cfg, 8, N)

    work = [(tree, trees[0], trees[0].out), (tree, trees[1], trees[1].out),
            (slot_mapped, None, torch.zeros_like(query))]
    slot_mapped(None, work[2][2])
    outs = [[torch.zeros_like(w[2]) for _ in range(80)] for w in work]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(3) as pool:
        for f in [pool.submit(lambda w, mine: [w[0](w[1], o) for o in mine], w, mine)
                  for w, mine in zip(work, outs)]:
            f.result()
    torch.cuda.synchronize()
    for w, mine in zip(work, outs):
        assert all(torch.equal(o, w[2]) for o in mine)


@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_chain_equals_the_paged_step(tq, cuda, scheme):
    """Trees without branches over a PagedBatch's pages: its own causal step's outputs, both within
    1e-3 of their row's largest value of the exact ones."""
    from turborag_amd.batched import PagedBatch
    b = PagedBatch(tq, scheme, [1500, 37, 300], [3, 8, 5], seed=560, device=cuda)
    b.append_new_tokens(seed=920)
    rows, row_seq, row_len = b.decode_rows(seed=921)
    tables = b.block_tables()
    want = torch.zeros_like(rows)
    b.attention(rows, row_seq, row_len, tables, want)
    # [8 GQA rows of a token, kv heads, D] -> [tokens, query heads, D]
    query = rows.view(16, 8, 2, 128).transpose(1, 2).reshape(16, 16, 128).contiguous()
    mask = torch.cat([tree_mask_from_parents(range(-1, w - 1)) for w in b.widths]).to(cuda)
    out = torch.zeros_like(query)
    b.tree_attention(query, *b.tree_rows(), mask, tables, out)
    got = out.view(16, 2, 8, 128).transpose(1, 2).reshape(rows.shape).double()
    want = want.double()
    err = ((got - want).abs().amax(-1) / want.abs().amax(-1)).max()
    assert float(err) < 2e-3
    b.close()


def test_one_step_of_the_three(tq, cuda):
    """Norm, rotation and append of a tree's tokens, then their attention, as a step runs them; and
    the same over turbo_prod pages by rotation and pack."""
    from oracle.step_oracle import norm_rope
    from turborag_amd.turboquant_wrapper import rope_table
    H, Hq, D, L = 2, 16, 128, 500
    parents = [-1, 0, 0, 1, 1, 4]
    n = len(parents)
    g = torch.Generator().manual_seed(16)
    qkv = torch.randn(L + n, Hq + 2 * H, D, generator=g).half()
    w = [(1 + 0.1 * torch.randn(D, generator=g)).half() for _ in range(2)]
    depth = [0] * n
    for j, up in enumerate(parents):
        depth[j] = 0 if up < 0 else depth[up] + 1
    pos = torch.cat([torch.arange(L), L + torch.tensor(depth)]).int()
    table = rope_table(1024, D)
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim = H, D
    mask = tree_mask_from_parents(parents)
    blocks = torch.randperm(40, generator=g)[:(L + n + 15) // 16].int()
    t = torch.arange(L + n)
    slots = (blocks[t // 16] * 16 + t % 16).int()
    dev = [x.to(cuda) for x in (qkv, pos, slots, table, *w)]
    q, k, v = dev[0][:, :Hq], dev[0][:, Hq:Hq + H], dev[0][:, Hq + H:]
    for scheme in ("dense", "turbo_prod"):
        layout = (tq.make_dense_layout_for if scheme == "dense" else tq.make_layout_for)(cfg)
        pool = tq.alloc_page_pool(40 * 16, layout, cfg)
        oq = torch.empty(L + n, Hq, D, dtype=FP16, device=cuda)
        if scheme == "dense":  # the prefill, then the step's tokens
            for part in (slice(0, L), slice(L, L + n)):
                tq.dense_rope_append(q[part], k[part], v[part], dev[1][part], dev[2][part], dev[3],
                                     oq[part], pool, layout, cfg, *dev[4:])
        else:
            ok = torch.empty(L + n, H, D, dtype=FP16, device=cuda)
            tq.qk_norm_rope(q, k, dev[1], dev[3], oq, ok, cfg, *dev[4:])
            tq.pack(ok, v.contiguous(), dev[2], pool, layout, cfg)
        out = torch.empty(n, Hq, D, dtype=FP16, device=cuda)
        start, prefix = (torch.tensor(x, dtype=torch.int32) for x in ([0, n], [L]))
        tq.tree_attn_output(scheme, oq[L:].contiguous(), pool, blocks[None].to(cuda), start.to(cuda),
                            prefix.to(cuda), mask.to(cuda), out, layout, cfg, L + n)
        want_q, tol_q = norm_rope(qkv[:, :Hq], w[0], pos, table, False, 1e-6)
        assert ((oq.cpu().double() - want_q).abs() <= tol_q).all()
        ref, tol, _ = tree_attention(scheme, oq[L:].cpu(), pool.cpu(), blocks[None], start, prefix, mask,
                                     layout, cfg, L + n)
        assert ((out.cpu().double() - ref).abs() <= tol).all()
