"""Attention weights per cached token (attn_weights) against float64, with
tolerances that count roundings (oracle/evict_oracle.py)."""
from __future__ import annotations

import pytest
import torch

from oracle.evict_oracle import attention_weights
from oracle.step_oracle import hadamard, signs
from test_gpu_tree import SCHEMES, Problem

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


class Weights:
    """A tree test's problem (sequences of cached tokens and query rows), and scores."""

    def __init__(self, tq, scheme, dtype, lens, widths, Hq, H, D, B=16, seed=0, causal=True, decay=1.0,
                 before=True, room=0, **kw):
        self.p = p = Problem(tq, scheme, dtype, lens, widths, Hq, H, D, B=B, seed=seed, **kw)
        self.causal, self.decay = causal, decay
        g = torch.Generator().manual_seed(seed + 1)
        self.T = p.tables.shape[1] * B if room is None else p.max_kv + room
        S = len(lens)
        self.scores = torch.full((S, H, self.T), 9.0)
        self.before = torch.rand(S, H, self.T, generator=g) * 3 if before else None
        self.max_kv = p.max_kv

    def upload(self, dev):
        p = self.p
        self.gpu = [x.to(dev) for x in (p.query, p.pool, p.tables, p.row_start, p.prefix)]
        self.out = self.scores.to(dev)
        self.inn = None if self.before is None else self.before.to(dev)

    def call(self, stream=0):
        p = self.p
        p.tq.attn_weights(p.scheme, *self.gpu, self.out, p.layout, p.cfg, self.max_kv, causal=self.causal,
                          scores_in=self.inn, decay=self.decay, stream=stream)

    def expect(self):
        p = self.p
        return attention_weights(p.scheme, p.query, p.pool, p.tables, p.row_start, p.prefix, p.layout, p.cfg,
                                 self.max_kv, self.causal, self.scores, self.before, self.decay)

    def compare(self, got, want=None):
        ref, tol = want or self.expect()
        d = (got.cpu().double() - ref).abs()
        worst = float((d / tol.clamp(min=1e-300)).nan_to_num(0.0).max())
        print(f"    worst {worst:.3f} of the tolerance", flush=True)
        assert (d <= tol).all(), f"worst {worst:.2f} of the tolerance, {int((d > tol).sum())} off"

    def check(self, dev):
        self.upload(dev)
        self.call()
        torch.cuda.synchronize()
        self.compare(self.out)
        return self.out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("lens,widths,Hq,H,B", [
    ([0], [1], 2, 1, 16),                       # a token that sees itself alone
    ([1], [1], 16, 2, 16),
    ([1143], [1], 16, 2, 16),                   # a decode step
    ([127, 0, 128, 15, 16, 17], [3, 4, 1, 2, 0, 8], 8, 4, 16),
    ([300, 5], [33, 70], 4, 2, 16),             # rows of more than one tile and block
    ([255, 256, 257], [5, 9, 2], 12, 2, 16),    # chunks that just end or begin
    ([900], [64], 16, 2, 16),                   # 512 rows: K is gone over twice
    ([2300], [33], 10, 1, 16),
    ([63, 200], [4, 5], 6, 3, 7),               # pages of other sizes
    ([40] * 70 + [0, 500], [3] * 71 + [0], 16, 1, 16),  # more than 64 sequences, 45 rows each
])
def test_shapes(tq, cuda, lens, widths, Hq, H, B, scheme, dtype, D):
    Weights(tq, scheme, dtype, lens, widths, Hq, H, D, B=B, seed=len(lens) + D).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("width", [2, 20])
def test_prefix_only(tq, cuda, scheme, dtype, width):
    """causal=False: every row attends the prefix and nothing behind it; a sequence without prefix
    has no token to score."""
    w = Weights(tq, scheme, dtype, [300, 0, 1, 77], [width] * 4, 8, 2, 128, causal=False, seed=5, decay=0.25)
    w.check(cuda)
    assert (w.out[1] == 9).all()


@pytest.mark.parametrize("width", [1, 9])
def test_no_scores_before(tq, cuda, width):
    w = Weights(tq, "dense", FP16, [500, 30], [width] * 2, 16, 2, 128, before=False, seed=6)
    w.check(cuda)
    w = Weights(tq, "dense", FP16, [500, 30], [width] * 2, 16, 2, 128, decay=0.0, seed=6)
    w.before[:] = float("nan")  # not read
    w.upload(cuda)
    w.call()
    torch.cuda.synchronize()
    w.before = None
    w.compare(w.out)


@pytest.mark.parametrize("width", [1, 9])
def test_adds_up_in_place(tq, cuda, width):
    """scores_in is scores: three steps add up, the last weighting the others."""
    w = Weights(tq, "turbo_mse", FP16, [400, 260], [width] * 2, 16, 2, 64, before=False, seed=7)
    w.scores = torch.rand(w.scores.shape)
    w.upload(cuda)
    for decay in (1.0, 0.5, 1.0):
        w.before, w.inn, w.decay = w.scores, w.out, decay
        ref, tol = w.expect()
        w.call()
        torch.cuda.synchronize()
        w.compare(w.out, (ref, tol))
        w.scores = w.out.cpu()


@pytest.mark.parametrize("width", [1, 9])
def test_sequences_without_rows(tq, cuda, width):
    """They get decay * scores_in up to their prefix; with no row in the call at all, too."""
    w = Weights(tq, "dense", BF16, [100, 300, 40], [0, width, 0], 8, 1, 128, decay=0.5, seed=8)
    out = w.check(cuda)
    assert torch.equal(out[0, 0, :100].cpu(), 0.5 * w.before[0, 0, :100])
    w = Weights(tq, "dense", BF16, [100, 300], [0, 0], 8, 1, 128, decay=0.5, seed=8)
    out = w.check(cuda)
    assert torch.equal(out[1, 0, :300].cpu(), 0.5 * w.before[1, 0, :300])


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("width", [2, 20])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_masked_values_do_not_reach(tq, cuda, scheme, dtype, width, value):
    """Keys behind a row's last token, past max_kv_len and in unmapped pages may hold anything."""
    w = Weights(tq, scheme, dtype, [300, 100], [width] * 2, 16, 2, 128, seed=9)
    p = w.p
    p.tables[0, 3] = -1
    w.max_kv = 300 + width // 2
    want = w.expect()
    for t in range(w.max_kv, 300 + width):
        p.fill_token(0, t, value)
    w.upload(cuda)
    w.call()
    torch.cuda.synchronize()
    w.compare(w.out, want)
    assert torch.equal(w.out[0, :, 48:64].cpu(), w.before[0, :, 48:64])  # the unmapped page's tokens
    assert (w.out[0, :, w.max_kv:] == 9).all()
    # a row's own future: the last token's keys reach the last row alone
    w = Weights(tq, scheme, dtype, [50], [width], 2, 1, 64, seed=10, before=False)
    want = w.expect()
    w.p.fill_token(0, 50 + width - 1, value)
    w.p.query[-1] = 0
    w.upload(cuda)
    w.call()
    torch.cuda.synchronize()
    assert torch.isnan(w.out[0, 0, :50 + width]).all()  # 0 * inf, NaN: that row's weights


@pytest.mark.parametrize("width", [1, 9])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 60.0, 3e3])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_logit_sizes(tq, cuda, scheme, dtype, width, scale):
    """Flat rows, rows of one token, and logits far beyond where their exponentials overflow."""
    Weights(tq, scheme, dtype, [700, 90], [width] * 2, 16, 2, 128, seed=11, q_scale=scale).check(cuda)


@pytest.mark.parametrize("scheme,dtype,q,k", [("dense", FP16, 6e4, 6e4), ("dense", BF16, 1e15, 1e15),
                                              ("turbo_prod", FP16, 6e4, 3e4), ("turbo_mse", FP16, 6e4, 3e4)])
@pytest.mark.parametrize("width", [1, 4, 9])
def test_huge_logits(tq, cuda, scheme, dtype, q, k, width):
    """Logits of 1e10 (bf16 1e31): two equal largest ones share a row's weight, and the others, many
    orders of magnitude below, get nothing (turbo_prod's two differ by their residuals: one takes it
    all).  Only exact operations are left: equal logits are the same sums, their difference from the
    maximum 0, the weights 1/2 or 1."""
    w = Weights(tq, scheme, dtype, [300], [width], 16, 2, 128, seed=23, causal=False, before=False)
    p = w.p
    p.query[:] = q
    if scheme == "dense":
        for t in range(300):
            p.fill_token(0, t, 1.0, "k")
        for t in (17, 290):
            p.fill_token(0, t, k, "k")
    else:
        # every token's codes are token 17's, whose product with the rotated query is positive
        for t in range(300):
            p.fill_token(0, t, 1e-3, "k")
        page, H, B, D = int(p.layout.page_size_bytes), 2, 16, 128
        off = int(p.layout.k4_codes_offset if scheme == "turbo_prod" else p.layout.k_codes_offset)
        for t in range(300):
            at = int(p.tables[0, t // B]) * page + off + t % B * H * D // 2
            p.pool[at:at + H * D // 2] = 0x88 if scheme == "turbo_mse" else 0x44
        had = hadamard(D)
        for h in range(H):
            turned = (torch.full((D,), float(q), dtype=torch.float64) * signs(h, D)) @ had
            top = int(turned.abs().argmax())
            # (the rotation of a constant row is one dim: its code is the level of the same sign)
            code = 15 if turned[top] > 0 else 0
            for t in range(300):
                at = int(p.tables[0, t // B]) * page + off + (t % B * H + h) * D // 2 + top // 2
                old = int(p.pool[at])
                p.pool[at] = (old & 0xF0) | code if top % 2 == 0 else (old & 0x0F) | code << 4
        for t in (17, 290):
            p.fill_token(0, t, k, "k")
    w.upload(cuda)
    w.call()
    torch.cuda.synchronize()
    got = w.out.cpu()[0, :, :300]
    want = w.expect()[0][0, :, :300].float()
    total = 8.0 * width
    if scheme == "turbo_prod":
        assert ((want[:, 17] == total) | (want[:, 290] == total)).all()
    else:
        assert (want[:, 17] == total / 2).all() and (want[:, 290] == total / 2).all()
    assert torch.equal(got, want)


@pytest.mark.parametrize("width", [1, 9])
def test_equal_logits(tq, cuda, width):
    """A zero query: every token that a row sees gets the same weight."""
    w = Weights(tq, "dense", FP16, [1000], [width], 8, 1, 128, seed=12, before=False)
    w.p.query.zero_()
    out = w.check(cuda)
    assert (out[0, 0, :1000] == out[0, 0, 0]).all()


def test_rows_sum_to_one(tq, cuda):
    """The weights of all tokens add up to the rows (40 of a kv head here, and 8)."""
    for width in (1, 5):
        w = Weights(tq, "turbo_prod", FP16, [3000, 100], [width] * 2, 16, 2, 128, seed=13, before=False)
        out = w.check(cuda)
        for s, n in enumerate((3000, 100)):
            total = out[s, :, :n + width].double().sum(1)
            # (each weight within 1e-5 of itself at logits of this size)
            assert ((total - 8 * width).abs() < 1e-5 * 8 * width).all()


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_long(tq, cuda, scheme, dtype):
    """Over 40,000 tokens: more chunks than a line of the merge, several workgroups of sums."""
    for width in (1, 6):
        Weights(tq, scheme, dtype, [40001], [width], 8, 1, 64, seed=14, before=False).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 8, 9])
def test_rows_per_sequence(tq, cuda, scheme, dtype, width):
    """8 to 72 rows of a kv head: the row counts at which another way is taken (16, 32, 64)."""
    Weights(tq, scheme, dtype, [600, 257], [width] * 2, 16, 2, 128, seed=19 + width).check(cuda)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("lens,widths,Hq,H", [
    ([600], [17], 16, 2),            # 136 rows: several blocks of a chunk, the last a part
    ([300, 1], [40, 40], 8, 1),      # 320 rows: more than a group of statistics
    ([40, 0, 500], [1, 90, 33], 8, 1),
    ([2000], [70], 8, 1),            # 560 rows: too much to store for dense pages
    ([17000], [10], 8, 1),           # 80 rows of a long sequence: read again, blocks shared
])
def test_many_rows(tq, cuda, scheme, dtype, lens, widths, Hq, H, D):
    """More than 64 rows of a kv head in few chunks: workgroups share a chunk's rows."""
    Weights(tq, scheme, dtype, lens, widths, Hq, H, D, seed=30 + sum(widths) % 7).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("D", [64, 128])
def test_uneven_rows(tq, cuda, scheme, dtype, D):
    """One sequence has far more rows than the average, which chooses the way; others have none."""
    widths = [1] * 30 + [40] + [0] * 29
    Weights(tq, scheme, dtype, [70] * 30 + [500] + [70] * 29, widths, 8, 1, D, seed=20).check(cuda)
    Weights(tq, scheme, dtype, [70] * 3 + [500], [1, 60, 0, 90], 8, 1, D, seed=21).check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
def test_many_sequences_on_large_workgroups(tq, cuda, scheme, dtype):
    """Workgroups enough for large ones in the sum over stored rows."""
    Weights(tq, scheme, dtype, [1500] + [20] * 70, [1] * 71, 16, 8, 64, seed=22, before=True).check(cuda)


def test_capacity_far_above_the_lengths(tq, cuda):
    for width in (1, 6):
        w = Weights(tq, "dense", FP16, [1000, 20], [width] * 2, 16, 2, 128, seed=15, extra_blocks=3000)
        w.max_kv = 40000
        w.scores = torch.full((2, 2, 40000), 9.0)
        w.before = torch.rand(2, 2, 40000)
        w.check(cuda)


def test_offsets_past_32_bits(tq, cuda):
    """Pages more than 4 GB into the pool."""
    H, D, B = 2, 128, 16
    w = Weights(tq, "dense", FP16, [400], [2], 16, H, D, seed=16)
    p = w.p
    page = int(p.layout.page_size_bytes)
    pages = p.pool.numel() // page
    far = (5 << 30) // page
    want = w.expect()
    w.upload(cuda)
    pool = torch.zeros((far + pages) * page, dtype=torch.uint8, device=cuda)
    pool[far * page:] = p.pool.to(cuda)
    w.gpu[1] = pool
    w.gpu[2] = torch.where(p.tables >= 0, p.tables + far, -1).to(cuda)
    w.call()
    torch.cuda.synchronize()
    w.compare(w.out, want)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("width", [1, 9])
def test_stream_and_graph(tq, cuda, scheme, dtype, width):
    """Captured on a stream after an eager call; every replay, with eager calls of other sizes
    between, has the eager result bit for bit, and lengths are read at every replay."""
    w = Weights(tq, scheme, dtype, [700, 300], [width] * 2, 16, 2, 128, seed=17)
    small = Weights(tq, scheme, dtype, [90], [2], 16, 2, 128, seed=18)
    w.upload(cuda)
    small.upload(cuda)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    w.call(st.cuda_stream)
    torch.cuda.synchronize()
    eager = w.out.clone()
    w.compare(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        w.call(st.cuda_stream)
    for _ in range(3):
        w.out.copy_(w.scores)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.out, eager)
        small.call(st.cuda_stream)
        torch.cuda.synchronize()
        small.compare(small.out)
    w.p.prefix = torch.tensor([650, 288], dtype=torch.int32)
    w.gpu[4].copy_(w.p.prefix)
    w.out.copy_(w.scores)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    w.compare(w.out)


def test_two_streams_at_once(tq, cuda):
    """Calls of different sizes on two streams, several in flight: each has its stream's workspace."""
    a = Weights(tq, "turbo_prod", FP16, [900, 300], [9, 1], 16, 2, 128, seed=50, before=False)
    b = Weights(tq, "dense", BF16, [2000], [12], 8, 2, 64, seed=51, before=False)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for w in (a, b):
        w.upload(cuda)
    torch.cuda.synchronize()
    for _ in range(8):
        for w, st in zip((a, b), streams):
            w.call(st.cuda_stream)
    torch.cuda.synchronize()
    for w in (a, b):
        w.compare(w.out)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("lens,widths", [([300, 90], [2, 1]), ([500], [20]), ([400, 17000], [12, 10])])
def test_padded_batch(tq, cuda, scheme, dtype, lens, widths):
    """Rows behind the last sequence's, as a padded batch has them, hold anything and reach nothing;
    the same pages under two sequences are scored for each."""
    w = Weights(tq, scheme, dtype, lens, widths, 16, 2, 128, seed=60)
    p = w.p
    if len(lens) == 2 and lens[1] < lens[0]:
        p.tables[1] = p.tables[0]
    p.query = torch.cat([p.query, torch.full((37, 16, 128), float("nan"), dtype=dtype)])
    w.check(cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("S,L,width", [(130, 1300, 1), (130, 700, 3), (70, 5000, 1), (130, 4000, 1)])
def test_many_sequences(tq, cuda, scheme, dtype, S, L, width):
    """Sequences enough for the sum's middle and largest workgroups, of uneven lengths."""
    lens = [(L * (k + 1)) // S for k in range(S)]
    lens[3] = 0
    Weights(tq, scheme, dtype, lens, [width] * S, 4, 2, 64, seed=90).check(cuda)
