"""Tree attention where logits are large (up to fp32's range): a row's weights
are then those of its largest logit alone, or of several that are equal, and its
output a mean of their values, whatever the logits' size.

Checked for every row: the output is finite and lies between the smallest and
the largest of the values that the row attends (per dimension, in the rotated
domain of compressed pages).  Checked where float64 decides it: the values of
the largest logit, if it is further above the others than the logits' rounding."""
from __future__ import annotations

import math

import pytest
import torch

from oracle.step_oracle import U32, cell_rows, hadamard, signs, tiny, unit
from test_gpu_tree import Problem

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
# widths, query and kv heads, tokens that the cache may hold beyond: tiles of 16, 32, 64, 128, 256 rows.
TILES = [(4, 2, 1, 0), (8, 12, 2, 300_000), (12, 16, 2, 300_000), (20, 16, 2, 300_000), (30, 32, 2, 300_000)]


def value_scales(p, lo, hi, seed=1):
    """Compressed pages: V's scales log-uniform in 2^lo .. 2^hi, one in nine of them 0."""
    g = torch.Generator().manual_seed(seed)
    page, cells = int(p.layout.page_size_bytes), p.cfg.block_size * p.cfg.num_kv_heads
    at = int(p.layout.v_scales_offset if p.scheme == "turbo_prod" else p.layout.v_norms_offset)
    v = p.pool.view(-1, page)
    sc = torch.exp2(lo + (hi - lo) * torch.rand(v.shape[0], cells, generator=g)).half()
    sc[torch.rand(sc.shape, generator=g) < 1 / 9] = 0
    v[:, at:at + 2 * cells] = sc.view(torch.uint8)


def dense_values(p, scale, seed=2):
    """Dense pages: V of its own size, N(0, scale^2)."""
    g = torch.Generator().manual_seed(seed)
    at, n = int(p.layout.v_offset), int(p.layout.v_bytes)
    v = p.pool.view(-1, int(p.layout.page_size_bytes))
    v[:, at:at + n] = (torch.randn(v.shape[0], n // 2, generator=g) * scale).to(p.dtype).view(torch.uint8)


def check(p, dev, least=0.5):
    got = p.run(dev)
    H, D = p.cfg.num_kv_heads, p.cfg.head_dim
    G = p.query.shape[1] // H
    turned, had = p.scheme != "dense", hadamard(D)
    assert torch.isfinite(got).all(), f"{int((~torch.isfinite(got)).sum())} values not finite"
    # Roundings of a mean of values v with weights that add up to 1: a weight's to 16 bits, the
    # output's; compressed pages: the codebook's 2^-13 and the rotation's log2(D) + 2.  64 U32: the sums.
    rel = unit(p.dtype) + 64 * U32 + (2.0 ** -13 + (math.log2(D) + 2) * U32 if turned else 0.0)
    decided = total = 0
    for s, w in enumerate(p.widths):
        r0, L = int(p.row_start[s]), p.lens[s]
        if not w:
            continue
        t = torch.arange(L + w)
        k, v = cell_rows(p.scheme, p.dtype, p.pool, p.layout, p.cfg, p.tables[s], t)
        words = p.mask[r0:r0 + w].long()
        j = (t - L).clamp(min=0)
        see = (t < L)[None] | ((words[:, j >> 5] >> (j & 31)[None]) & 1).bool()
        see = see.repeat_interleave(G, 0)
        for h in range(H):
            q = p.query[r0:r0 + w, h * G:(h + 1) * G].double().reshape(-1, D)
            o = got[r0:r0 + w, h * G:(h + 1) * G].reshape(-1, D)
            out_err = unit(p.dtype) * o.abs() + tiny(p.dtype)
            if turned:
                q, o = (q * signs(h, D)) @ had, (o * signs(h, D)) @ had
                out_err = out_err.sum(1, keepdim=True) / math.sqrt(D)
            x = (q @ k[:, h].T) / math.sqrt(D)
            # a logit's rounding: as in step_oracle.tree_attention, twice for a difference
            err = (q.abs() @ k[:, h].abs().T) / math.sqrt(D) * 2 * (
                (D + 8) * U32 + (2.0 ** -21 + (math.log2(D) + 2) * U32 if turned else 0.0))
            x, err = x.masked_fill(~see, -math.inf), err.masked_fill(~see, 0.0)
            vv = v[:, h]
            size = vv.abs().max()
            lo = torch.where(see[:, :, None], vv, math.inf).min(1).values
            hi = torch.where(see[:, :, None], vv, -math.inf).max(1).values
            tol = out_err + rel * size
            assert (o >= lo - tol).all() and (o <= hi + tol).all(), (s, h)
            top, at = x.max(1)
            gap = top[:, None] - x - err.max(1, keepdim=True).values
            gap.scatter_(1, at[:, None], math.inf)
            # the others' weights together: below 2^-30 of the largest
            sure = gap.min(1).values > 21 + math.log(len(t))
            one = vv[at]
            # (a value's own size here, and what is left of the others)
            tol = out_err + rel * (one.abs().sum(1, keepdim=True) / math.sqrt(D) if turned else one.abs()) \
                + 2.0 ** -30 * size + (2.0 ** -25 * 2.7 * math.sqrt(D) if turned else 0.0)
            if turned:  # an error of the rotated values, all of one row's together
                tol = tol * math.sqrt(D)
            assert ((o - one).abs() <= tol)[sure].all(), (s, h)
            decided += int(sure.sum())
            total += len(sure)
    print(f"    {decided} of {total} rows decided", flush=True)
    assert decided >= least * total


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,q_scale,kv_scale", [
    (FP16, 3e3, 3e3), (FP16, 5e3, 5e3), (FP16, 1e4, 1e4), (FP16, 1.2e4, 1e3),
    (BF16, 1e4, 1e4), (BF16, 1e5, 1e5), (BF16, 1e6, 1e6), (BF16, 1e9, 1e8), (BF16, 1e15, 1e15)])
@pytest.mark.parametrize("widths,Hq,H,room", TILES)
def test_dense(tq, cuda, monkeypatch, widths, Hq, H, room, dtype, q_scale, kv_scale, D):
    monkeypatch.setattr(Problem, "room", room)
    print(f"[large logits] {dtype} {q_scale} {kv_scale} {widths=} {Hq=} {D=}", flush=True)
    p = Problem(tq, "dense", dtype, [70, 300, 0], [widths, max(widths - 2, 1), 1], Hq, H, D, seed=61,
                q_scale=q_scale, kv_scale=kv_scale)
    dense_values(p, 1.0)
    check(p, cuda)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
@pytest.mark.parametrize("q_scale,kv_scale", [(1e3, 1e3), (5e3, 5e3), (1e4, 1.5e4)])
# (rotated back, values of scale 2^12 are N(0, 2^24) over the dimensions: below 65,504 to 16 sigma)
@pytest.mark.parametrize("scales", [(-1, 1), (-20, 12)])
@pytest.mark.parametrize("widths,Hq,H,room", TILES)
def test_compressed(tq, cuda, monkeypatch, scheme, widths, Hq, H, room, q_scale, kv_scale, scales, D):
    monkeypatch.setattr(Problem, "room", room)
    print(f"[large logits] {scheme} {q_scale} {kv_scale} {scales} {widths=} {Hq=} {D=}", flush=True)
    p = Problem(tq, scheme, FP16, [70, 300, 0], [widths, max(widths - 2, 1), 1], Hq, H, D, seed=62,
                q_scale=q_scale, kv_scale=kv_scale)
    value_scales(p, *scales)
    check(p, cuda)


@pytest.mark.parametrize("dtype,a,b", [(FP16, 8.0, 8.0), (FP16, 512.0, 512.0), (FP16, 4096.0, 4096.0),
                                       (BF16, 2.0 ** 20, 2.0 ** 17), (BF16, 2.0 ** 50, 2.0 ** 40)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("widths,Hq,H,room", TILES)
def test_equal_logits_share(tq, cuda, monkeypatch, widths, Hq, H, room, dtype, a, b, sign):
    """Logits that fp32 holds exactly, several of them equal: the mean of their values.  With
    sign -1 all logits are negative."""
    monkeypatch.setattr(Problem, "room", room)
    D = 128
    g = torch.Generator().manual_seed(63)
    lens = [200, 77]
    p = Problem(tq, "dense", dtype, lens, [widths, 1], Hq, H, D, seed=63)
    dense_values(p, 1.0)
    # q: a single dimension of size a; k: there b times 1 .. 6 (or their negatives), random elsewhere
    dim = torch.randint(0, D, (p.query.shape[0], Hq), generator=g)
    p.query.zero_()
    p.query.scatter_(2, dim[..., None], a)
    at, n = int(p.layout.k_offset), int(p.layout.k_bytes)
    v = p.pool.view(-1, int(p.layout.page_size_bytes))
    v[:, at:at + n] = (torch.randint(1, 7, (v.shape[0], n // 2), generator=g) * (sign * b)).to(
        dtype).view(torch.uint8)
    got = p.run(cuda)
    G = Hq // H
    for s, w in enumerate(p.widths):
        r0, L = int(p.row_start[s]), lens[s]
        t = torch.arange(L + w)
        k, v = cell_rows("dense", dtype, p.pool, p.layout, p.cfg, p.tables[s], t)
        for j in range(w):
            see = (t < L) | ((int(p.mask[r0 + j, 0]) >> (t - L).clamp(min=0)) & 1).bool()
            for i in range(Hq):
                x = k[:, i // G, dim[r0 + j, i]].masked_fill(~see, -math.inf) * a / math.sqrt(D)
                # (differences of a b / sqrt(D): 5.6 and more, or nothing)
                pr = torch.softmax(x, 0)
                ref = pr @ v[:, i // G]
                size = pr @ v[:, i // G].abs()
                # logits are exact; the exponent's rounding at 2^-24 of an argument below 2^24 of
                # weights that count is below 2^-18
                tol = size * (unit(dtype) + 2.0 ** -18 + 64 * U32) + unit(dtype) * ref.abs() + tiny(dtype)
                assert ((got[r0 + j, i] - ref).abs() <= tol).all(), (s, j, i)


@pytest.mark.parametrize("scheme,dtype", [("dense", FP16), ("dense", BF16), ("turbo_prod", FP16),
                                          ("turbo_mse", FP16)])
@pytest.mark.parametrize("widths,Hq,H,room", TILES)
def test_rows_of_all_sizes(tq, cuda, monkeypatch, widths, Hq, H, room, scheme, dtype):
    """Rows of one tile with logits from 1e-3 to 1e8: each as exact as it is among its like."""
    monkeypatch.setattr(Problem, "room", room)
    p = Problem(tq, scheme, dtype, [1070, 300, 0], [widths, max(widths - 2, 1), 1], Hq, H, 128, seed=64,
                kv_scale=2e3)
    g = torch.Generator().manual_seed(65)
    size = 10.0 ** (-6 + 10 * torch.rand(*p.query.shape[:2], 1, generator=g))
    p.query = (p.query.float() * size).to(dtype)
    if scheme == "dense":
        dense_values(p, 1.0)
    else:
        value_scales(p, -3, 3)
    check(p, cuda, least=0.0)
    p.check(cuda)
