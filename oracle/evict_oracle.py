"""float64 restatement of positions with several axes and of the eviction
operators (attention weights per cached token, selection, compaction), on the
CPU, with the error that the weights' roundings may leave."""
from __future__ import annotations

import math

import torch

from oracle.step_oracle import U32, cell_rows, hadamard, signs, tiny, unit


def norm_rope_axes(x, weight, pos, table, axis, interleaved, eps):
    """(y, tolerance) of x [N, heads, D], pos [axes, N], pair i by axis[i]: as
    step_oracle.norm_rope, whose count of roundings this has."""
    y = x.double()
    D = y.shape[-1]
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    half = table.shape[1] // 2
    out, size = y.clone(), y.abs()
    for i in range(half):
        p = pos[axis[i]].long()
        c, s = table[p, i].double()[:, None], table[p, half + i].double()[:, None]
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = y[..., ia], y[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
        size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return out, unit(x.dtype) * out.abs() + 32 * U32 * size + tiny(x.dtype)


def attention_weights(scheme, query, pool, tables, row_start, prefix, layout, cfg, max_kv, causal, scores,
                      scores_in=None, decay=1.0):
    """(scores, tolerance) float64 [S, H, tokens].

    A logit (in natural units) is a sum of D products in fp32, its scale and the
    difference from the row's maximum: D + 12 roundings of at most sum |q k| /
    sqrt(D).  Compressed pages: q and k in two fp16 parts, 2^-22 of each product
    three times (k's, q's and the parts' left-out product) < 2^-20, and a rotated q
    off by log2(D) + 2 roundings of |q|_1 / sqrt(D).  A weight moves by its own
    logit's error and by the largest of its row's (through the sum); its
    exponential, the row's sum (the tokens' chunks in 16 lines) and the reciprocal
    add 64 + chunks / 16 of U32, and the sum over the rows as many as it has terms
    in a line (32, or an eighth of them) and 8; then the scores read and added: 3."""
    H, D = cfg.num_kv_heads, cfg.head_dim
    Hq = query.shape[1]
    G = Hq // H
    out, tol = scores.double().clone(), torch.zeros(scores.shape, dtype=torch.float64)
    turned = scheme != "dense"
    had = hadamard(D)
    for s in range(prefix.numel()):
        r0, r1, L = int(row_start[s]), int(row_start[s + 1]), max(int(prefix[s]), 0)
        n = max(r1 - r0, 0)
        end = min(L + (n if causal else 0), max_kv)
        if not end:
            continue
        t = torch.arange(end)
        mapped = tables[s][t // cfg.block_size] >= 0
        k = torch.zeros(end, H, D, dtype=torch.float64)
        if n:
            k[mapped] = cell_rows(scheme, query.dtype, pool, layout, cfg, tables[s], t[mapped])[0]
        ka = k.abs()
        if scheme == "turbo_prod" and n and mapped.any():  # level and residual are separate products
            res = residuals(pool, layout, cfg, tables[s], t[mapped])
            ka[mapped] += 2 * res
        limit = torch.full((n,), min(L, max_kv)) if not causal else \
            (L + 1 + torch.arange(n)).clamp(max=max_kv)
        see = ((t[None] < limit[:, None]) & mapped[None]).repeat_interleave(G, 0)
        for h in range(H):
            got, err = torch.zeros(end, dtype=torch.float64), torch.zeros(end, dtype=torch.float64)
            if n:
                q = query[r0:r1, h * G:(h + 1) * G].double().reshape(-1, D)
                one = q.abs().sum(1, keepdim=True) / math.sqrt(D)
                if turned:
                    q = (q * signs(h, D)) @ had
                x = (q @ torch.where(mapped[:, None], k[:, h], 0.0).T) / math.sqrt(D)
                size = (q.abs() @ ka[:, h].T) / math.sqrt(D)
                dx = (D + 12) * U32 * size
                if turned:
                    dx = dx + 2.0 ** -20 * size + (math.log2(D) + 2) * U32 * one * ka[:, h].sum(1) / math.sqrt(D)
                x = x.masked_fill(~see, -math.inf)
                dx = dx.masked_fill(~see, 0.0)
                top = x.max(1, keepdim=True).values
                dead = top == -math.inf
                w = torch.exp(x - torch.where(dead, 0.0, top))
                w = torch.where(dead, 0.0, w / torch.where(dead, 1.0, w.sum(1, keepdim=True)))
                got = w.sum(0)
                R = n * G
                each = 2 * (dx + dx.max(1, keepdim=True).values) + (64 + end / 128 / 16) * U32
                err = (w * each).sum(0) + got * (max(min(R, 32), R / 8) + 8) * U32
            if scores_in is not None and decay:
                old = decay * scores_in[s, h, :end].double()
                got = got + old
                err = err + 3 * U32 * (old.abs() + got.abs())
            out[s, h, :end] = got
            tol[s, h, :end] = err + got.abs() * U32 + 2.0 ** -126
    return out, tol


def residuals(pool, layout, cfg, ids, t):
    """The size of turbo_prod's residual part of a K value, [len(t), H, 1]."""
    H, B = cfg.num_kv_heads, cfg.block_size
    page = ids[t // B].long() * int(layout.page_size_bytes)
    cell = (t % B)[:, None] * H + torch.arange(H)

    def scale(off):
        at = page[:, None] + int(off) + cell * 2
        return pool[at[..., None] + torch.arange(2)].contiguous().view(torch.float16).double()

    return (scale(layout.k_residual_scales_offset) * scale(layout.k_scales_offset)).abs()


def select(scores, kv_len, budget, sink, recent):
    """(kept, new lengths, their scores) of select_kv, by sorting (score, place)."""
    S, H, T = scores.shape
    kept = torch.full((S, H, budget), -1, dtype=torch.int32)
    moved = torch.zeros(S, H, T)
    new = torch.zeros(S, dtype=torch.int32)
    for s in range(S):
        L = min(max(int(kv_len[s]), 0), T)
        new[s] = min(L, budget)
        for h in range(H):
            x = scores[s, h, :L].tolist()
            if L <= budget:
                ids = list(range(L))
            else:
                mid = sorted(range(sink, L - recent),
                             key=lambda t: (1, 0.0, t) if x[t] != x[t] else (0, -x[t], t))
                ids = sorted(list(range(sink)) + mid[:budget - sink - recent] + list(range(L - recent, L)))
            kept[s, h, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            moved[s, h, :len(ids)] = scores[s, h, ids]
    return kept, new, moved


def regions(scheme, layout, cfg):
    """(byte offset, bytes per cell) of every region of a page."""
    D = cfg.head_dim
    if scheme == "dense":
        return [(int(layout.k_offset), 2 * D), (int(layout.v_offset), 2 * D)]
    if scheme == "turbo_prod":
        return [(int(layout.k4_codes_offset), D // 2), (int(layout.v4_codes_offset), D // 2)] + [
            (int(o), 2) for o in (layout.k_residual_scales_offset, layout.k_scales_offset,
                                  layout.v_scales_offset)]
    return [(int(layout.k_codes_offset), D // 2), (int(layout.v_codes_offset), D // 2),
            (int(layout.k_norms_offset), 2), (int(layout.v_norms_offset), 2)]


def compact(scheme, pool, tables, kept, layout, cfg, out_tables=None):
    """The pool after compact_kv, cell by cell."""
    H, B = cfg.num_kv_heads, cfg.block_size
    page = int(layout.page_size_bytes)
    to, out = tables if out_tables is None else out_tables, pool.clone()
    for s, h, j in (kept >= 0).nonzero().tolist():
        t = int(kept[s, h, j])
        if t // B >= tables.shape[1] or j // B >= to.shape[1]:
            continue
        a, b = int(tables[s, t // B]), int(to[s, j // B])
        if a < 0 or b < 0 or (out_tables is None and t <= j):
            continue
        for off, n in regions(scheme, layout, cfg):
            src, dst = a * page + off + (t % B * H + h) * n, b * page + off + (j % B * H + h) * n
            out[dst:dst + n] = pool[src:src + n]
    return out
