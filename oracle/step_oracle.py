"""float64 restatement of the speculative step's operators (norm + rotation,
append to dense pages, tree attention), with the error that each entry's
roundings may leave, on the CPU.

Tolerances count roundings.  u(t) = eps(t) / 2 is one rounding to t relative to
the value; u32 = 2^-24.
"""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
K3 = torch.tensor([-2.1513, -1.34326, -0.755526, -0.244919, 0.244919, 0.755526, 1.34326, 2.1513])
V4 = torch.tensor([-2.7326, -2.0690, -1.6180, -1.2562, -0.9423, -0.6568, -0.3880, -0.1284,
                   0.1284, 0.3880, 0.6568, 0.9423, 1.2562, 1.6180, 2.0690, 2.7326])


def unit(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half the distance of the smallest subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def agrees(got, ref, tol, dtype: torch.dtype):
    """Where got (float64 of a dtype value) is within tol of ref.  From half a
    step past dtype's largest value on (65,520 in fp16: the largest 65,504 and
    half of its step of 32) rounding to nearest gives infinity, so an infinity of
    ref's sign agrees where ref may lie there."""
    top = torch.finfo(dtype).max * (1 + unit(dtype) / 2)
    over = torch.isinf(got) & (got.sign() == ref.sign()) & (ref.abs() + tol >= top)
    return ((got - ref).abs() <= tol) | over


def norm_rope(x, weight, pos, table, interleaved, eps):
    """(y, tolerance) of x [N, heads, D] (CPU), both float64.

    fp32 error: the sum of D <= 128 squares has at most 24 roundings on any
    path (16 in a lane or 1, then up to 6 between lanes), half of that through the
    root; root, division, two products and the bf16/fp16 inputs' exact widening
    add 4, the rotation's product and sum 2: 18 < 32 of U32 relative to |a| + |b|."""
    y = x.double()
    D = y.shape[-1]
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    rot = table.shape[1]
    c = table[pos.long(), :rot // 2].double()[:, None]
    s = table[pos.long(), rot // 2:].double()[:, None]
    i = torch.arange(rot // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out, size = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return out, unit(x.dtype) * out.abs() + 32 * U32 * size + tiny(x.dtype)


def hadamard(D: int) -> torch.Tensor:
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < D:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(D)


def signs(h: int, D: int) -> torch.Tensor:
    return (1 - 2 * ((torch.arange(D) + h) % 2)).double()


def cell_rows(scheme, dtype, pool, layout, cfg, ids, t):
    """K and V [len(t), H, D] float64 of tokens t of a sequence with page ids
    `ids`, as the pages hold them (rotated for the compressed schemes)."""
    H, D, B = cfg.num_kv_heads, cfg.head_dim, cfg.block_size
    page = ids[t // B].long() * int(layout.page_size_bytes)
    cell = (t % B)[:, None] * H + torch.arange(H)

    def field(off, size):
        at = page[:, None] + off + cell * size
        return pool[(at[..., None] + torch.arange(size))]

    if scheme == "dense":
        return tuple(field(int(o), 2 * D).contiguous().view(dtype).double()
                     for o in (layout.k_offset, layout.v_offset))

    def scale(off):
        return field(int(off), 2).contiguous().view(torch.float16).double()

    def nibbles(off):
        b = field(int(off), D // 2)
        return torch.stack([b & 15, b >> 4], -1).flatten(-2).long()

    if scheme == "turbo_prod":
        n = nibbles(layout.k4_codes_offset)
        k = K3.double()[n & 7] + torch.where(n > 7, 1.0, -1.0) * scale(layout.k_residual_scales_offset)
        return (k * scale(layout.k_scales_offset),
                V4.double()[nibbles(layout.v4_codes_offset)] * scale(layout.v_scales_offset))
    return (V4.double()[nibbles(layout.k_codes_offset)] * scale(layout.k_norms_offset),
            V4.double()[nibbles(layout.v_codes_offset)] * scale(layout.v_norms_offset))


def tree_attention(scheme, query, pool, tables, row_start, prefix, mask, layout, cfg, max_kv,
                   weight=None):
    """(output, tolerance, rows written) float64 [N, Hq, D] of CPU tensors.

    Roundings: weights (`weight` of each; by default to the pages' 16-bit type,
    half a step of fp16 or bf16; 2 U32 of their exponential's argument and sum
    apart), the output once.  A
    logit is a sum of D products in fp32: D + 4 roundings of at most sum |q k|,
    and the argument's own 2.  Compressed pages: q and k as fp16 pairs (2^-21 of
    each product together), V's levels within 2^-13 of the codebook, and the
    rotations' log2(D) + 2 roundings of q and o."""
    H, D = cfg.num_kv_heads, cfg.head_dim
    N, Hq = query.shape[:2]
    G = Hq // H
    out = torch.zeros(N, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    written = torch.zeros(N, dtype=torch.bool)
    turned = scheme != "dense"
    had = hadamard(D)
    if weight is None:
        weight = unit(query.dtype)
    for s in range(prefix.numel()):
        r0, r1, L = int(row_start[s]), int(row_start[s + 1]), int(prefix[s])
        n = r1 - r0
        if n <= 0:
            continue
        written[r0:r1] = True
        t = torch.arange(min(L + n, max_kv))
        t = t[tables[s][t // cfg.block_size] >= 0] if t.numel() else t
        if not t.numel():
            continue
        k, v = cell_rows(scheme, query.dtype, pool, layout, cfg, tables[s], t)
        j = (t - L).clamp(min=0)
        words = torch.zeros(n, (n + 31) // 32 + 1, dtype=torch.int64)
        m = min(words.shape[1], mask.shape[1])
        words[:, :m] = mask[r0:r1, :m].long()
        see = (t < L)[None] | ((words[:, j >> 5] >> (j & 31)[None]) & 1).bool()
        see &= (t < L)[None] | (j < 32 * mask.shape[1])[None]
        for h in range(H):
            rows = slice(h * G, (h + 1) * G)
            q = query[r0:r1, rows].double().reshape(-1, D)
            if turned:
                q = (q * signs(h, D)) @ had
            sh = see.repeat_interleave(G, 0)
            used = sh.any(0)
            kk, vv, sh = k[used, h], v[used, h], sh[:, used]
            x = (q @ kk.T) / math.sqrt(D)
            size = (q.abs() @ kk.abs().T) / math.sqrt(D)
            x = x.masked_fill(~sh, -math.inf)
            top = x.max(1, keepdim=True).values if x.shape[1] else torch.zeros(n * G, 1)
            dead = ~sh.any(1, keepdim=True)
            w = torch.exp(x - torch.where(dead, 0.0, top)).masked_fill(~sh, 0.0)
            w = w / torch.where(dead, 1.0, w.sum(1, keepdim=True))
            # a value that no row of this call sees differently may be infinite: 0 * inf
            o = torch.where(w[:, :, None] > 0, w[:, :, None] * vv, 0.0).sum(1) \
                if not torch.isfinite(vv).all() else w @ vv
            big = w @ vv.abs().nan_to_num(0.0, 0.0, 0.0)
            dl = (D + 8) * U32 + (2.0 ** -21 + (math.log2(D) + 2) * U32 if turned else 0.0)
            arg = (size.masked_fill(~sh, 0.0).max(1, keepdim=True).values if x.shape[1]
                   else torch.zeros(n * G, 1)) * dl
            # (weights and their sum each move by arg; 64 U32 the sums' own roundings, which
            # grow with the logarithm of the tokens: chunks, lanes and waves are summed apart)
            e = big * (weight + 2 * arg + 64 * U32 + (2.0 ** -13 if turned else 0.0))
            # fp16 weights are multiples of 2^-24 where they are subnormal, so half of that off; a
            # row's largest weight is 2^11 or more: 2^-25 / 2^11 of it each
            if query.dtype == torch.float16:
                e = e + 2.0 ** -36 * vv.abs().nan_to_num(0.0, 0.0, 0.0).sum(0)
            if turned:
                o = (o @ had) * signs(h, D)
                e = e.sum(1, keepdim=True).expand_as(e) / math.sqrt(D)
            o = o.view(n, G, D)
            out[r0:r1, rows] = o
            tol[r0:r1, rows] = e.reshape(n, G, D) + unit(query.dtype) * o.abs() + tiny(query.dtype)
    return out, tol, written
