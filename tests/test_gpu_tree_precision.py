"""Precision of the tree attention's weights and logits, below what its output's
own rounding hides: sums that are small beside the values' sizes (dense pages,
value by value), and two tokens of nearly equal logits and opposite values,
whose output is half the logits' difference times the value row."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.step_oracle import agrees, tree_attention, unit
from test_gpu_tree import Problem
from turborag_amd.synthetic import as_u16, kv_tokens_major

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
B = 16
FAR = 300_000  # tokens that the cache may hold: tiles as for many tokens


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("lens,widths,Hq,H,room", [
    ([40, 9], [3, 2], 8, 2, 0),                   # tiles of 16 rows
    ([3000], [5], 16, 2, 0),
    ([500, 40], [7, 7], 8, 2, FAR),               # 32
    ([500, 40], [7, 7], 16, 2, FAR),              # 64
    ([500, 40], [14, 14], 16, 2, FAR),            # 128
    ([500, 40], [30, 30], 32, 2, FAR),            # 256
])
def test_weights(tq, cuda, monkeypatch, lens, widths, Hq, H, room, dtype, D):
    """A weight in two parts of the pages' type is off by a half step of a half step."""
    monkeypatch.setattr(Problem, "room", room)
    p = Problem(tq, "dense", dtype, lens, widths, Hq, H, D, seed=71, q_scale=0.02)
    got = p.run(cuda)
    ref, tol, _ = tree_attention("dense", p.query, p.pool, p.tables, p.row_start, p.prefix, p.mask,
                                 p.layout, p.cfg, p.max_kv, weight=unit(dtype) ** 2)
    d = (got - ref).abs()
    print(f"    worst {float((d / tol).max()):.2f} of the tolerance", flush=True)
    assert agrees(got, ref, tol, dtype).all()


def _two_tokens(tq, cuda, scheme, n, G, H, D, room, q, pool, cfg, layout):
    """Output [n G, H, D] of query rows q that attend the page's first two tokens."""
    tokens = max(2 + n, room)
    tables = torch.full((1, -(-tokens // B)), -1, dtype=torch.int32, device=cuda)
    tables[0, 0] = 0
    query = q.view(n, G, H, D).transpose(1, 2).reshape(n, H * G, D).contiguous().to(cuda)
    out = torch.full_like(query, 7.0)
    tq.tree_attn_output(scheme, query, pool.to(cuda), tables,
                        torch.tensor([0, n], dtype=torch.int32, device=cuda),
                        torch.tensor([2], dtype=torch.int32, device=cuda),
                        torch.zeros(n, (n + 31) // 32, dtype=torch.int32, device=cuda), out, layout, cfg,
                        tables.shape[1] * B)
    torch.cuda.synchronize()
    return out.cpu().view(n, H, G, D).transpose(1, 2).reshape(n * G, H, D)


def _near_queries(k0, k1, Q, H, D):
    """fp16 queries with <q, k0> = <q, k1> = 20 to 85 sqrt(D) but for their rounding."""
    rng = np.random.default_rng(3)
    u = k0 + k1 + 2 * rng.standard_normal((Q, H, D))
    d = k0 - k1
    u -= (u * d).sum(-1, keepdims=True) / (d * d).sum(-1, keepdims=True) * d
    u *= rng.uniform(20, 85, (Q, H, 1)) * D ** 0.5 / (u * k0).sum(-1, keepdims=True)
    return torch.from_numpy(u).half()


def _rms(out, ref, v):
    """Of the logits' difference that the outputs show."""
    e = ((out - ref) * v).sum(-1) / (v * v).sum(-1)
    return 2 * np.sqrt((e ** 2).mean())


# drafted tokens, query heads per kv head, kv heads, room: tiles of 16, 32, 64, 128, 256 rows
SIZES = [(2, 8, 32, 0), (4, 8, 16, FAR), (8, 8, 8, FAR), (16, 8, 4, FAR), (40, 8, 2, FAR)]


@pytest.mark.parametrize("n,G,H,room", SIZES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_near_equal_logits_compressed(tq, oracle, cuda, scheme, D, n, G, H, room):
    """The difference's rms error within that of the reference's fp32 arithmetic, times 1.25 for
    the scatter of an rms, and for more roundings near the logit's magnitude.  The matrix cores round
    after every eight products (1 + 1 of two eights, added to 2^24 by one instruction, stays
    2^24; of the same eight it gives 2^24 + 2).  Of a logit of head_dim 128, K and q in two parts
    each, that is sixteen sums at i / 16 of it (squares: 5.8) and, of the parts' other two products,
    eight each at 1/4, 1/2 and 3/4 (7.0), and one of K's scale: 13.8.  Head_dim 64: eight at i / 8
    (3.2), eight at 1/2 (2.0), one: 6.2.  The reference's pairwise tree has the equivalent of two."""
    prod = scheme == "turbo_prod"
    k, v = kv_tokens_major(2, H, D, seed=5)
    v[1] = -v[0]
    slots = np.arange(2, dtype=np.int32)
    pool = (oracle.prod_pack if prod else oracle.mse_pack)(as_u16(k), as_u16(v), slots, 1, B)
    kd = (oracle.prod_dequant if prod else oracle.mse_dequant)(pool, slots, H, D, B)[0]
    q = _near_queries(*kd.view(np.float16).astype(np.float64), n * G, H, D)
    f64 = oracle.prod_attention_f64 if prod else oracle.mse_attention_f64
    f32 = oracle.prod_attention_f32 if prod else oracle.mse_attention_f32
    ref = f64(as_u16(q), pool, slots, B)
    fp32 = np.asarray(f32(as_u16(q), pool, slots, B)).view(np.float16).astype(np.float64)
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim = H, D
    layout = tq.make_layout_for(cfg) if prod else tq.make_mse_layout_for(cfg)
    out = _two_tokens(tq, cuda, scheme, n, G, H, D, room, q, torch.from_numpy(pool), cfg, layout)
    vv = v[0].double().numpy()
    got, want = _rms(out.double().numpy(), ref, vv), _rms(fp32.reshape(ref.shape), ref, vv)
    print(f"    rms {got:.2e}, fp32 {want:.2e}: {got / want:.2f}", flush=True)
    assert got <= 1.25 * math.sqrt((13.8 if D == 128 else 6.2) / 2) * want


@pytest.mark.parametrize("n,G,H,room", SIZES)
@pytest.mark.parametrize("D", [64, 128])
def test_near_equal_logits_dense(tq, cuda, D, n, G, H, room):
    """As above, with K and q in one part, against a pairwise tree in fp32: 5.8 and 3.2 against two,
    and one for the division by sqrt(128)."""
    k, v = (x.half() for x in kv_tokens_major(2, H, D, seed=5))
    v[1] = -v[0]
    kd = k.double().numpy()
    q = _near_queries(kd[0], kd[1], n * G, H, D)
    cfg = tq.default_config()
    cfg.num_kv_heads, cfg.head_dim = H, D
    layout = tq.make_dense_layout_for(cfg)
    pool = torch.zeros(int(layout.page_size_bytes), dtype=torch.uint8)
    for x, at in ((k, layout.k_offset), (v, layout.v_offset)):
        b = x.contiguous().view(-1).view(torch.uint8)
        pool[int(at):int(at) + b.numel()] = b
    out = _two_tokens(tq, cuda, "dense", n, G, H, D, room, q, pool, cfg, layout)

    def outputs(dtype, total):
        x = [total(q.numpy().astype(dtype) * k[t].numpy().astype(dtype)) / dtype(math.sqrt(D))
             for t in range(2)]
        return np.tanh((x[0] - x[1]).astype(np.float64) / 2)[..., None] * v[0].double().numpy()

    def pairwise(x):
        while x.shape[-1] > 1:
            x = x[..., 0::2] + x[..., 1::2]
        return x[..., 0]

    ref = outputs(np.float64, lambda x: x.sum(-1))
    fp32 = outputs(np.float32, pairwise).astype(np.float16).astype(np.float64)
    vv = v[0].double().numpy()
    got, want = _rms(out.double().numpy(), ref, vv), _rms(fp32, ref, vv)
    print(f"    rms {got:.2e}, fp32 {want:.2e}: {got / want:.2f}", flush=True)
    assert got <= 1.25 * math.sqrt(5.8 / 3 if D == 128 else 3.2 / 2) * want


@pytest.mark.parametrize("scheme", ["turbo_prod", "turbo_mse"])
def test_chain_is_as_exact_as_the_paged_step(tq, cuda, scheme):
    """Trees without branches over a PagedBatch's pages: error against float64 in the mean no more
    than the paged entry's (times 1.02 for its scatter over 32,768 values, about 0.4%)."""
    from turborag_amd.batched import PagedBatch
    from turborag_amd.turboquant_wrapper import tree_mask_from_parents
    b = PagedBatch(tq, scheme, [1500, 37, 300], [3, 8, 5], seed=560, device=cuda)
    b.append_new_tokens(seed=920)
    rows, row_seq, row_len = b.decode_rows(seed=921)
    tables = b.block_tables()
    paged = torch.zeros_like(rows)
    b.attention(rows, row_seq, row_len, tables, paged)
    query = rows.view(16, 8, 2, 128).transpose(1, 2).reshape(16, 16, 128).contiguous()
    start, prefix = b.tree_rows()
    mask = torch.zeros(16, 1, dtype=torch.int32)
    for s, w in enumerate(b.widths):
        r = int(start[s])
        mask[r:r + w] = tree_mask_from_parents(range(-1, w - 1))
    out = torch.zeros_like(query)
    b.tree_attention(query, start, prefix, mask.to(cuda), tables, out)
    ref, _, _ = tree_attention(scheme, query.cpu(), b.pool.cpu().reshape(-1), tables.cpu(), start.cpu(),
                               prefix.cpu(), mask, b.layout, b.cfg, 1 << 20)
    paged = paged.view(16, 8, 2, 128).transpose(1, 2).reshape(query.shape)
    tree, line = (float((x.cpu().double() - ref).pow(2).mean().sqrt()) for x in (out, paged))
    print(f"    rms error: tree {tree:.3e}, paged {line:.3e}", flush=True)
    assert tree <= 1.02 * line
    b.close()
