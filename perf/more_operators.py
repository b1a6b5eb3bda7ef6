"""Timed calls of the operators of long documents with images or video in a
cache of bounded size: positions with several axes, and eviction from the cache
by accumulated attention weight.

``run`` computes them from elementary torch operations in float32, or with
``own`` through the library's entry points.  ``exact`` states them again in
float64.  Inputs are drawn on the GPU from the seed; compressed pages are
written here byte for byte, in the layouts of ``include/turboquant.h``.

Kinds:

* ``rope``: RMS norm (optional) and rotation of q and k, every pair of dims by
  the position on its own axis (time, height, width);
* ``append``: the same with K rotated into, and V copied into, a dense page
  pool through a slot mapping;
* ``weights``: what the last tokens' softmax weights on every cached token add
  up to over a kv head's query rows, added to the scores of earlier steps;
* ``select``: the tokens of every kv head that a budget keeps (the first ones,
  the last ones, the highest scores), and their scores moved up;
* ``compact``: the kept tokens' cells moved to the front of their sequences.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16       # tokens per page (the library's default configuration)
EPS = 1e-6
BASE = 10000.0  # of the rotation's angles
POSITIONS = 40960

_tq = None


def _lib():
    global _tq
    if _tq is None:
        from turborag_amd.turboquant_wrapper import TurboQuantWrapper
        _tq = TurboQuantWrapper()
    return _tq


# ── the cases ────────────────────────────────────────────────────────────── #

def listed() -> list[dict]:
    return [
        # One new token of one sequence, 16 query heads on 2 kv heads: nothing but latency.
        dict(name="axes_1", kind="rope", dtype="fp16", q_heads=16, heads=2, dim=128, tokens=1,
             norm=True, interleaved=False, axes="16,24,24", turns=False),
        # The prefill of a document with images, in bf16: blocks of pairs for time, height, width.
        dict(name="axes_8k", kind="rope", dtype="bf16", q_heads=16, heads=2, dim=128, tokens=8192,
             norm=True, interleaved=False, axes="16,24,24", turns=False),
        # One image and a question at the store's default head shape, the axes' pairs in turn.
        dict(name="axes_append_d64_1143", kind="append", dtype="fp16", q_heads=14, heads=2, dim=64,
             tokens=1143, norm=False, interleaved=True, axes="12,10,10", turns=True),
        # A whole video of 32K tokens into the dense cache, the axes' pairs in turn.
        dict(name="axes_append_32k", kind="append", dtype="fp16", q_heads=16, heads=2, dim=128,
             tokens=32768, norm=True, interleaved=False, axes="24,20,20", turns=True),
        # A decode step of one sequence over a short document: the scores' smallest update.
        dict(name="weights_1143", kind="weights", scheme="dense", dtype="fp16", q_heads=16, heads=2,
             dim=128, seqs=1, shortest=1143, longest=1143, width=1, add=True),
        # The last 32 tokens of a 32K document's prefill look back over it, once.
        dict(name="weights_window_32k", kind="weights", scheme="dense", dtype="fp16", q_heads=16,
             heads=2, dim=128, seqs=1, shortest=32768, longest=32768, width=32, add=False),
        # A decode step of 32 ragged sequences over dense bf16 pages, added up: the largest.
        dict(name="weights_32seq", kind="weights", scheme="dense", dtype="bf16", q_heads=16, heads=2,
             dim=128, seqs=32, shortest=1024, longest=32768, width=1, add=True),
        # Up to 8 accepted tokens of 32 ragged sequences over compressed pages.
        dict(name="weights_32seq_prod", kind="weights", scheme="turbo_prod", dtype="fp16", q_heads=16,
             heads=2, dim=128, seqs=32, shortest=300, longest=8192, width=8, add=True),
        # A short document cut to 256 tokens.
        dict(name="select_1143", kind="select", heads=2, seqs=1, shortest=1143, longest=1143,
             budget=256, sink=4, recent=32),
        # 32 ragged sequences cut to 2,048 tokens each.
        dict(name="select_32seq", kind="select", heads=2, seqs=32, shortest=1024, longest=32768,
             budget=2048, sink=4, recent=64),
        # A window that slides, in place: the first tokens and the last ones of 12 sequences.
        dict(name="compact_window_mse_d64", kind="compact", scheme="turbo_mse", dtype="fp16", heads=2,
             dim=64, seqs=12, shortest=2100, longest=6001, budget=1000, sink=4, in_place=True),
        # Tokens by their scores into pages of their own (the originals stay, for other requests).
        dict(name="compact_32seq", kind="compact", scheme="dense", dtype="bf16", heads=2, dim=128,
             seqs=32, shortest=1024, longest=32768, budget=4096, sink=4, in_place=False),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rope", "append", "weights", "weights", "weights", "select", "compact", "compact"])
    q_heads, heads = rng.choice([(16, 2), (14, 2), (8, 1), (16, 4), (32, 8), (4, 4), (12, 4)])
    dim = rng.choice([64, 128])
    c = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), q_heads=q_heads, heads=heads, dim=dim)
    if kind in ("rope", "append"):
        c["tokens"] = _log_int(rng, 1, 32768 * 16 * 128 // (q_heads * dim) if q_heads > 8 else 32768)
        c["tokens"] = min(c["tokens"], 32768 if dim * heads <= 256 else 8192)
        count, pairs = rng.choice([2, 3, 3, 4]), dim // 2
        cuts = sorted(rng.sample(range(1, pairs // 4), count - 1))  # in steps of 4 pairs, or of one
        step = rng.choice([1, 4])
        cuts = [0] + [x * step for x in cuts] + [pairs]
        c["axes"] = ",".join(str(b - a) for a, b in zip(cuts, cuts[1:]))
        c.update(norm=rng.random() < 0.5, interleaved=rng.random() < 0.3, turns=rng.random() < 0.5)
        return c
    c["seqs"] = _log_int(rng, 1, 32)
    # cells (sequence, token, head, dim) up to about those of the largest listed case
    c["longest"] = _log_int(rng, 16, min(32768, 32 * 16000 * 256 // (c["seqs"] * heads * dim)))
    c["shortest"] = max(1, c["longest"] // rng.choice([1, 4, 30]))
    if kind == "select":
        c["longest"] = _log_int(rng, 16, 2 * 32 * 16000 // (c["seqs"] * heads))
        c["longest"] = min(c["longest"], 131072)
        c["shortest"] = max(1, c["longest"] // rng.choice([1, 4, 30]))
        c["budget"] = _log_int(rng, 1, min(8192, c["longest"]))
        c["sink"] = min(rng.choice([0, 4, 16]), c["budget"])
        c["recent"] = min(rng.choice([0, 32, 200]), c["budget"] - c["sink"])
        del c["dtype"], c["q_heads"], c["dim"]
        return c
    c["scheme"] = rng.choice(["dense", "dense", "turbo_prod", "turbo_mse"])
    if c["scheme"] != "dense":
        c["dtype"] = "fp16"
    if kind == "weights":
        c["width"] = _log_int(rng, 1, max(1, min(64, 256 // c["seqs"])))
        c["add"] = rng.random() < 0.5
        return c
    c["in_place"] = rng.random() < 0.5
    c["sink"] = rng.choice([0, 1, 4, 16])
    if c["in_place"]:  # a window no longer than what is evicted before it
        c["shortest"] = max(2, c["longest"] // rng.choice([1, 4]))
        c["budget"] = _log_int(rng, 1, max(1, (c["shortest"] - 11) // 2))
        c["shortest"] = max(c["shortest"], 2 * c["budget"] + 11)
        c["longest"] = max(c["longest"], c["shortest"])
    else:
        c["budget"] = _log_int(rng, 1, min(8192, c["longest"]))
    c["sink"] = min(c["sink"], c["budget"])
    del c["q_heads"]
    return c


# ── inputs ───────────────────────────────────────────────────────────────── #

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _pages(n: int) -> int:
    return (n + PAGE - 1) // PAGE


def _outliers(x: torch.Tensor) -> torch.Tensor:
    """Scales each head's four outlier channels of x [n, H, D] by 8, in place."""
    H, D = x.shape[1:]
    for h in range(H):
        x[:, h, [(7 * h + 13 * j + 5) % D for j in range(4)]] *= 8.0
    return x


def _lens(c: dict) -> list[int]:
    """Cached tokens of every sequence."""
    S, lo, hi = c["seqs"], c["shortest"], c["longest"]
    lens = [lo + (hi - lo) * s // (S - 1) if S > 1 else hi for s in range(S)]
    lens = [max(1, n - (s * 5) % 11) for s, n in enumerate(lens)]
    random.Random(S).shuffle(lens)
    return lens


def _widths(c: dict) -> list[int]:
    """Query tokens of every sequence (its last ones)."""
    W = c["width"]
    return [W - (s * 3) % max(1, (W + 1) // 2) for s in range(c["seqs"])]


def _table(n: int, dim: int) -> torch.Tensor:
    """cos | sin of every position's angles, [n, dim] fp32."""
    f = BASE ** (-torch.arange(0, dim, 2, device="cuda").double() / dim)
    a = torch.arange(n, device="cuda").double()[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _sections(c: dict) -> list[int]:
    return [int(x) for x in c["axes"].split(",")]


def _axis_of_pair(c: dict) -> list[int]:
    """The axis that turns each pair: blocks of pairs, or dealt in turn to the axes that have some
    left."""
    left = _sections(c)
    if not c["turns"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


def _positions(c: dict, seed: int) -> torch.Tensor:
    """[axes, tokens] int32: text, where all axes count alike, and images between it, whose tokens
    share a time and count rows and columns."""
    N, A = c["tokens"], len(_sections(c))
    rng = random.Random(seed)
    rows, at, base = [], 0, rng.randrange(1000)
    while at < N:
        n = min(N - at, rng.randrange(1, 400))
        rows.append((torch.arange(n) + base).expand(A, n))
        at, base = at + n, base + n
        if at < N:
            h, w = rng.randrange(4, 40), rng.randrange(4, 40)
            n = min(N - at, h * w)
            i = torch.arange(n)
            grid = [torch.zeros(n, dtype=torch.long), i // w, i % w, i % 2][:A]
            rows.append(torch.stack(grid) + base)
            at, base = at + n, base + max(h, w)
    return torch.cat(rows, 1).clamp(max=POSITIONS - 1).int().cuda()


def _rope_state(c: dict, seed: int) -> dict:
    g, N, Hq, H, D = _gen(seed), c["tokens"], c["q_heads"], c["heads"], c["dim"]
    dt = _DTYPES[c["dtype"]]
    # q, k and v as the views of one fused projection's output, as a model has them
    qkv = torch.randn(N, Hq + 2 * H, D, generator=g, device="cuda")
    _outliers(qkv[:, Hq:Hq + H])
    qkv = qkv.to(dt)
    s = dict(case=c, q=qkv[:, :Hq], k=qkv[:, Hq:Hq + H], v=qkv[:, Hq + H:],
             table=_table(POSITIONS, D), pos=_positions(c, seed), qw=None, kw=None,
             axis=torch.tensor(_axis_of_pair(c), device="cuda"))
    if c["norm"]:
        s["qw"], s["kw"] = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)
                            for _ in range(2))
    s["out_q"] = torch.empty(N, Hq, D, dtype=dt, device="cuda")
    if c["kind"] == "rope":
        s["out_k"] = torch.empty(N, H, D, dtype=dt, device="cuda")
        return s
    P = _pages(N) + 3
    perm = torch.randperm(P, generator=g, device="cuda")
    t = torch.arange(N, device="cuda")
    s["slots"] = (perm[t // PAGE] * PAGE + t % PAGE).int()
    s["pages"] = torch.zeros(P, 2, PAGE, H, D, dtype=dt, device="cuda")
    return s


_K3 = [-2.1513, -1.34326, -0.755526, -0.244919, 0.244919, 0.755526, 1.34326, 2.1513]
_V4 = [-2.7326, -2.0690, -1.6180, -1.2562, -0.9423, -0.6568, -0.3880, -0.1284,
       0.1284, 0.3880, 0.6568, 0.9423, 1.2562, 1.6180, 2.0690, 2.7326]


def _levels(values: list[float]) -> torch.Tensor:
    return torch.tensor(values, device="cuda")  # the codebooks are fp32


def _cells(g: torch.Generator, rows: int, D: int, key: bool):
    """Codes [rows, D / 2], RMS [rows] and (turbo_prod K) residual RMS of rotated rows, as packing
    K/V with outlier channels leaves them: N(0, 1) values, an RMS around 1.7."""
    y = torch.randn(rows, D, generator=g, device="cuda")
    lv = _levels(_K3 if key else _V4)
    n = torch.bucketize(y, (lv[1:] + lv[:-1]) / 2)
    res = None
    if key:
        e = y - lv[n]
        res = e.square().mean(1).sqrt().half()
        n = n | ((e >= 0).long() << 3)
    n = n.to(torch.uint8)
    rms = (1.7 * torch.exp(0.15 * torch.randn(rows, generator=g, device="cuda"))).half()
    return n[:, 0::2] | (n[:, 1::2] << 4), rms, res


def _pool(c: dict, g: torch.Generator, P: int) -> torch.Tensor:
    """A pool of P pages, [P, page bytes] uint8."""
    H, D, prod = c["heads"], c["dim"], c["scheme"] == "turbo_prod"
    if c["scheme"] == "dense":
        pool = torch.empty(P, 2, PAGE, H, D, dtype=_DTYPES[c["dtype"]], device="cuda")
        for lo in range(0, P, 4096):
            part = torch.randn(pool[lo:lo + 4096].shape, generator=g, device="cuda")
            pool[lo:lo + 4096] = _outliers(part.view(-1, H, D)).view(part.shape)
        return pool.view(torch.uint8).reshape(P, -1)
    parts = []
    for lo in range(0, P, 4096):
        n = min(4096, P - lo)
        cells = n * PAGE * H

        def region(x):
            b = x.contiguous().view(torch.uint8).reshape(n, -1)
            pad = 0 if prod else -b.shape[1] % 256  # turbo_mse regions are 256-byte aligned
            return torch.nn.functional.pad(b, (0, pad))

        kc, ks, kr = _cells(g, cells, D, prod)
        vc, vs, _ = _cells(g, cells, D, False)
        parts.append(torch.cat([region(x) for x in
                                ((kc, kr, ks, vc, vs) if prod else (kc, vc, ks, vs))], 1))
    return torch.cat(parts)


def _tables(order: torch.Tensor, counts: list[int]) -> torch.Tensor:
    """Block tables [S, most] of sequences that take their pages from `order` one behind another."""
    tables = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables


def _weights_state(c: dict, seed: int) -> dict:
    g, H, D = _gen(seed), c["heads"], c["dim"]
    lens, widths = _lens(c), _widths(c)
    total = [n + w for n, w in zip(lens, widths)]
    counts = [_pages(n) for n in total]
    P, T = sum(counts), max(total)
    pool = _pool(c, g, P)
    tables = _tables(torch.randperm(P, generator=g, device="cuda").int(), counts)
    start = torch.tensor([sum(widths[:i]) for i in range(len(widths) + 1)], dtype=torch.int32,
                         device="cuda")
    q = torch.randn(sum(widths), c["q_heads"], D, generator=g, device="cuda").to(_DTYPES[c["dtype"]])
    s = dict(case=c, pool=pool.reshape(-1), tables=tables, start=start, q=q, most=T, before=None,
             prefix=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             scores=torch.zeros(len(lens), H, T, device="cuda"))
    if c["add"]:  # the scores of a few hundred steps
        s["before"] = torch.exp(2 * torch.randn(len(lens), H, T, generator=g, device="cuda"))
    return s


def _select_state(c: dict, seed: int) -> dict:
    g, S, H = _gen(seed), c["seqs"], c["heads"]
    lens = _lens(c)
    T = max(lens)
    # heavy tails, high first tokens, and some that no row ever looked at
    x = torch.exp(2.5 * torch.randn(S, H, T, generator=g, device="cuda"))
    x[..., :4] *= 1000.0
    x[torch.rand(S, H, T, generator=g, device="cuda") < 0.02] = 0.0
    return dict(case=c, scores=x, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                kept=torch.empty(S, H, c["budget"], dtype=torch.int32, device="cuda"),
                new_len=torch.empty(S, dtype=torch.int32, device="cuda"), moved=torch.empty_like(x))


def _compact_state(c: dict, seed: int) -> dict:
    g, S, H, B = _gen(seed), c["seqs"], c["heads"], c["budget"]
    lens = _lens(c)
    T = max(lens)
    counts = [_pages(n) for n in lens]
    fresh = [] if c["in_place"] else [_pages(min(n, B)) for n in lens]
    P = sum(counts) + sum(fresh)
    pool = _pool(c, g, P)
    order = torch.randperm(P, generator=g, device="cuda").int()
    n = torch.tensor(lens, device="cuda")[:, None, None]
    t = torch.arange(T, device="cuda")
    if c["in_place"]:
        key = torch.where(t >= n - (B - c["sink"]), 1.0, 0.0).expand(S, H, T).clone()
    else:
        key = torch.rand(S, H, T, generator=g, device="cuda")
    key[..., :c["sink"]] = 2.0
    key = torch.where(t < n, key, -1.0)
    kept = key.topk(min(B, T), dim=-1).indices
    kept = torch.where(kept < n, kept, T).sort(dim=-1).values
    kept = torch.nn.functional.pad(torch.where(kept < T, kept, -1), (0, max(0, B - T)), value=-1)
    return dict(case=c, pool=pool.reshape(-1), tables=_tables(order, counts), kept=kept.int(),
                out_tables=None if c["in_place"] else _tables(order[sum(counts):], fresh))


def prepare(case: dict, seed: int) -> dict:
    make = {"weights": _weights_state, "select": _select_state, "compact": _compact_state}
    return make.get(case["kind"], _rope_state)(case, seed)


# ── one pass ─────────────────────────────────────────────────────────────── #

def _run_own(s: dict):
    c, tq = s["case"], _lib()
    if c["kind"] == "select":
        tq.select_kv(s["scores"], s["lens"], s["kept"], s["new_len"], sink=c["sink"],
                     recent=c["recent"], out_scores=s["moved"])
        return s["kept"], s["new_len"], s["moved"]
    if "cfg" not in s:  # a serving program makes these once
        s["cfg"] = cfg = tq.default_config()
        cfg.num_kv_heads, cfg.head_dim, cfg.block_size = c["heads"], c["dim"], PAGE
        kind = c.get("scheme", "dense")
        s["layout"] = (tq.make_layout_for if kind == "turbo_prod" else tq.make_mse_layout_for
                       if kind == "turbo_mse" else tq.make_dense_layout_for)(cfg)
        if "axes" in c:
            from turborag_amd.turboquant_wrapper import rope_axes
            s["axes"] = rope_axes(_sections(c), in_turn=c["turns"])
    cfg, layout = s["cfg"], s["layout"]
    if c["kind"] == "rope":
        tq.qk_norm_rope(s["q"], s["k"], s["pos"], s["table"], s["out_q"], s["out_k"], cfg,
                        q_weight=s["qw"], k_weight=s["kw"], eps=EPS, interleaved=c["interleaved"],
                        axes=s["axes"])
        return s["out_q"], s["out_k"]
    if c["kind"] == "append":
        tq.dense_rope_append(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["table"], s["out_q"],
                             s["pages"].view(torch.uint8), layout, cfg, q_weight=s["qw"],
                             k_weight=s["kw"], eps=EPS, interleaved=c["interleaved"], axes=s["axes"])
        return s["out_q"], s["pages"]
    if c["kind"] == "weights":
        tq.attn_weights(c["scheme"], s["q"], s["pool"], s["tables"], s["start"], s["prefix"],
                        s["scores"], layout, cfg, s["most"], scores_in=s["before"])
        return s["scores"]
    tq.compact_kv(c["scheme"], s["pool"], s["tables"], s["kept"], layout, cfg,
                  out_block_tables=s["out_tables"])
    return _pool_out(s)


def _pool_out(s: dict) -> torch.Tensor:
    c = s["case"]
    return s["pool"].view(_DTYPES[c["dtype"]]) if c["scheme"] == "dense" else s["pool"]


def _rotated(s: dict, x, weight):
    """x [n, heads, D] normed and rotated, float32."""
    y, pos = x.float(), s["pos"]
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    half = s["table"].shape[1] // 2
    pair = torch.arange(half, device="cuda")
    at = pos.long()[s["axis"]].T  # [n, pairs]
    cos, sin = s["table"][at, pair][:, None], s["table"][at, pair + half][:, None]
    if s["case"]["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = y[..., :half], y[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _hadamard(D: int, dtype) -> torch.Tensor:
    h = torch.ones(1, 1, dtype=dtype, device="cuda")
    while h.shape[0] < D:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(D)


def _nibbles(codes: torch.Tensor) -> torch.Tensor:
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()


def _fields(c: dict) -> list[tuple[str, int, int]]:
    """(name, byte offset, bytes per cell) of a page's regions."""
    H, D = c["heads"], c["dim"]
    if c["scheme"] == "dense":
        return [("k", 0, 2 * D), ("v", PAGE * H * 2 * D, 2 * D)]
    prod = c["scheme"] == "turbo_prod"
    out, at = [], 0
    for name, n in ([("kc", D // 2), ("kr", 2), ("ks", 2), ("vc", D // 2), ("vs", 2)] if prod else
                    [("kc", D // 2), ("vc", D // 2), ("ks", 2), ("vs", 2)]):
        out.append((name, at, n))
        at += PAGE * H * n if prod else (PAGE * H * n + 255) // 256 * 256
    return out


def _page_bytes(c: dict) -> int:
    name, at, n = _fields(c)[-1]
    end = at + PAGE * c["heads"] * n
    return (end + 255) // 256 * 256 if c["scheme"] == "turbo_mse" else end


def _region(s: dict, at: int, n: int) -> torch.Tensor:
    """A region of every page, [pages, 16, H, n] bytes (a view of the pool)."""
    c = s["case"]
    pool = s["pool"].view(-1, _page_bytes(c))
    return pool[:, at:at + PAGE * c["heads"] * n].view(-1, PAGE, c["heads"], n)


def _pool_k(s: dict) -> torch.Tensor:
    """K of every page [pages, 16, H, D], float32."""
    c = s["case"]
    f = {name: _region(s, at, n).contiguous() for name, at, n in _fields(c) if name[0] == "k"}
    if c["scheme"] == "dense":
        return f["k"].view(_DTYPES[c["dtype"]]).float()
    D, H = c["dim"], c["heads"]
    n = _nibbles(f["kc"])
    if "kr" in f:
        k = _levels(_K3)[n & 7] + torch.where(n >= 8, 1.0, -1.0) * f["kr"].view(torch.float16).float()
    else:
        k = _levels(_V4)[n]
    sign = 1.0 - 2.0 * ((torch.arange(D, device="cuda") + torch.arange(H, device="cuda")[:, None]) % 2)
    return (k * f["ks"].view(torch.float16).float()) @ _hadamard(D, torch.float32) * sign


def _plain_weights(s: dict) -> torch.Tensor:
    c = s["case"]
    Hq, H, D, W = c["q_heads"], c["heads"], c["dim"], c["width"]
    G, S = Hq // H, s["prefix"].numel()
    at = s["tables"].clamp(min=0).long()
    k = _pool_k(s)[at].view(S, -1, H, D).transpose(1, 2).contiguous()[:, :, :s["most"]]
    T = k.shape[2]
    start, prefix = s["start"].long(), s["prefix"].long()[:, None, None]
    node = torch.arange(W, device="cuda")
    row = start[:-1, None] + node                     # [S, W]
    live = row < start[1:, None]
    row = row.clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().view(S, W, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, W * G, D)
    t = torch.arange(T, device="cuda")
    seen = (t <= prefix + node[:, None]) & live[..., None]               # [S, W, T]
    seen = seen[:, None, :, None].expand(S, H, W, G, T).reshape(S, H, W * G, T)
    x = (q @ k.transpose(2, 3).contiguous()) / math.sqrt(D)
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    got = (p / p.sum(-1, keepdim=True).clamp_min(1e-30)).sum(2)          # [S, H, T]
    if s["before"] is not None:
        got = s["before"] + got
    kv = prefix + (start[1:] - start[:-1])[:, None, None]
    s["scores"].copy_(torch.where(t < kv, got, s["scores"]))
    return s["scores"]


def _plain_select(s: dict):
    c, x = s["case"], s["scores"]
    T, B = x.shape[2], c["budget"]
    n = s["lens"].long()[:, None, None]
    t = torch.arange(T, device="cuda")
    key = torch.where((t < c["sink"]) | (t >= n - c["recent"]), math.inf, x)
    key = torch.where(t < n, key, -math.inf)
    best = key.sort(dim=-1, descending=True, stable=True).indices[..., :B]
    j = torch.arange(best.shape[-1], device="cuda")
    kept = torch.where(j < n, best, T).sort(dim=-1).values
    count = s["lens"].clamp(max=B)
    s["new_len"].copy_(count)
    s["kept"].fill_(-1)
    s["kept"][..., :kept.shape[-1]] = torch.where(kept < T, kept, -1)
    s["moved"].zero_()
    s["moved"][..., :kept.shape[-1]] = torch.where(kept < T, x.gather(2, kept.clamp(max=T - 1)), 0.0)
    return s["kept"], s["new_len"], s["moved"]


def _plain_compact(s: dict) -> torch.Tensor:
    c, kept = s["case"], s["kept"].long()
    S, H, B = kept.shape
    to = s["tables"] if s["out_tables"] is None else s["out_tables"]
    j = torch.arange(B, device="cuda").expand(S, H, B)
    live = kept >= 0
    seq, head = (torch.arange(n, device="cuda").view(v).expand(S, H, B)[live]
                 for n, v in ((S, (S, 1, 1)), (H, (1, H, 1))))
    src, dst = kept[live], j[live]
    sp, dp = s["tables"][seq, src // PAGE].long(), to[seq, dst // PAGE].long()
    for _, at, n in _fields(c):
        region = _region(s, at, n)
        region[dp, dst % PAGE, head] = region[sp, src % PAGE, head]
    return _pool_out(s)


def run(state: dict):
    s, c = state, state["case"]
    if own:
        return _run_own(s)
    if c["kind"] == "weights":
        return _plain_weights(s)
    if c["kind"] == "select":
        return _plain_select(s)
    if c["kind"] == "compact":
        return _plain_compact(s)
    q, k = (_rotated(s, x, w).to(x.dtype) for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
    if c["kind"] == "rope":
        return q, k
    slot = s["slots"].long()
    s["pages"][slot // PAGE, 0, slot % PAGE] = k
    s["pages"][slot // PAGE, 1, slot % PAGE] = s["v"]
    return q, s["pages"]


# ── what a pass cannot do without ────────────────────────────────────────── #

def work(case: dict) -> dict:
    c, H = case, case["heads"]
    if c["kind"] in ("rope", "append"):
        N, Hq, D = c["tokens"], c["q_heads"], c["dim"]
        moved = (Hq + H + (H if c["kind"] == "append" else 0)) * D * 2 * 2
        b = N * (moved + 4 * D + 4 * len(_sections(c)) + (4 if c["kind"] == "append" else 0))
        return {"bytes": b, "flops": N * (Hq + H) * D * (7 if c["norm"] else 3)}
    lens = _lens(c)
    if c["kind"] == "select":  # scores in, indexes out, scores out
        T = max(lens)
        return {"bytes": 4 * H * (sum(lens) + c["seqs"] * (c["budget"] + T)), "flops": H * sum(lens)}
    if c["kind"] == "compact":
        moved = sum(min(n, c["budget"]) for n in lens)
        if c["in_place"]:  # the first tokens stay
            moved -= sum(min(n, c["sink"]) for n in lens)
        return {"bytes": moved * H * (2 * sum(n for _, _, n in _fields(c)) + 4), "flops": 0}
    Hq, D, widths = c["q_heads"], c["dim"], _widths(c)
    key = sum(n for name, _, n in _fields(c) if name[0] == "k")
    cells = sum(n + w for n, w in zip(lens, widths)) * H
    seen = sum(w * n + w * (w + 1) // 2 for n, w in zip(lens, widths))
    return {"bytes": cells * (key + (8 if c["add"] else 4)) + 2 * sum(widths) * Hq * D,
            "flops": 2 * D * Hq * seen}


# ── the same in float64 ──────────────────────────────────────────────────── #

def _exact_rope(x, weight, s, c):
    y = x.double()
    if weight is not None:
        y = y / (y.square().sum(-1, keepdim=True) / c["dim"] + EPS).sqrt() * weight.double()
    # as complex numbers times e^(i angle), axis by axis
    half = c["dim"] // 2
    pair = (y.unflatten(-1, (half, 2)) if c["interleaved"] else
            y.unflatten(-1, (2, half)).transpose(-1, -2)).contiguous()
    z = torch.view_as_complex(pair)
    out = torch.zeros_like(z)
    whole = torch.complex(s["table"][:, :half].double(), s["table"][:, half:].double())
    for a in range(s["pos"].shape[0]):
        mine = torch.tensor([i for i, b in enumerate(_axis_of_pair(c)) if a == b], dtype=torch.long,
                            device="cuda")
        out[..., mine] = z[..., mine] * whole[s["pos"][a].long()][:, None, mine]
    z = torch.view_as_real(out)
    return (z if c["interleaved"] else z.transpose(-1, -2)).reshape(y.shape)


def _exact_weights(c, s):
    H, D, G = c["heads"], c["dim"], c["q_heads"] // c["heads"]
    out = torch.zeros(s["scores"].shape, dtype=torch.float64, device="cuda")
    had = _hadamard(D, torch.float64)
    f = {name: _region(s, at, n) for name, at, n in _fields(c) if name[0] == "k"}
    at = 0
    for i, (n, w) in enumerate(zip(_lens(c), _widths(c))):
        ids = s["tables"][i, :_pages(n + w)].long()
        own_row = torch.arange(w, device="cuda")
        past = torch.arange(n + w, device="cuda") > n + own_row[:, None]
        for h in range(H):
            q = s["q"][at:at + w, h * G:(h + 1) * G].double().reshape(-1, D)
            b = {name: x[ids, :, h].flatten(0, 1)[:n + w].contiguous() for name, x in f.items()}
            if "k" in b:
                k = b["k"].view(_DTYPES[c["dtype"]]).double()
            else:  # in the rotated domain: the transform is orthogonal
                q = (q * (1 - 2 * ((torch.arange(D, device="cuda") + h) % 2)).double()) @ had
                code = _nibbles(b["kc"])
                k = (_levels(_V4).double()[code] if "kr" not in b else
                     _levels(_K3).double()[code % 8] +
                     (2.0 * (code // 8) - 1.0) * b["kr"].view(torch.float16).double())
                k = k * b["ks"].view(torch.float16).double()
            x = (q @ k.T.contiguous()) * D ** -0.5
            x = x.masked_fill(past.repeat_interleave(G, 0), -math.inf)
            out[i, h, :n + w] = torch.softmax(x, -1).sum(0)
            if s["before"] is not None:
                out[i, h, :n + w] += s["before"][i, h, :n + w].double()
        at += w
    return out


def _exact_select(c, s):
    S, H, T = s["scores"].shape
    B = c["budget"]
    kept = torch.full((S, H, B), -1, dtype=torch.int32, device="cuda")
    moved = torch.zeros(S, H, T, dtype=torch.float64, device="cuda")
    count = torch.zeros(S, dtype=torch.int32, device="cuda")
    for i, n in enumerate(_lens(c)):
        count[i] = m = min(n, B)
        for h in range(H):
            ids = torch.arange(n, device="cuda")
            if n > B:
                first, last = ids[:c["sink"]], ids[n - c["recent"]:]
                mid = ids[c["sink"]:n - c["recent"]]
                v = s["scores"][i, h][mid].double()
                want = B - c["sink"] - c["recent"]
                if want:
                    edge = v.topk(want).values[-1]  # everything above it, then the first equal ones
                    above, equal = mid[v > edge], mid[v == edge]
                    mid = torch.cat([above, equal[:want - above.numel()]])
                ids = torch.cat([first, mid[:want], last]).sort().values
            kept[i, h, :m] = ids.int()
            moved[i, h, :m] = s["scores"][i, h][ids].double()
    return kept, count, moved


def _exact_compact(c, s):
    """Token by token through byte addresses of the whole pool."""
    pool, H = s["pool"].clone(), c["heads"]
    to = s["tables"] if s["out_tables"] is None else s["out_tables"]
    for i in range(c["seqs"]):
        for h in range(H):
            src = s["kept"][i, h].long()
            src = src[src >= 0]
            dst = torch.arange(src.numel(), device="cuda")
            for _, at, n in _fields(c):
                byte = torch.arange(n, device="cuda")

                def place(table, t):
                    return (table[i, t // PAGE].long() * _page_bytes(c) + at +
                            (t % PAGE * H + h) * n)[:, None] + byte

                pool[place(to, dst)] = s["pool"][place(s["tables"], src)]
    return pool.view(_DTYPES[c["dtype"]]).double() if c["scheme"] == "dense" else pool


def exact(case: dict, seed: int):
    c, s = case, prepare(case, seed)
    if c["kind"] == "weights":
        return _exact_weights(c, s)
    if c["kind"] == "select":
        return _exact_select(c, s)
    if c["kind"] == "compact":
        return _exact_compact(c, s)
    q, k = _exact_rope(s["q"], s["qw"], s, c), _exact_rope(s["k"], s["kw"], s, c)
    if c["kind"] == "rope":
        return q, k
    pages = torch.zeros(s["pages"].shape, dtype=torch.float64, device="cuda")
    flat = pages.transpose(0, 1).reshape(2, -1, c["heads"], c["dim"])  # [K or V, slot, H, D]
    flat[0].index_copy_(0, s["slots"].long(), k)
    flat[1].index_copy_(0, s["slots"].long(), s["v"].double())
    return q, flat.view(2, -1, PAGE, c["heads"], c["dim"]).transpose(0, 1).contiguous()
