"""Batched paged decode with append-quantize (a serving step over many
sequences), on the library's allocator, block table, pack and paged
attention entry points.

A ``PagedBatch`` holds S sequences in one page pool.  Pages come from the
library's LIFO allocator; the prefill is appended page by page in a seeded
random order of sequences, so every sequence's pages are scattered over the
pool.  One ``step`` appends w_s new tokens to every sequence (one pack
launch over all of them, slots from the block table) and runs decode
attention for 8 GQA rows per new token (one paged-attention launch), the
rows of new token j attending L_s + j + 1 tokens (causal over the new
tokens).  The reference does the same work with one pack call per sequence
and one fused_attention_output call per sequence and position, each with a
per-token slot map (tq_backend/turboquant_wrapper.py; the C5 serving
configuration).  The new tokens may also form trees (``tree_attention``): a
row then attends the prefix and the new tokens of its mask, not all before it.
``add_weights`` and ``evict`` keep the caches to a budget: the scores that the
steps' attention weights add up to choose the tokens that stay.
"""
from __future__ import annotations

import numpy as np
import torch

from turborag_amd.synthetic import fisher_yates, gqa_rows, kv_tokens_major
from turborag_amd.synthetic import query as draw_query
from turborag_amd.turboquant_wrapper import BlockTable, PageAllocator, TurboQuantWrapper


class PagedBatch:
    def __init__(self, tq: TurboQuantWrapper, scheme: str, lens, widths, *, kv_heads: int = 2,
                 q_heads: int = 16, head_dim: int = 128, block_size: int = 16, seed: int = 500,
                 device: torch.device | None = None, capacity: int = 0) -> None:
        """lens cached tokens and widths new ones of every sequence.  capacity: the tokens that a
        sequence may come to hold (a budget and a step's new tokens), for which there are pages;
        otherwise, for those of the first step and a page more for each."""
        self.tq, self.scheme = tq, scheme
        self.dev = device or torch.device("cuda", 0)
        self.lens = [int(x) for x in lens]
        self.widths = [int(x) for x in widths]
        self.S = len(self.lens)
        self.H, self.D, self.B = kv_heads, head_dim, block_size
        self.group = q_heads // kv_heads  # GQA rows per kv head and token
        cfg = tq.default_config()
        cfg.num_kv_heads, cfg.head_dim, cfg.block_size = kv_heads, head_dim, block_size
        self.cfg = cfg
        self.prod = scheme == "turbo_prod"
        self.layout = tq.make_layout_for(cfg) if self.prod else tq.make_mse_layout_for(cfg)
        B = block_size
        most = [max(L + w, capacity) for L, w in zip(self.lens, self.widths)]
        pages = sum(self._pages(n) for n in most) + self.S
        self.pool = torch.zeros(pages * self.layout.page_size_bytes, dtype=torch.uint8,
                                device=self.dev)
        self.alloc = PageAllocator(tq, self.layout.page_size_bytes, pages, device_pool=self.pool)
        self.table = BlockTable(self.alloc, B)
        self.max_blocks = max(self._pages(n) for n in most)
        self.seed = seed
        self._prefill()

    # ── helpers ─────────────────────────────────────────────────────── #

    def _held(self, s: int) -> int:
        """Tokens that the block table holds of sequence s."""
        try:
            return self.table.num_tokens(s)
        except KeyError:  # none so far
            return 0

    def _pages(self, tokens: int) -> int:
        return (tokens + self.B - 1) // self.B

    def _pack(self, k: torch.Tensor, v: torch.Tensor, slots: list[int]) -> None:
        self._last_pack = (k.to(self.dev), v.to(self.dev),
                           torch.tensor(slots, dtype=torch.int32, device=self.dev))
        self.repack()

    def repack(self, stream: int = 0) -> None:
        """Issue the last pack launch again (same tokens into the same slots:
        idempotent), e.g. to time the append of a step.  Not after an eviction of
        any token: others lie in those slots then, or their pages are given back."""
        if self._last_pack is None:
            raise RuntimeError("repack: the last append's tokens have been moved by evict")
        k, v, s = self._last_pack
        (self.tq.pack if self.prod else self.tq.mse_pack)(k, v, s, self.pool, self.layout,
                                                          self.cfg, stream=stream)

    def _prefill(self) -> None:
        """Every sequence's first L_s tokens, appended one page at a time in a
        seeded random order of sequences (scattered pages)."""
        self.kv = [kv_tokens_major(L, self.H, self.D, seed=self.seed + 3 + s)
                   for s, L in enumerate(self.lens)]
        pages = []
        for s, L in enumerate(self.lens):
            pages += [s] * ((L + self.B - 1) // self.B)
        todo = [pages[i] for i in fisher_yates(len(pages), self.seed + 2)]
        done = [0] * self.S
        keys, vals, slots = [], [], []
        for s in todo:
            n = min(self.B, self.lens[s] - done[s])
            slots += self.table.build_slot_map(s, n)
            keys.append(self.kv[s][0][done[s]:done[s] + n])
            vals.append(self.kv[s][1][done[s]:done[s] + n])
            done[s] += n
        self._pack(torch.cat(keys), torch.cat(vals), slots)

    def block_tables(self) -> torch.Tensor:
        """[S, max_blocks], or wider where a sequence has more pages by now; -1 behind them."""
        blocks = [self.table.blocks(s) for s in range(self.S)]
        bt = torch.full((self.S, max(self.max_blocks, *map(len, blocks))), -1, dtype=torch.int32)
        for s, b in enumerate(blocks):
            bt[s, :len(b)] = torch.tensor(b, dtype=torch.int32)
        return bt.to(self.dev)

    def slots_of(self, s: int, n: int) -> np.ndarray:
        """The first n tokens' slots of sequence s (page * B + position)."""
        b = np.asarray(self.table.blocks(s), dtype=np.int64)
        t = np.arange(n)
        return (b[t // self.B] * self.B + t % self.B).astype(np.int32)

    # ── one serving step ───────────────────────────────────────────── #

    def append_new_tokens(self, seed: int) -> tuple[list, list]:
        """w_s new tokens per sequence, quantized into (newly allocated)
        pages with one pack launch; returns the new K/V per sequence.  Refused,
        with nothing appended, where the pool has not the pages."""
        need = sum(self._pages(self._held(s) + w) - self._pages(self._held(s)) for s, w in enumerate(self.widths))
        if need > self.alloc.num_free():
            raise RuntimeError(f"append_new_tokens: out of blocks, {need} pages are needed, {self.alloc.num_free()} "
                               "are free (capacity: tokens that a sequence may come to hold)")
        keys, vals, slots, new = [], [], [], []
        for s, w in enumerate(self.widths):
            k, v = kv_tokens_major(w, self.H, self.D, seed=seed + s)
            slots += self.table.build_slot_map(s, w)
            keys.append(k)
            vals.append(v)
            new.append((k, v))
        self._pack(torch.cat(keys), torch.cat(vals), slots)
        return new

    def decode_rows(self, seed: int):
        """Query rows of the step: for sequence s and new token j, the 8 GQA
        rows of every kv head ([8, H, D]), attending L_s + j + 1 tokens."""
        q, row_seq, row_len = [], [], []
        for s, (L, w) in enumerate(zip(self.lens, self.widths)):
            for j in range(w):
                qh = draw_query(self.group * self.H, self.D, seed=seed + 1000 * s + j)
                q.append(gqa_rows(qh, self.H))
                row_seq += [s] * self.group
                row_len += [L + j + 1] * self.group
        query = torch.cat(q).contiguous().to(self.dev)
        return (query, torch.tensor(row_seq, dtype=torch.int32, device=self.dev),
                torch.tensor(row_len, dtype=torch.int32, device=self.dev))

    def attention(self, query, row_seq, row_len, block_tables, out, stream: int = 0) -> None:
        self.tq.paged_attn_output(self.scheme, query, self.pool, block_tables, row_seq, row_len,
                                  out, self.layout, self.cfg,
                                  max(L + w for L, w in zip(self.lens, self.widths)), stream)

    def tree_rows(self):
        """The sequences' new tokens as trees of drafted tokens: (row_start,
        prefix_len) of tree_attention."""
        start = np.concatenate([[0], np.cumsum(self.widths)])
        return (torch.tensor(start, dtype=torch.int32, device=self.dev),
                torch.tensor(self.lens, dtype=torch.int32, device=self.dev))

    def tree_attention(self, query, row_start, prefix_len, tree_mask, block_tables, out,
                       stream: int = 0) -> None:
        """Attention of the appended tokens as trees: query / out [sum of widths,
        query heads, D], tree_mask their bits (tree_mask_from_parents)."""
        self.tq.tree_attn_output(self.scheme, query, self.pool, block_tables, row_start, prefix_len,
                                 tree_mask, out, self.layout, self.cfg,
                                 max(L + w for L, w in zip(self.lens, self.widths)), stream)

    # ── eviction ───────────────────────────────────────────────────── #

    def add_weights(self, query, row_start, prefix_len, block_tables, scores, decay: float = 1.0,
                    stream: int = 0) -> None:
        """Adds the weights that the appended tokens' rows (tree_rows, query
        [sum of widths, query heads, D]) give to every cached token up to their own
        to scores [S, H, tokens]."""
        self.tq.attn_weights(self.scheme, query, self.pool, block_tables, row_start, prefix_len, scores,
                             self.layout, self.cfg, max(L + w for L, w in zip(self.lens, self.widths)),
                             scores_in=scores, decay=decay, stream=stream)

    def evict(self, scores, budget: int, block_tables, sink: int = 4, recent: int = 32, new_widths=None,
              stream: int = 0) -> list[int]:
        """Cuts every sequence to at most `budget` tokens (its first `sink`, last
        `recent` and highest scores): cells and scores are moved to the front, and
        the pages behind go back to the allocator.  The sequences' tokens are those
        that their block tables hold; new_widths: the new tokens of the next step,
        refused where the pool has not the pages.  Returns their lengths.  Positions
        go on from the tokens ever appended, not from what is left.  (On another
        stream: an append, which stores on the default one, waits for it first.)"""
        held = [self._held(s) for s in range(self.S)]
        if max(held) > scores.shape[-1] or max(held) > block_tables.shape[-1] * self.B:
            raise ValueError(f"evict: scores and block_tables must hold {max(held)} tokens")
        left = [min(n, budget) for n in held]
        if new_widths is not None:
            new_widths = [int(x) for x in new_widths]
            if len(new_widths) != self.S or min(new_widths) < 0:
                raise ValueError(f"evict: new_widths must be {self.S} widths >= 0")
            need = sum(self._pages(n + w) for n, w in zip(left, new_widths))
            if need > self.alloc.num_pages:
                raise ValueError(f"evict: new_widths need {need} pages, the pool has {self.alloc.num_pages}")
        # (allocated for the stream that uses them: their memory is given back on it)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.dev) if stream
                               else torch.cuda.default_stream(self.dev)):
            kept = torch.empty(self.S, self.H, budget, dtype=torch.int32, device=self.dev)
            lens = torch.tensor(held, dtype=torch.int32, device=self.dev)
            self.tq._compact_checks(self.scheme, self.pool, block_tables, kept, self.cfg)  # before scores move
            self.tq.select_kv(scores, lens, kept, sink=sink, recent=recent, out_scores=scores,
                              stream=stream)
            self.tq.compact_kv(self.scheme, self.pool, block_tables, kept, self.layout, self.cfg,
                               stream=stream)
        if left != held:
            self._last_pack = None
        self.lens = left
        for s, n in enumerate(self.lens):
            if n < held[s]:
                self.table.truncate(s, n)
        if new_widths is not None:
            self.widths = new_widths
        return list(self.lens)

    def close(self) -> None:
        self.table.close()
        self.alloc.close()
