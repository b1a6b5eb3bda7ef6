"""hipStreamPerThread: one handle, a stream of each host thread's.  Calls of several
threads run beside each other, each with a workspace of its own."""
from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from test_gpu_tree import Problem

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # hipStreamPerThread


def test_threads_on_their_own_streams(tq, cuda):
    trees = [Problem(tq, "dense", torch.float16, [30000, 900], [5, 9], 16, 2, 128, seed=91),
             Problem(tq, "turbo_prod", torch.float16, [9000], [40], 16, 2, 128, seed=92),
             Problem(tq, "turbo_mse", torch.float16, [7000] * 4, [6] * 4, 16, 2, 64, seed=93)]
    for p in trees:
        p.run(cuda)
    outs = [[torch.zeros_like(p.out) for _ in range(40)] for p in trees]
    torch.cuda.synchronize()

    def work(p, mine):
        for o in mine:
            tq.tree_attn_output(p.scheme, *p.gpu, o, p.layout, p.cfg, p.max_kv, stream=PER_THREAD)

    with ThreadPoolExecutor(3) as pool:
        for f in [pool.submit(work, p, mine) for p, mine in zip(trees, outs)]:
            f.result()
        torch.cuda.synchronize()
    for p, mine in zip(trees, outs):
        assert all(torch.equal(o, p.out) for o in mine)
    tq.release_workspaces()
