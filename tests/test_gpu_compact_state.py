"""In-place compaction over a workspace that another call's kernels write over, as two
graphs of one stream do that are replayed at once against the rule: the state is forced
from the host (tq_test_compact), and nothing out of bounds is touched."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle.evict_oracle import compact
from test_gpu_evict import _compact, _kept
from test_gpu_tree import SCHEMES, Problem

pytestmark = pytest.mark.gpu


@pytest.fixture
def state(tq):
    f = tq.lib.tq_test_compact
    f.argtypes, f.restype = [ctypes.c_uint32], ctypes.c_int
    yield f
    f(0)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("first", [0x7FFFFFFF, 0x80000000, 0xFF800000, 0xFFFFF000, 100])
def test_tickets_out_of_range(tq, cuda, state, scheme, dtype, first):
    """Any bits (those of -infinity among them) where a row's tickets lie: a workgroup whose ticket
    names no chunk, above them all or below 0 as a signed number, moves nothing."""
    p = Problem(tq, scheme, dtype, [900, 700], [0, 0], 2, 2, 128, seed=61)
    kept = _kept(2, 2, [900, 700], 600, "random", seed=62)
    state(first)
    assert torch.equal(_compact(tq, cuda, p, kept), p.pool)
    state(0)
    assert torch.equal(_compact(tq, cuda, p, kept), compact(scheme, p.pool, p.tables, kept, p.layout, p.cfg))
