"""Attention weights of large logits where K is gone over twice: the statistics and
the weights take every logit for the same number, so that a row's weights add up to 1."""
from __future__ import annotations

import pytest
import torch

from test_gpu_tree import SCHEMES
from test_gpu_weights import Weights

pytestmark = pytest.mark.gpu

# A logit in powers of two, y, is one number per row and token.  A row's sum of 2^(y - M) over
# its tokens and its weights 2^(y - M) / sum then differ by roundings alone:
#   exponents: y - m and m - M in the sum (m a chunk's maximum; what lies between several maxima
#   adds up to m - M), y - M in the weight, by 2^-24 of the at most 32 at which a term counts:
#   3 * 32 * 2^-24 * ln 2 = 4.0e-6;
#   exponentials, off by 2^-23 each: 16 in a line of the sum's merges, one in the weight: 2.0e-6;
#   sums, at most 64 additions in a line over tokens, chunks and rows: 3.8e-6.
# Together 9.8e-6 of a row.  A logit that is rounded in one pass and not in the other moves its
# weight by up to 2^-24 |y| ln 2: 4.1e-3 at 1e5, 12% at 3e6.
TOLERANCE = 2e-5


def _weights(tq, scheme, dtype, lens, widths, y, **kw):
    """A row's largest |logit| is near y: 6 of 17,000 at keys and queries of size 1, by 1.3 more on
    compressed pages."""
    return Weights(tq, scheme, dtype, lens, widths, 8, 2, 128, before=False, kv_scale=256.0,
                   q_scale=y / 256 / 6, **kw)


def _rows_add_up(w, cuda):
    w.upload(cuda)
    w.call()
    torch.cuda.synchronize()
    rows = 4 * w.p.widths[0]
    end = int(w.p.prefix[0]) + (w.p.widths[0] if w.causal else 0)
    off = (w.out[0, :, :end].double().sum(1) / rows - 1).abs().max().item()
    print(f"    off by {off:.2e}", flush=True)
    assert off <= TOLERANCE


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("y", [1e3, 1e5, 1e6, 3e6, 1e7])
def test_rows_that_end_inside_a_tile(tq, cuda, scheme, dtype, y):
    """84 rows of a kv head, in tiles of 16: the last one has 12 that are none."""
    _rows_add_up(_weights(tq, scheme, dtype, [17000], [21], y, seed=101, causal=False), cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("y", [1e5, 1e6, 3e6])
def test_rows_that_see_nothing_of_a_chunk(tq, cuda, scheme, dtype, y):
    """The last chunk begins at a token that two of a tile's four see; its logits are the largest."""
    w = _weights(tq, scheme, dtype, [17142], [20], y / 8, seed=102)
    p = w.p
    page, B, H, D = int(p.layout.page_size_bytes), 16, 2, 128
    for t in range(17152, 17162):
        at, tib = int(p.tables[0, t // B]) * page, t % B
        if scheme == "dense":
            k = p.cell_bytes(0, t)[0]
            k = p.pool[k:k + H * 2 * D].view(dtype)
        else:
            off = int(p.layout.k_scales_offset if scheme == "turbo_prod" else p.layout.k_norms_offset)
            k = p.pool[at + off + tib * H * 2:at + off + (tib + 1) * H * 2].view(torch.float16)
        k *= 8
    _rows_add_up(w, cuda)


@pytest.mark.parametrize("scheme,dtype", SCHEMES)
@pytest.mark.parametrize("y", [1e6, 3.5e6, 6e6])
def test_rows_of_other_sizes_in_a_tile(tq, cuda, scheme, dtype, y):
    """Logits on both sides of 2^22, from where on they are rounded before their difference."""
    w = _weights(tq, scheme, dtype, [17000], [21], y, seed=103)
    w.p.query[:, ::2] *= 0.25
    w.p.query[::3] *= 0.5
    _rows_add_up(w, cuda)
