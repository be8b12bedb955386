"""The serving operators where their parts meet: items without key tiles, refused reservations, graphs, streams.

Values by the same 64-bit restatements and tolerances as test_text_gpu.py.
"""

from __future__ import annotations

import pytest
import torch

from test_text_gpu import cache, check, ints, pages_want, queries, starts_of

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- many rows: items without key tiles among others


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,hd", [(15, 5, 64), (8, 2, 128)])
@pytest.mark.parametrize(
    "lens", [[0] * 9 + [16384, 300], [16384] + [0] * 9 + [300] + [0] * 17 + [129], [640] + [0] * 700 + [70], [0] * 300]
)
def test_rows_of_empty_sequences(lens, heads, kv, hd, causal):
    """Runs of sequences that hold nothing, longer than a CTA's list of items, before, between and after others."""
    from so101_smolvla_edge_b200 import ops

    c = cache(lens, kv, hd, 64, seed=201)
    counts = [50] * len(lens)
    q = queries(sum(counts), heads, hd, seed=202)
    got = ops.attention_pages(q, c, 0, heads, starts_of(counts), max_q=50, causal=causal)
    assert ops.device_status() == 0
    check(got, *pages_want(q, c, 0, heads, counts, range(len(lens)), causal, hd**-0.5))


@pytest.mark.parametrize("hd", [64, 128])
def test_many_items_key_by_key(hd):
    """Sequences whose scales are no powers of two, more than a list of items of them on every CTA, others among them."""
    from so101_smolvla_edge_b200 import ops

    lens = [60 + (i * 37) % 70 for i in range(330)]
    c = cache(lens, 4, hd, 32, seed=211)
    for s in range(len(lens)):
        if s % 11:
            ids = c.table[s, : -(-lens[s] // 32)].long()
            c.v_scale[:, ids] *= 1.25
    counts = [30] * len(lens)
    q = queries(sum(counts), 12, hd, seed=212)
    got = ops.attention_pages(q, c, 0, 12, starts_of(counts), max_q=30)
    assert ops.device_status() == 0
    check(got, *pages_want(q, c, 0, 12, counts, range(len(lens)), True, hd**-0.5))
