"""Attention over the 8-bit pages for many rows per sequence (a chunk, the rest of a prompt), against the same
64-bit restatement and by the same tolerances as the few-row cases of test_text_gpu.py.

The rounding points are the same (q and P to f16, the result to bf16). Where parts of a long sequence are
joined, a part's weight is the exponential of a sum of the maximum and a logarithm, both fp32: |m| below 2^8
here, so 2^-16 of a weight, inside the 5%.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_text_gpu import cache, check, ints, pages_want, queries, rope, starts_of

pytestmark = pytest.mark.gpu


def run(c, q, heads, counts, seqs, causal=True, layer=0, **kw):
    from so101_smolvla_edge_b200 import ops

    return ops.attention_pages(
        q, c, layer, heads, starts_of(counts), ints(list(seqs)), max_q=max(counts), causal=causal, **kw
    )


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,heads,kv,hd", [(64, 15, 5, 64), (16, 3, 1, 64), (32, 8, 2, 128), (64, 3, 3, 128)])
def test_ragged(causal, page, heads, kv, hd):
    """Rows around every tile edge, lengths around every key tile's, an empty sequence, sequences with
    fewer tokens than rows, none, and one with a single row; queries rotated; a second layer."""
    lens = [128, 127, 129, 300, 0, 1, 640, 90, 257, 200]
    counts = [128, 43, 86, 200, 66, 70, 100, 0, 1, 257]
    seqs = [0, 2, 1, 3, 4, 5, 6, 7, 8, 9]
    c = cache(lens, kv, hd, page, layers=2, seed=41)
    q = queries(sum(counts), heads, hd, seed=42)
    cos, sin = rope(torch.arange(sum(counts)) % 500, hd)
    got = run(c, q, heads, counts, seqs, causal, layer=1, cos=cos, sin=sin, scale=0.15)
    want, tol = pages_want(q, c, 1, heads, counts, seqs, causal, 0.15, cos, sin)
    check(got, want, tol)
    at = sum(counts[:4])
    assert (got[at : at + 66] == 0).all()  # nothing cached
    if causal:
        assert (got[at + 66 : at + 66 + 69] == 0).all()  # one token cached: only the last row sees it
    from so101_smolvla_edge_b200 import ops

    assert ops.device_status() == 0


@pytest.mark.parametrize("lens,counts", [([9000], [300]), ([4000, 70, 2500], [50, 70, 150]), ([3000] * 40, [65] * 40)])
@pytest.mark.parametrize("heads,kv,hd", [(6, 2, 64), (8, 2, 128)])
def test_parts(lens, counts, heads, kv, hd):
    """Sequences that several CTAs share; repeatable; peaked scores."""
    c = cache(lens, kv, hd, 64, seed=51)
    q = queries(sum(counts), heads, hd, seed=52, big=4.0)
    got = run(c, q, heads, counts, range(len(lens)))
    check(got, *pages_want(q, c, 0, heads, counts, range(len(lens)), True, hd**-0.5))
    for _ in range(3):
        assert torch.equal(got, run(c, q, heads, counts, range(len(lens))))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("spread", [20, 32, 60])
def test_scales_far_apart(hd, spread):
    """Pages whose value scales are up to 2^60 apart, the large ones where only later rows see them, and
    pages of zeros (the smallest scale) among them: each row to its own tolerance."""
    lens, counts = [700, 260], [640, 100]
    c = cache(lens, 2, hd, 64, seed=61)
    for s in range(2):
        for p in range(-(-lens[s] // 64)):
            id = int(c.table[s, p])
            c.v_scale[0, id] = 2.0 ** -(10 + (spread if p % 3 == 0 else 0))
            c.k_scale[0, id] = 2.0 ** (-5 - p % 4)
            if p == 1:
                c.v[0, id], c.v_scale[0, id] = 0, 2.0**-126
    q = queries(sum(counts), 6, hd, seed=62)
    got = run(c, q, 6, counts, range(2))
    check(got, *pages_want(q, c, 0, 6, counts, range(2), True, hd**-0.5))


def test_scales_that_are_no_powers_of_two():
    """A cache that another program filled: any scale is read as it is."""
    c = cache([500], 2, 64, 32, seed=71)
    c.k_scale *= 1.3
    c.v_scale *= 0.7
    q = queries(100, 6, 64, seed=72)
    got = run(c, q, 6, [100], [0])
    check(got, *pages_want(q, c, 0, 6, [100], [0], True, 0.125))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_lost_page(hd, which):
    """A page whose scale is NaN: rows that do not see it are as if it were not there."""
    c = cache([400], 1, hd, 64, seed=81)
    q = queries(300, 4, hd, seed=82)
    want, tol = pages_want(q, c, 0, 4, [300], [0], True, hd**-0.5)
    getattr(c, which)[0, int(c.table[0, 4])] = math.nan  # tokens 256 on: rows 156 on
    got = run(c, q, 4, [300], [0])
    check(got[:156], want[:156], tol[:156])
    assert got[156:].isnan().all()


def test_queries_not_finite_and_zero():
    """A row of NaN is NaN, alone; a row of zeros weighs its keys alike."""
    c = cache([400], 1, 64, 64, seed=91)
    q = queries(100, 4, 64, seed=92).clone()
    q[17] = 0
    want, tol = pages_want(q, c, 0, 4, [100], [0], False, 0.125)
    q[40, :64] = math.nan
    got = run(c, q, 4, [100], [0], causal=False)
    rows = torch.arange(100, device="cuda") != 40
    check(got[rows], want[rows], tol[rows])
    check(got[40:41, 64:], want[40:41, 64:], tol[40:41, 64:])
    assert got[40, :64].isnan().all()


@pytest.mark.parametrize("group", [1, 7, 65, 200])
def test_groups(group):
    """Heads per kv head that do not divide a row tile."""
    c = cache([150, 80], 1, 64, 16, seed=101)
    counts = [80, 70]
    q = queries(150, group, 64, seed=102)
    got = run(c, q, group, counts, range(2))
    check(got, *pages_want(q, c, 0, group, counts, range(2), True, 0.125))


def test_rows_at_eight_bytes_and_graph():
    """An output whose rows start on 8 bytes only; the launch replayed from a graph with other data."""
    from so101_smolvla_edge_b200 import ops

    c = cache([300, 290], 2, 64, 64, seed=111)
    counts, st, sq = [90, 120], starts_of([90, 120]), ints([0, 1])
    q = queries(210, 6, 64, seed=112)
    wide = torch.zeros(210, 6 * 64 + 4, device="cuda", dtype=torch.bfloat16)
    out = wide[:, 4:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.attention_pages(q, c, 0, 6, st, sq, max_q=120, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.attention_pages(q, c, 0, 6, st, sq, max_q=120, out=out)
    torch.cuda.current_stream().wait_stream(s)
    q.copy_(queries(210, 6, 64, seed=113))
    out.zero_()
    g.replay()
    check(out, *pages_want(q, c, 0, 6, counts, range(2), True, 0.125))
    assert (wide[:, :4] == 0).all()


@pytest.mark.parametrize("rows,heads", [(66, 1), (1, 3), (13, 2)])
def test_long_lists(rows, heads):
    """More sequences than a CTA's threads look at in one pass, some empty, one long among them."""
    lens = [(37 * i) % 90 for i in range(1000)]
    lens[700] = 3000
    counts = [rows if i % 7 else 0 for i in range(1000)] if rows > 1 else [1] * 1000
    c = cache(lens, 1, 64, 16, seed=121)
    q = queries(sum(counts), heads, 64, seed=122)
    got = run(c, q, heads, counts, range(1000))
    check(got, *pages_want(q, c, 0, heads, counts, range(1000), True, 0.125))
