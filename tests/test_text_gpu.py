"""Packed-prompt attention and the 8-bit paged cache against 64-bit restatements of their formulas.

Tolerances, per output value, come from where the kernels round (A = sum_j w_j |v_j| with the exact
weights w, S = scale * sum_d |q_d k_d| maximised over the visible keys):

    P rounded to bf16 (packed) or f16 (pages)   2^-8 A or 2^-11 A
    the result rounded to bf16                  2^-8 A
    q rounded after its rotation (packed, bf16) or to f16 (pages): logits off by d <= S 2^-8 or
    S 2^-11, fp32 sums of hd products by S hd 2^-23: weights off by at most expm1(2 d), so expm1(2 d) A

(half an ulp is 2^-8 of a bf16 value, 2^-11 of an f16 one at most), with 5% on top for the products of those. Codes, scales, tables, lengths and counts are equal.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts_of(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return ints(s)


def rope(pos, hd):
    inv = 10000.0 ** (-torch.arange(0, hd // 2, device="cuda") * 2.0 / hd)
    a = torch.as_tensor(pos, device="cuda").float()[:, None] * inv
    return torch.cos(a), torch.sin(a)


def turn(x, cos, sin):
    """x (rows, heads, hd) rotated in its own precision, each operation rounded."""
    a, b = x.chunk(2, -1)
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attend(q, k, v, last, scale, round_q, round_p):
    """One head in 64 bits, row i over keys 0..last[i]: (out, tolerance)."""
    q, k, v = q.double(), k.double(), v.double()
    hide = torch.arange(k.shape[0], device=q.device)[None] > last[:, None]
    # a key that no row sees may hold anything
    k = torch.where((~hide).any(0)[:, None], k, 0.0)
    v = torch.where((~hide).any(0)[:, None], v, 0.0)
    s = (q @ k.T * scale).masked_fill(hide, -math.inf)
    w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    size = (q.abs() @ k.abs().T * scale).masked_fill(hide, 0.0).amax(-1, keepdim=True) if k.shape[0] else 0.0
    d = size * (round_q + q.shape[1] * 2**-23)
    a = w @ v.abs()
    return w @ v, 1.05 * a * (round_p + 2**-8 + torch.expm1(2 * d)) + 1e-30


def check(got, want, tol):
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - tol
    assert over.max() <= 0, float(over.max())


# ------------------------------------------------------------------------------------- packed prompts


def packed_case(lens, heads, kv, hd, seed=0, big=1.0, tail=0):
    rows = sum(lens) + tail
    x = torch.randn(rows, (heads + 2 * kv) * hd, device="cuda", generator=gen(seed)).to(torch.bfloat16)
    x[:, : heads * hd] *= big
    return x[:, : heads * hd], x[:, heads * hd : (heads + kv) * hd], x[:, (heads + kv) * hd :]


def packed_want(q, k, v, lens, heads, kv, hd, scale, cos, sin):
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    qr = q.double().reshape(-1, heads, hd)
    if cos is not None:
        qr = turn(qr, cos, sin)
    at = 0
    for n in lens:
        for h in range(heads):
            g = h // (heads // kv)
            sl = slice(at, at + n)
            if n:
                o, t = attend(qr[sl, h], k[sl, g * hd : (g + 1) * hd], v[sl, g * hd : (g + 1) * hd],
                              torch.arange(n, device="cuda"), scale, 2**-8 if cos is not None else 0.0, 2**-8)  # fmt: skip
                out[sl, h * hd : (h + 1) * hd], tol[sl, h * hd : (h + 1) * hd] = o, t
        at += n
    return out, tol


@pytest.mark.parametrize("heads,kv,hd", [(15, 5, 64), (4, 4, 64), (7, 1, 64), (8, 2, 128), (16, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1, 0], [127, 128, 129], [241], [1] * 70, [5, 700, 64, 33]])
def test_packed(lens, heads, kv, hd):
    from so101_smolvla_edge_b200 import ops

    q, k, v = packed_case(lens, heads, kv, hd, seed=sum(lens))
    got = ops.attention_packed(q, k, v, starts_of(lens), max(lens), heads, kv)
    check(got, *packed_want(q, k, v, lens, heads, kv, hd, hd**-0.5, None, None))
    assert torch.equal(got, ops.attention_packed(q, k, v, starts_of(lens), max(lens), heads, kv))
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads,kv,hd", [(15, 5, 64), (8, 2, 128)])
def test_packed_rope_scale_and_rows_outside(heads, kv, hd):
    """Rotated queries, another scale, rows past the last sequence left alone."""
    from so101_smolvla_edge_b200 import ops

    lens = [30, 300]
    q, k, v = packed_case(lens, heads, kv, hd, seed=3, tail=9)
    cos, sin = rope(torch.cat([torch.arange(n) for n in lens] + [torch.zeros(9)]), hd)
    out = torch.full((339, heads * hd), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attention_packed(q, k, v, starts_of(lens), 300, heads, kv, cos=cos, sin=sin, scale=0.3, out=out)
    want, tol = packed_want(q, k, v, lens, heads, kv, hd, 0.3, cos, sin)
    check(out[:330], want[:330], tol[:330])
    assert (out[330:] == 7.0).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_long_and_peaked(hd):
    """Several thousand keys; scores of hundreds, so that the running maximum moves far."""
    from so101_smolvla_edge_b200 import ops

    lens = [2113]
    q, k, v = packed_case(lens, 4, 2, hd, seed=5, big=32.0)
    got = ops.attention_packed(q, k, v, starts_of(lens), 2113, 4, 2)
    check(got, *packed_want(q, k, v, lens, 4, 2, hd, hd**-0.5, None, None))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_packed_values_that_a_row_must_not_see(hd, bad):
    """NaN and infinities in later tokens, in another sequence and past the last one."""
    from so101_smolvla_edge_b200 import ops

    lens = [150, 90]
    q, k, v = (t.clone() for t in packed_case(lens, 6, 2, hd, seed=6, tail=40))
    want, tol = packed_want(q, k, v, lens, 6, 2, hd, hd**-0.5, None, None)
    for t in (k, v):
        t[100] = bad  # rows 0..99 of the first sequence must not see it
        t[200] = bad  # rows 150..199 of the second
        t[240:] = bad
    got = ops.attention_packed(q, k, v, starts_of(lens), 150, 6, 2)
    fine = [*range(100), *range(150, 200)]
    check(got[fine], want[fine], tol[fine])
    assert not torch.isfinite(got[100:150].float()).all(1).any()
    assert not torch.isfinite(got[200:240].float()).all(1).any()


def test_packed_refusals():
    from so101_smolvla_edge_b200 import ops

    q, k, v = packed_case([20], 4, 2, 64)
    st = starts_of([20])
    with pytest.raises(ValueError):
        ops.attention_packed(q.float(), k, v, st, 20, 4, 2)
    with pytest.raises(ValueError):
        ops.attention_packed(q[:, :192], k, v, st, 20, 4, 2)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k[:, :96], v[:, :96], st, 20, 4, 2)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k, v, st.long(), 20, 4, 2)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k, v, st, 20, 4, 2, scale=0.0)
    with pytest.raises(ValueError):
        ops.attention_packed(q, k, v, st, 20, 4, 2, cos=torch.zeros(20, 32, device="cuda"))
    with pytest.raises(ValueError):
        ops.attention_packed(q.cpu(), k, v, st, 20, 4, 2)
    assert ops.attention_packed(q[:0], k[:0], v[:0], starts_of([0]), 1, 4, 2).shape == (0, 256)


# ------------------------------------------------------------------------------------- the paged cache


def cache(lens, kv, hd, page, layers=1, seed=0, spare=5, seqs=None):
    """A cache in use: pages out of order, junk in unused slots, NaN scales in unused pages."""
    from so101_smolvla_edge_b200.pages import KvPages

    g = gen(seed)
    need = [-(-n // page) for n in lens]
    pool = sum(need) + spare
    c = KvPages(layers, pool, kv, hd, seqs or len(lens), max(max(lens), 1), page)
    c.k.copy_(torch.randint(-127, 128, c.k.shape, device="cuda", generator=g, dtype=torch.int8))
    c.v.copy_(torch.randint(-127, 128, c.v.shape, device="cuda", generator=g, dtype=torch.int8))
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    used = []
    for i, n in enumerate(need):
        ids, order = order[:n], order[n:]
        used += ids
        c.table[i, :n] = ints(ids)
        c.lengths[i] = lens[i]
    for s in (c.k_scale, c.v_scale):
        s.fill_(math.nan)
        s[:, used] = 2.0 ** torch.randint(-8, -4, (layers, len(used), kv), device="cuda", generator=g).float()
    c.refs[used] = 1
    return c


def rows_of(c, layer, seq, which):
    """A sequence's cached keys or values, (tokens, kv, hd) in 64 bits."""
    n = int(c.lengths[seq])
    ids = c.table[seq, : -(-n // c.page)].long()
    codes, scale = (c.k, c.k_scale) if which == "k" else (c.v, c.v_scale)
    x = codes[layer][ids].double() * scale[layer][ids].double()[..., None, None]
    return x.transpose(1, 2).reshape(-1, c.n_kv, c.head_dim)[:n]


def pages_want(q, c, layer, heads, counts, seqs, causal, scale, cos=None, sin=None):
    hd, group = c.head_dim, heads // c.n_kv
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    qr = q.double().reshape(-1, heads, hd)
    if cos is not None:
        qr = turn(qr, cos, sin)
    at = 0
    for i, m in enumerate(counts):
        k, v = (rows_of(c, layer, seqs[i], w) for w in "kv")
        n = k.shape[0]
        last = torch.arange(n - m, n, device="cuda") if causal else torch.full((m,), n - 1, device="cuda")
        for h in range(heads):
            sl = slice(at, at + m)
            if n and m:
                o, t = attend(qr[sl, h], k[:, h // group], v[:, h // group], last, scale, 2**-11 + 2**-20, 2**-11)
                out[sl, h * hd : (h + 1) * hd], tol[sl, h * hd : (h + 1) * hd] = o, t
        at += m
    return out, tol


def queries(rows, heads, hd, seed=1, big=1.0):
    x = torch.randn(rows, heads * hd + 64, device="cuda", generator=gen(seed)).to(torch.bfloat16) * big
    return x[:, : heads * hd]


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 300, 1025]


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv,hd", [(15, 5, 64), (2, 2, 64), (8, 1, 128), (20, 1, 64), (40, 1, 128)])
def test_pages_single_tokens(page, heads, kv, hd):
    from so101_smolvla_edge_b200 import ops

    c = cache(LENS, kv, hd, page, layers=2, seed=page)
    q = queries(len(LENS), heads, hd)
    got = ops.attention_pages(q, c, 1, heads)
    check(got, *pages_want(q, c, 1, heads, [1] * len(LENS), range(len(LENS)), True, hd**-0.5))
    assert (got[0] == 0).all()
    assert torch.equal(got, ops.attention_pages(q, c, 1, heads))
    assert ops.device_status() == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("page,heads,kv,hd", [(64, 15, 5, 64), (16, 6, 2, 64), (32, 8, 2, 128), (64, 3, 3, 128)])
def test_pages_several_tokens(causal, page, heads, kv, hd):
    """Rows per sequence from none to more than one CTA's tile, in another order than the cache's; a
    sequence with fewer tokens than rows (its first rows see nothing)."""
    from so101_smolvla_edge_b200 import ops

    lens = [64, 3, 700, 291, 0, 130]
    counts, seqs = [5, 50, 0, 7, 1, 70], [2, 3, 0, 1, 4, 5]
    c = cache(lens, kv, hd, page, seed=11)
    q = queries(sum(counts), heads, hd, seed=12)
    cos, sin = rope(torch.arange(sum(counts)) % 300, hd)
    got = ops.attention_pages(q, c, 0, heads, starts_of(counts), ints(seqs), max_q=70, causal=causal, cos=cos, sin=sin, scale=0.2)
    want, tol = pages_want(q, c, 0, heads, counts, seqs, causal, 0.2, cos, sin)
    check(got, want, tol)
    if causal:  # sequence 1 has 3 tokens and 7 rows: rows 0..3 see nothing
        assert (got[55:59] == 0).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("hd,heads,kv", [(64, 15, 5), (128, 8, 1)])
def test_pages_long(hd, heads, kv):
    """Sequences long enough to be read in parts, beside short ones; repeatable; peaked scores."""
    from so101_smolvla_edge_b200 import ops

    lens = [20011, 7, 5000]
    c = cache(lens, kv, hd, 64, seed=21)
    q = queries(3, heads, hd, seed=22, big=8.0)
    got = ops.attention_pages(q, c, 0, heads)
    check(got, *pages_want(q, c, 0, heads, [1] * 3, range(3), True, hd**-0.5))
    for _ in range(3):
        assert torch.equal(got, ops.attention_pages(q, c, 0, heads))


def test_pages_scale_lost_in_a_page_that_a_row_does_not_see():
    from so101_smolvla_edge_b200 import ops

    c = cache([130], 2, 64, 64, seed=31)
    q = queries(4, 6, 64, seed=32)
    want, tol = pages_want(q, c, 0, 6, [4], [0], True, 0.125)
    for s in (c.k_scale, c.v_scale):
        s[0, int(c.table[0, 2])] = math.nan  # tokens 128, 129: rows 2 and 3
    got = ops.attention_pages(q, c, 0, 6, starts_of([4]), max_q=4)
    check(got[:2], want[:2], tol[:2])
    assert got[2:].isnan().all()


def test_pages_past_32_bits():
    """The last pages of a cache of more than 2^32 codes."""
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.pages import KvPages

    kv, hd, page, pool = 8, 128, 64, 66000
    c = KvPages(1, pool, kv, hd, 2, 256, page)
    assert c.k.numel() > 2**32
    c.table[1] = ints([pool - 1, 3, pool - 2, pool - 3])
    c.refs[c.table[1].long()] = 1
    c.lengths[1] = 200
    x = torch.randn(200, 2 * kv * hd, device="cuda", generator=gen(41)).to(torch.bfloat16)
    ops.kv_append(c, 0, x[:, : kv * hd], x[:, kv * hd :], starts_of([200]), ints([1]), max_new=200)
    k, v = ops.kv_read(c, 0, starts_of([200]), 200, ints([1]))
    for got, want in ((k, x[:, : kv * hd]), (v, x[:, kv * hd :])):
        step = 2.0 ** math.ceil(math.log2(float(want.abs().max()) / 127))
        assert (got.float() - want.float()).abs().max() <= step / 2
    q = queries(1, 16, hd, seed=42)
    got = ops.attention_pages(q, c, 0, 16, None, ints([1]))
    check(got, *pages_want(q, c, 0, 16, [1], [1], True, hd**-0.5))
    ops.kv_compact(c)
    assert c.table[1].tolist() == [2, 3, 1, 0]
    assert torch.equal(got, ops.attention_pages(q, c, 0, 16, None, ints([1])))
    assert ops.device_status() == 0


# -------------------------------------------------------------------------------------------- appending


def step_of(amax):
    """The smallest power of two s with amax <= 127 s, from 2^-126 to 2^121, in exact arithmetic."""
    if not math.isfinite(amax):
        return math.nan
    m, e = math.frexp(amax)
    return 2.0 ** min(max(e - 7 + (1 if m > 127 / 128 else 0), -126), 121) if amax else 2.0**-126


def append_model(c, layer, x, counts, seqs, which):
    """The codes and scales after an append of x (rows, kv, hd in fp32), page by page."""
    codes = (c.k if which == "k" else c.v)[layer].cpu().clone()
    scale = (c.k_scale if which == "k" else c.v_scale)[layer].cpu().clone()
    table, lengths, x = c.table.cpu(), c.lengths.cpu(), x.double().cpu()
    seen = torch.zeros(codes.shape[0], c.page, dtype=torch.bool)
    at = 0
    for m, s in zip(counts, seqs):
        n = int(lengths[s])
        for p in range((n - m) // c.page, -(-n // c.page)):
            lo, hi = max(n - m, p * c.page), min(n, (p + 1) * c.page)
            held, id = lo - p * c.page, int(table[s, p])
            if hi <= lo:
                continue
            new = x[at + lo - (n - m) : at + hi - (n - m)]
            seen[id, : held + hi - lo] = True
            for h in range(c.n_kv):
                was = float(scale[id, h]) if held else 0.0
                st = max(was, step_of(float(new[:, h].abs().max()))) if was == was else math.nan
                scale[id, h] = st
                codes[id, h, :held] = torch.round(codes[id, h, :held].double() * (was / st)).to(torch.int8)
                codes[id, h, held : held + hi - lo] = torch.round(new[:, h] / st).clamp(-127, 127).to(torch.int8)
        at += m
    return codes, scale, seen


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("page,kv,hd", [(16, 2, 64), (32, 3, 128), (64, 5, 64), (64, 1, 128)])
def test_append(page, kv, hd, turned):
    """New tokens across page ends, into part-filled pages with smaller and larger scales, into none."""
    from so101_smolvla_edge_b200 import ops

    counts, seqs = [1, 200, 0, 3, page, 40], [4, 0, 1, 5, 2, 3]
    lens = [230, 5, 2 * page, 40, 17, page + 3]  # by sequence; seqs[i] takes its last counts[i] tokens
    c = cache(lens, kv, hd, page, layers=2, seed=51)
    rows = sum(counts)
    x = torch.randn(rows, 2 * kv * hd, device="cuda", generator=gen(52)) * torch.logspace(-3, 2, rows, device="cuda")[:, None]
    x = x.to(torch.bfloat16)
    k, v = x[:, : kv * hd], x[:, kv * hd :]
    cos, sin = rope(torch.arange(rows) * 3, hd) if turned else (None, None)
    kx = k.float().reshape(rows, kv, hd)
    kx = turn(kx, cos, sin) if turned else kx
    want = {"k": append_model(c, 1, kx, counts, seqs, "k"), "v": append_model(c, 1, v.float().reshape(rows, kv, hd), counts, seqs, "v")}
    before = [t[0].clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    for _ in range(2):  # appending the same rows again changes nothing
        ops.kv_append(c, 1, k, v, starts_of(counts), ints(seqs), max_new=200, cos=cos, sin=sin)
        for w, codes, scale in (("k", c.k, c.k_scale), ("v", c.v, c.v_scale)):
            wc, ws, seen = want[w]
            at = seen[:, None, :, None].expand_as(wc)
            assert torch.equal(codes[1].cpu()[at], wc[at])
            assert torch.equal(scale[1].cpu()[seen.any(1)], ws[seen.any(1)])
    for t, b in zip((c.k, c.v, c.k_scale, c.v_scale), before):  # the other layer
        assert torch.equal(t[0], b) or t[0].isnan().any()
    lens_read = [min(n, 70) for n in lens]
    first = [n - m for n, m in zip(lens, lens_read)]
    got = ops.kv_read(c, 1, starts_of(lens_read), sum(lens_read), first=ints(first))
    for w, y in zip("kv", got):
        at = 0
        for s, (f, m) in enumerate(zip(first, lens_read)):
            assert torch.equal(y[at : at + m].double(), rows_of(c, 1, s, w)[f:].reshape(m, -1))
            at += m
    assert ops.device_status() == 0


@pytest.mark.parametrize("values", ["zero", "tiny", "huge", "edge"])
def test_append_ends_of_the_scale(values):
    from so101_smolvla_edge_b200 import ops

    c = cache([5], 1, 64, 16, seed=61)
    x = {"zero": torch.zeros(5, 64), "tiny": torch.full((5, 64), 1e-39), "huge": torch.full((5, 64), 3.3e38),
         "edge": torch.tensor([127.0, 127.5, 63.5, 254.0, -127.0])[:, None].expand(5, 64)}[values]  # fmt: skip
    x = x.to(torch.bfloat16).cuda()
    want = append_model(c, 0, x.float().reshape(5, 1, 64), [5], [0], "k")
    ops.kv_append(c, 0, x, x, starts_of([5]), max_new=5)
    id = int(c.table[0, 0])
    assert torch.equal(c.k[0, id, :, :5].cpu(), want[0][id, :, :5])
    assert torch.equal(c.k_scale[0, id].cpu(), want[1][id])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_append_not_finite(bad):
    """The page's scale is lost for good, the other pages and heads stay."""
    from so101_smolvla_edge_b200 import ops

    c = cache([40], 2, 64, 16, seed=62)
    x = torch.randn(40, 256, device="cuda", generator=gen(63)).to(torch.bfloat16)
    x[20, 3] = bad
    ops.kv_append(c, 0, x[:, :128], x[:, 128:], starts_of([40]), max_new=40)
    ids = c.table[0].long()
    lost = c.k_scale[0][ids].isnan()
    assert lost.tolist() == [[False, False], [True, False], [False, False]]
    assert not c.v_scale[0][ids].isnan().any()
    c.lengths[0] = 40
    y = torch.ones(2, 128, dtype=torch.bfloat16, device="cuda")
    c.lengths[0] = 30  # two tokens into the page that is lost
    ops.kv_append(c, 0, y, y, starts_of([2]), max_new=2)
    assert c.k_scale[0][ids].isnan().tolist() == lost.tolist()


def test_append_one_by_one_stays_within_a_step():
    """Single tokens of growing size: every earlier one is within one step of what was written."""
    from so101_smolvla_edge_b200 import ops

    c = cache([16], 1, 64, 16, seed=64)
    x = (torch.randn(16, 64, device="cuda", generator=gen(65)) * torch.logspace(0, 1, 16, device="cuda")[:, None]).to(torch.bfloat16)
    for t in range(16):
        c.lengths[0] = t + 1
        ops.kv_append(c, 0, x[t : t + 1], x[t : t + 1])
    k, _ = ops.kv_read(c, 0, starts_of([16]), 16)
    step = float(c.k_scale[0, int(c.table[0, 0]), 0])
    assert step == step_of(float(x.float().abs().max()))
    assert (k.float() - x.float()).abs().max() <= step


# ---------------------------------------------------------------------------------------------- pages


class Model:
    """The cache's bookkeeping on the host, page contents as labels."""

    def __init__(self, pool, seqs, width, page):
        self.refs, self.table, self.len = [0] * pool, [[] for _ in range(seqs)], [0] * seqs
        self.page, self.width = page, width

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def reserve(self, seqs, tokens):
        need = [-(-(self.len[s] + t) // self.page) - len(self.table[s]) for s, t in zip(seqs, tokens)]
        free = self.free_pages()
        if sum(need) > len(free) or any(self.len[s] + t > self.width * self.page for s, t in zip(seqs, tokens)):
            return False
        for s, t, n in zip(seqs, tokens, need):
            for _ in range(n):
                p = free.pop(0)
                self.refs[p] = 1
                self.table[s].append(p)
            self.len[s] += t
        return True

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.len[s] = [], 0

    def fork(self, parents, children):
        copies = sum(1 for p in parents if self.len[p] % self.page)
        if copies > len(self.free_pages()) or any(self.len[c] for c in children):
            return False
        free = self.free_pages()
        for p, c in zip(parents, children):
            whole = self.len[p] // self.page
            self.table[c] = self.table[p][:whole]
            for q in self.table[c]:
                self.refs[q] += 1
            if self.len[p] % self.page:
                q = free.pop(0)
                self.refs[q] = 1
                self.table[c] = self.table[c] + [q]
            self.len[c] = self.len[p]
        return True

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        to = dict(zip([p for p, r in enumerate(self.refs) if r and p >= live], [p for p, r in enumerate(self.refs) if not r and p < live]))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = [[to.get(p, p) for p in t] for t in self.table]


@pytest.mark.parametrize("seed", range(6))
def test_pages_life(seed):
    """Random reserves, forks, frees and compactions against the model; what sequences hold stays theirs. The last
    two have a table and a pool that are too large for a plan in shared memory."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.pages import KvPages

    rng = random.Random(seed)
    page, width = rng.choice([16, 32, 64]), 6
    pool, n = [(40, 24), (3000, 24), (25, 1500), (60, 24), (50, 3000), (9000, 24)][seed]
    kv, hd, layers = rng.choice([1, 3]), 64, 2
    c, m = KvPages(layers, pool, kv, hd, n, width * page, page), Model(pool, n, width, page)
    held = {}  # sequence -> its tokens as written (tokens, 2, layers, kv, hd)

    def same():
        assert c.lengths.tolist() == m.len and c.refs.tolist() == m.refs
        assert c.table.tolist() == [t + [-1] * (width - len(t)) for t in m.table]
        for s, x in held.items():
            for layer in range(layers):
                got = ops.kv_read(c, layer, starts_of([m.len[s]]), m.len[s], ints([s]))
                for i in range(2):
                    assert torch.equal(got[i], x[:, i, layer].reshape(len(x), -1))

    refused = 0
    for _ in range(40):
        do = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        idle = [s for s in range(n) if not m.len[s]]
        busy = [s for s in range(n) if m.len[s]]
        if do == "reserve":
            seqs = rng.sample(range(n), rng.randint(1, 4))
            tokens = [rng.randint(0, 2 * page) for _ in seqs]
            ops.kv_reserve(c, ints(seqs), ints(tokens))
            if m.reserve(seqs, tokens):
                # values that every scale holds exactly: one power of two per sequence and small codes
                new = torch.randint(-64, 65, (sum(tokens), 2, layers, kv, hd), device="cuda").to(torch.bfloat16)
                new[..., 0] = 127.0
                if sum(tokens):
                    for layer in range(layers):
                        ops.kv_append(c, layer, new[:, 0, layer].reshape(-1, kv * hd), new[:, 1, layer].reshape(-1, kv * hd),
                                      starts_of(tokens), ints(seqs), max_new=2 * page)  # fmt: skip
                at = 0
                for s, t in zip(seqs, tokens):
                    held[s] = torch.cat([held[s], new[at : at + t]]) if s in held else new[at : at + t]
                    at += t
            else:
                refused += 1
                assert ops.device_status() == L.ERR_PAGES
                L.lib().so101_clear_device_status()
        elif do == "fork" and busy and len(idle) > 1:
            children = rng.sample(idle, rng.randint(1, min(4, len(idle))))
            parents = [rng.choice(busy) for _ in children]
            ops.kv_fork(c, ints(parents), ints(children))
            if m.fork(parents, children):
                for p, ch in zip(parents, children):
                    held[ch] = held[p].clone()
            else:
                refused += 1
                assert ops.device_status() == L.ERR_PAGES
                L.lib().so101_clear_device_status()
        elif do == "free" and busy:
            seqs = rng.sample(busy, rng.randint(1, min(3, len(busy))))
            ops.kv_free(c, ints(seqs + seqs[:1]))  # a sequence named twice is freed once
            m.free(seqs)
            for s in seqs:
                held.pop(s)
        elif do == "compact":
            ops.kv_compact(c)
            m.compact()
        held = {s: x for s, x in held.items() if len(x)}
        same()
    assert refused or seed != 2
    assert ops.device_status() == 0


def test_pages_copy():
    from so101_smolvla_edge_b200 import ops

    c = cache([100], 3, 64, 16, layers=3, seed=71, spare=9)
    want = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    src, dst = c.table[0, :3].tolist(), [p for p, r in enumerate(c.refs.tolist()) if r == 0][:3]
    for t in want:
        t[:, dst] = t[:, src].clone()
    ops.kv_copy(c, ints(src), ints(dst))
    for t, w in zip((c.k, c.v, c.k_scale, c.v_scale), want):
        assert torch.equal(torch.nan_to_num(t.float(), nan=-1.0), torch.nan_to_num(w.float(), nan=-1.0))


def test_indices_out_of_range_are_recorded():
    """What the host cannot see: rows, sequences and pages that do not exist are skipped and recorded."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200 import ops

    def recorded():
        got = ops.device_status()
        L.lib().so101_clear_device_status()
        return got == L.ERR_PAGES

    c = cache([40, 20], 2, 64, 16, seed=81)
    q = queries(2, 4, 64)
    x = torch.ones(2, 128, dtype=torch.bfloat16, device="cuda")
    before = c.k.clone()
    ops.attention_pages(q, c, 0, 4, None, ints([0, 7]))
    assert recorded()
    ops.kv_append(c, 0, x, x, None, ints([-1, 2]))
    assert recorded() and torch.equal(c.k, before)
    ops.kv_append(c, 0, x, x, starts_of([1, 3]), max_new=3)
    assert recorded()
    ops.kv_read(c, 0, starts_of([1, 21]), 22)
    assert recorded()
    ops.kv_copy(c, ints([0]), ints([c.n_pages]))
    assert recorded()
    ops.kv_fork(c, ints([0]), ints([1]))  # not empty
    assert recorded() and c.lengths.tolist() == [40, 20]
    ops.kv_reserve(c, ints([5]), ints([1]))
    assert recorded()
    ops.kv_free(c, ints([9]))
    assert recorded()
    c.table[1, 0] = c.n_pages + 3
    ops.attention_pages(q, c, 0, 4)
    assert recorded()
    p = packed_case([20], 4, 2, 64)
    ops.attention_packed(*p, ints([0, 21]), 20, 4, 2)
    assert recorded()
    ops.attention_packed(*p, ints([0, 12, 5]), 20, 4, 2)
    assert recorded()


def test_cache_refusals():
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.pages import KvPages

    for bad in (dict(page=48), dict(head_dim=96), dict(n_pages=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            KvPages(**{**dict(n_layers=1, n_pages=4, n_kv=2, head_dim=64, max_seqs=2, max_len=64, page=16), **bad})
    c = KvPages(1, 4, 2, 64, 2, 64, 16)
    with pytest.raises(ValueError):
        KvPages.adopt(c.k, c.v, c.k_scale[..., :1], c.v_scale, c.table, c.lengths, c.refs)
    with pytest.raises(ValueError):
        KvPages.adopt(c.k, c.v.float(), c.k_scale, c.v_scale, c.table, c.lengths, c.refs)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.kv_append(c, 1, x, x)  # no such layer
    with pytest.raises(ValueError):
        ops.kv_append(c, 0, x, x[:1])
    with pytest.raises(ValueError):
        ops.kv_append(c, 0, x, x, ints([0, 1]), ints([0, 1]))
    with pytest.raises(ValueError):
        ops.attention_pages(x, c, 0, 3)  # 3 heads over 2 kv heads
    with pytest.raises(ValueError):
        ops.attention_pages(torch.zeros(2, 192, dtype=torch.bfloat16, device="cuda"), c, 0, 3)
    with pytest.raises(ValueError):
        ops.attention_pages(x, c, 0, 2, max_q=0)
    with pytest.raises(ValueError):
        ops.kv_reserve(c, ints([0]), ints([1, 2]))
    with pytest.raises(ValueError):
        ops.kv_fork(c, ints([0]), torch.zeros(1, device="cuda"))
    assert ops.attention_pages(x[:0], c, 0, 2, ints([0])).shape == (0, 128)


# --------------------------------------------------------------------------------- streams and graphs


def test_graph_and_streams():
    """A captured step (append and attention) replays with new rows; two streams do not disturb each other."""
    from so101_smolvla_edge_b200 import ops

    heads, kv, hd = 15, 5, 64
    lens = [3000, 5000]
    c = cache(lens, kv, hd, 64, seed=91)
    x = torch.randn(2, (heads + 2 * kv) * hd, device="cuda", generator=gen(92)).to(torch.bfloat16)
    q, k, v = x[:, : heads * hd], x[:, heads * hd : (heads + kv) * hd], x[:, (heads + kv) * hd :]
    out = torch.empty(2, heads * hd, dtype=torch.bfloat16, device="cuda")

    def step():
        ops.kv_append(c, 0, k, v)
        ops.attention_pages(q, c, 0, heads, out=out)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    x.copy_(torch.randn(x.shape, device="cuda", generator=gen(93)).to(torch.bfloat16))
    g.replay()
    torch.cuda.synchronize()
    check(out, *pages_want(q, c, 0, heads, [1, 1], [0, 1], True, hd**-0.5))
    alone = out.clone()
    others = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for o in others:
            with torch.cuda.stream(o):
                got.append(ops.attention_pages(q, c, 0, heads))
    torch.cuda.synchronize()
    assert all(torch.equal(y, alone) for y in got)
