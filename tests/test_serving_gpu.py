"""The serving operators where their parts meet: items without key tiles, refused reservations, graphs, streams.

Values by the same 64-bit restatements and tolerances as test_text_gpu.py.
"""

from __future__ import annotations

import pytest
import torch

from test_text_gpu import attend, cache, check, ints, packed_case, pages_want, queries, rope, starts_of, turn
from test_text_tower_gpu import TOKEN, bundle, off, plain  # noqa: F401 (bundle: a fixture)

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


def test_long_items_key_by_key_hold_nobody_up():
    """Several items of 131072 keys that go key by key on every CTA (seconds of them), ordinary ones behind them: whoever waits
    for those goes on waiting. All sequences share the pages of two."""
    from so101_smolvla_edge_b200 import ops

    long, short, n, heads = 131072, 300, 148, 16
    lens = ([long] * 3 + [short]) * n
    base = cache([long, short], 1, 64, 64, seed=215)
    base.v_scale[:, base.table[0, : long // 64].long()] *= 1.5
    c = type(base).adopt(base.k, base.v, base.k_scale, base.v_scale, base.table[[0, 0, 0, 1] * n].contiguous(), ints(lens), base.refs)
    q = queries(2 * 16, heads, 64, seed=216)
    counts = [16] * len(lens)
    rows = torch.cat([q[:16].repeat(3, 1), q[16:]]).repeat(n, 1)
    got = ops.attention_pages(rows, c, 0, heads, starts_of(counts), max_q=16)
    assert ops.device_status() == 0
    want, tol = pages_want(q, base, 0, heads, [16, 16], [0, 1], True, 0.125)
    got = got.reshape(n, 64, -1)
    check(got[:, 48:], want[16:].expand(n, -1, -1), tol[16:])
    for i in range(3):
        check(got[:, 16 * i : 16 * i + 16], want[:16].expand(n, -1, -1), tol[:16])


def test_packed_rows_again_in_a_long_prompt():
    """An infinity in the last values of a long prompt: the rows before it that share its tile are taken again, key by key
    (seconds of it), while the CTA's other rows wait."""
    from so101_smolvla_edge_b200 import ops

    n, hd, bad = 420_000, 64, 60
    x = torch.randn(n, 3 * hd, device="cuda", generator=torch.Generator("cuda").manual_seed(218)).to(torch.bfloat16)
    q, k, v = x[:, :hd], x[:, hd : 2 * hd], x[:, 2 * hd :]
    rows = torch.cat([torch.randint(0, n, (200,), generator=torch.Generator().manual_seed(219)), torch.arange(n - 300, n)]).cuda()
    fine = rows < n - bad
    want, tol = zip(*(attend(q[r], k, v, r, hd**-0.5, 0.0, 2**-8) for r in rows[fine].split(50)))
    v[n - bad] = float("inf")
    got = ops.attention_packed(q, k, v, ints([0, n]), n, 1, 1)
    assert ops.device_status() == 0
    check(got[rows[fine]], torch.cat(want), torch.cat(tol))
    assert not torch.isfinite(got[n - bad :]).any()


@pytest.mark.parametrize("lens", [[300, 77, 128], [43] * 90, [1, 700]])
@pytest.mark.parametrize("heads,kv,hd", [(15, 5, 64), (6, 2, 128), (3, 3, 128)])
def test_rotated_queries_keep_two_parts(lens, heads, kv, hd):
    """Scores of tens, where a rotated query rounded to bf16 once would show: what is left of it after two parts is 2^-16
    of a value (the rest of the tolerance as in test_text_gpu.py)."""
    from so101_smolvla_edge_b200 import ops

    q, k, v = packed_case(lens, heads, kv, hd, seed=229, big=16.0)
    cos, sin = rope(torch.cat([torch.arange(n) for n in lens]), hd)
    got = ops.attention_packed(q, k, v, starts_of(lens), max(lens), heads, kv, cos=cos, sin=sin)
    qr, at = turn(q.double().reshape(-1, heads, hd), cos, sin), 0
    for n in lens:
        for h in range(heads):
            sl, g = slice(at, at + n), h // (heads // kv) * hd
            want, tol = attend(qr[sl, h], k[sl, g : g + hd], v[sl, g : g + hd], torch.arange(n, device="cuda"), hd**-0.5, 2**-16, 2**-8)
            check(got[sl, h * hd : (h + 1) * hd], want, tol)
        at += n
    assert ops.device_status() == 0


# ------------------------------------------------------------------------------ a reservation that is refused


def test_append_after_a_refused_reservation():
    """The pool runs out: what the sequences hold (a part-filled page, whole pages shared by a fork) stays as it was, through
    every layer's append, until a later reservation is met."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.pages import KvPages

    c = KvPages(2, 6, 2, 64, 4, 128, 16)
    x = torch.randn(64, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(221)).to(torch.bfloat16)

    def append(seqs, counts):
        rows = x[: sum(counts)] * (4.0 if sum(counts) < 4 else 1.0)  # larger ones: they would raise the scales
        for layer in range(2):
            ops.kv_append(c, layer, rows[:, :128], rows[:, 128:], starts_of(counts), ints(seqs), max_new=max(counts))

    ops.kv_reserve(c, ints([0, 2]), ints([32, 21]))  # two pages that a fork shares, and one and a part
    append([0, 2], [32, 21])
    ops.kv_fork(c, ints([0]), ints([1]))
    ops.kv_reserve(c, ints([3]), ints([30]))
    append([3], [30])  # all six pages are in use
    assert ops.device_status() == 0
    state = (c.k, c.v, c.k_scale, c.v_scale, c.table, c.lengths, c.refs)
    before = [t.clone() for t in state]
    ops.kv_reserve(c, ints([1, 2, 3]), ints([1, 1, 1]))  # sequence 1 needs a page
    append([1, 2, 3], [1, 1, 1])
    assert all(torch.equal(t, b) for t, b in zip(state, before))
    assert ops.device_status() == L.ERR_PAGES
    L.lib().so101_clear_device_status()
    ops.kv_free(c, ints([3]))
    ops.kv_reserve(c, ints([1, 2, 3]), ints([1, 1, 1]))
    append([1, 2, 3], [1, 1, 1])
    assert ops.device_status() == 0 and c.lengths.tolist() == [32, 33, 22, 1]
    for s in (1, 2, 3):
        k, _ = ops.kv_read(c, 1, ints([0, 1]), 1, ints([s]), first=ints([int(c.lengths[s]) - 1]))
        want = x[s - 1 : s, :128] * 4.0
        assert (k.float() - want.float()).abs().max() <= want.float().abs().max() / 63.5


@pytest.mark.parametrize("n", [4, 900])
def test_reserve_with_a_sequence_named_twice(n):
    """Each entry alone would fit, both together would pass the table row's end: nothing changes."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.pages import KvPages

    c = KvPages(1, 2 * n + 8, 1, 64, n, 64, 16)
    ops.kv_reserve(c, ints([n - 1]), ints([20]))
    state = (c.table, c.lengths, c.refs)
    before = [t.clone() for t in state]
    others = list(range(n - 2))
    ops.kv_reserve(c, ints([n - 1, *others, n - 1]), ints([40, *[1] * (n - 2), 40]))
    assert ops.device_status() == L.ERR_PAGES
    L.lib().so101_clear_device_status()
    assert all(torch.equal(t, b) for t, b in zip(state, before))
    ops.kv_reserve(c, ints([n - 1, *others]), ints([40, *[1] * (n - 2)]))
    assert ops.device_status() == 0 and c.lengths.tolist() == [1] * (n - 2) + [0, 60]


# ------------------------------------------------------------------------------------------- the text tower


def test_tower_goes_on_after_the_pool_ran_out(bundle):  # noqa: F811
    """Steps that find no page leave the cache as it is, those after them too; check says so once and sets the counts
    right, and the sequences go on where they stood."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200.text_tower import TextTower

    g = torch.Generator().manual_seed(231)
    dim = bundle.spec.text_dim
    tower = TextTower(bundle, n_pages=6, max_seqs=6, max_len=128, page=32)
    text = {q: torch.randn(n, dim, generator=g) for q, n in ((0, 64), (1, 40))}
    tower.prompt(torch.cat(list(text.values())).cuda(), [64, 40], [0, 1])
    tower.fork([0, 1], [2, 3])  # 2 shares both pages of 0; 3 copies a part: five pages
    text[2], text[3] = text[0], text[1]
    tower.prompt(torch.randn(3, dim, generator=g).cuda(), [3], [4])  # the sixth
    tower.check()
    pages = tower.pages
    state = [t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.lengths, pages.refs)]
    for seqs in ([0, 1, 3], [1, 3], [2], [1]):  # 0 and 2 need a page; 1 and 3 do not, but went along with 0
        tower.step(5.0 * torch.randn(len(seqs), dim, generator=g).cuda(), seqs)
    tower.fork([1], [5])
    with pytest.raises(L.KernelError):
        tower.check()
    for t, was in zip((pages.k, pages.v, pages.k_scale, pages.v_scale, pages.table, pages.lengths, pages.refs), state):
        assert torch.equal(t, was)
    tower.check()
    assert tower.lengths == pages.lengths.tolist() == [64, 40, 64, 40, 3, 0]
    tower.free([4])
    rows = torch.randn(3, dim, generator=g)
    got = tower.step(rows.cuda(), [2, 1, 3])
    tower.check()
    for i, q in enumerate((2, 1, 3)):
        assert off(got[i], plain(bundle, torch.cat([text[q], rows[i : i + 1]]))[-1]) <= TOKEN


def test_tower_does_not_wait_for_the_device(bundle):  # noqa: F811
    """Prompts, tokens, forks, frees and compactions without a copy that the host waits for."""
    from so101_smolvla_edge_b200.text_tower import TextTower

    tower = TextTower(bundle, n_pages=30, max_seqs=6, max_len=128, page=32)
    x = torch.randn(60, bundle.spec.text_dim, device="cuda", generator=torch.Generator("cuda").manual_seed(233))

    def turn_of_it():
        tower.prompt(x[:50], [40, 10], [0, 1])
        tower.fork([0, 1], [2, 3])
        tower.step(x[:4], [0, 1, 2, 3])
        tower.step(x[:9], [1, 3], [4, 5])
        tower.free([0, 1, 2, 3])
        tower.compact()

    turn_of_it()  # what the first turn builds
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        turn_of_it()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    tower.check()


def test_tower_refuses_what_it_does_not_have(bundle):  # noqa: F811
    """Numbers outside the cache (negative ones count from the end of a Python list), a child that is a parent too,
    lists of two lengths; nothing changes. No sequences at all are fine."""
    from so101_smolvla_edge_b200.text_tower import TextTower

    tower = TextTower(bundle, n_pages=8, max_seqs=4, max_len=64, page=32)
    x = torch.zeros(5, bundle.spec.text_dim, device="cuda")
    tower.prompt(x, [5], [3])
    for call in (
        lambda: tower.free([-1]),
        lambda: tower.free([4]),
        lambda: tower.fork([-1], [0]),
        lambda: tower.fork([3], [-2]),
        lambda: tower.fork([3], [4]),
        lambda: tower.fork([3, 0], [0, 1]),
        lambda: tower.fork([3], [0, 1]),
        lambda: tower.cached(0, -1),
        lambda: tower.step(x[:1], [-1]),
    ):
        with pytest.raises(ValueError):
            call()
    assert tower.lengths == tower.pages.lengths.tolist() == [0, 0, 0, 5]
    assert tower.prompt(x[:0], [], []).shape == tower.step(x[:0], []).shape == (0, bundle.spec.text_dim)
    tower.fork([], [])
    tower.free([])
    tower.fork([3], [0])
    tower.check()
    assert tower.lengths == tower.pages.lengths.tolist() == [5, 0, 0, 5]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one(bundle):  # noqa: F811
    from so101_smolvla_edge_b200.text_tower import TextTower

    x = torch.randn(9, bundle.spec.text_dim, generator=torch.Generator().manual_seed(235))
    got = []
    for dev in ("cuda:0", "cuda:1"):  # the first is current throughout
        tower = TextTower(bundle, n_pages=8, max_seqs=2, max_len=64, page=32, device=dev)
        rows = x.to(dev)
        out = [tower.prompt(rows[:7], [7], [0])]
        tower.fork([0], [1])
        out.append(tower.step(rows[7:], [0, 1]))
        tower.compact()
        tower.check()
        got.append([y.cpu() for y in (*out, *tower.cached(1, 0))])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_tickets_after_a_wait_that_ran_out(monkeypatch):
    """What a call that gave up leaves behind (tickets counted in part, put there by hand) goes with the status."""
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200 import ops

    c = cache([9000, 5000], 2, 64, 64, seed=237)
    q = queries(2, 6, 64, seed=238)
    want = ops.attention_pages(q, c, 0, 6)
    stream = torch.cuda.current_stream()
    ops.pages_workspace(stream.device.index, stream.cuda_stream).tickets.fill_(1)
    with monkeypatch.context() as m:
        m.setattr(ops, "device_status", lambda: L.ERR_TIMEOUT)
        ops.clear_device_status()
    assert ops.device_status() == 0
    assert torch.equal(ops.attention_pages(q, c, 0, 6), want)


# ------------------------------------------------------------------------------------------ graphs of attention


def attention_graphs(n):
    """Graphs of single tokens over long sequences (read in parts, so that partials and tickets are in use), captured
    on torch's own capture stream without a call before them, each with a cache, queries and a result of its own."""
    from so101_smolvla_edge_b200 import ops

    out = []
    for i in range(n):
        c = cache([4000 + 700 * i, 9000], 2, 64, 64, seed=241 + i)
        q = queries(2, 6, 64, seed=251 + i)
        y = torch.empty(2, 384, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(8):
                ops.attention_pages(q, c, 0, 6, out=y)
        out.append((g, c, q, y))
    return out


def test_graphs_captured_on_one_stream_replayed_on_several():
    from so101_smolvla_edge_b200 import ops

    graphs = attention_graphs(4)
    want = [pages_want(q, c, 0, 6, [1, 1], [0, 1], True, 0.125) for _, c, q, _ in graphs]
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, *_), s in reversed(list(zip(graphs, streams))):  # the first captured is not the first replayed
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.attention_pages(graphs[0][2], graphs[0][1], 0, 6)
    torch.cuda.synchronize()
    for (_, _, _, y), w in zip(graphs, want):
        check(y, *w)
    check(eager, *want[0])
    assert ops.device_status() == 0


def test_a_graph_beside_eager_calls_on_its_capture_stream():
    from so101_smolvla_edge_b200 import ops

    c = cache([9000, 5000], 2, 64, 64, seed=261)
    q = queries(2, 6, 64, seed=262)
    want = pages_want(q, c, 0, 6, [1, 1], [0, 1], True, 0.125)
    y = torch.empty(2, 384, dtype=torch.bfloat16, device="cuda")
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for _ in range(8):
            ops.attention_pages(q, c, 0, 6, out=y)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(t):
            g.replay()
        with torch.cuda.stream(s):
            got += [ops.attention_pages(q, c, 0, 6) for _ in range(4)]
    torch.cuda.synchronize()
    check(y, *want)
    assert all(torch.equal(x, y) for x in got)
    assert ops.device_status() == 0


def test_a_graphs_workspace_goes_with_it():
    import gc
    import time

    from so101_smolvla_edge_b200 import ops

    c, q = cache([9000], 2, 64, 64, seed=271), queries(1, 6, 64, seed=272)
    attention_graphs(1)  # what a first capture leaves for good
    ops.attention_pages(q, c, 0, 6)
    gc.collect()
    torch.cuda.synchronize()
    time.sleep(0.5)  # the driver may say a little later that a graph is gone
    ops.attention_pages(q, c, 0, 6)
    before = torch.cuda.memory_allocated()
    graphs = attention_graphs(3)
    assert torch.cuda.memory_allocated() >= before + 3 * (40 << 20)
    del graphs
    gc.collect()
    for _ in range(100):
        ops.attention_pages(q, c, 0, 6)
        if torch.cuda.memory_allocated() <= before:
            break
        time.sleep(0.02)
    assert torch.cuda.memory_allocated() <= before


def test_a_graph_outlives_the_program():
    """A process that ends with a graph alive ends well."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys
sys.path[:0] = ['.', 'tests']
from test_serving_gpu import attention_graphs
import builtins, torch
builtins.kept = attention_graphs(2)
[g.replay() for g, *_ in builtins.kept]
torch.cuda.synchronize()
"""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr


def test_a_single_row_of_any_stride():
    """A row whose stride says nothing (a transposed column) is a row like another."""
    from so101_smolvla_edge_b200 import ops

    c, d = (cache([70], 2, 64, 64, seed=281) for _ in range(2))
    for one, two in ((lambda t: t, c), (lambda t: t.reshape(-1, 1).clone().t(), d)):
        g = torch.Generator("cuda").manual_seed(282)
        q, k, v = (one(torch.randn(1, n, device="cuda", generator=g).to(torch.bfloat16)) for n in (384, 128, 128))
        ops.kv_append(two, 0, k, v)
        two.got = (ops.attention_pages(q, two, 0, 6), ops.attention_packed(q, k, v, ints([0, 1]), 1, 6, 2))
    assert d.k.equal(c.k) and all(torch.equal(a, b) for a, b in zip(c.got, d.got))
