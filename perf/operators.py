"""The packed-prompt attention and the 8-bit paged K/V cache, case by case: inputs, plain forms, 64-bit values.

Four operators of a text tower that serves many sequences:

    prompt   causal grouped-query attention over whole prompts packed end to end (ops.attention_packed)
    append   new keys (rotated) and values into 8-bit pages, and the touched pages read back as rows
             (ops.kv_append, ops.kv_read)
    pages    attention of each sequence's last tokens over its 8-bit pages (ops.attention_pages)
    fork / compact   sharing, copying, freeing and moving the cache's pages (ops.kv_free, kv_fork, kv_compact)

`own` chooses between the plain torch form and the framework's calls. The cache: int8 codes
(layer, page, kv head, token, dim) with one power-of-two scale for each page and kv head, for keys and values
apart; a table row of page numbers for each sequence (-1 past its pages), its length, and how many sequences
hold each page.
"""

from __future__ import annotations

import random

import torch

own = False

# The text tower's own heads (15 query, 5 kv, 64 wide, 16 layers) and prompts: one to four cameras of 64 rows,
# 48 instruction tokens and a state row. The 32 / 8 / 128 heads are a larger decoder's.


def listed() -> list[dict]:
    return [
        # one robot's prompt, one layer: latency
        {"name": "prompt one", "op": "prompt", "seqs": 1, "lo": 241, "hi": 241, "heads": 15, "kv": 5, "hd": 64, "rope": True},
        # 64 robots with one to four cameras and instructions of different lengths
        {"name": "prompt batch", "op": "prompt", "seqs": 64, "lo": 113, "hi": 305, "heads": 15, "kv": 5, "hd": 64, "rope": True},
        # one long document on the larger heads
        {"name": "prompt long", "op": "prompt", "seqs": 1, "lo": 8191, "hi": 8191, "heads": 32, "kv": 8, "hd": 128, "rope": False},
        # one decoding step of 64 sequences
        {"name": "append step", "op": "append", "seqs": 64, "lo": 1, "hi": 1, "old": 241, "kv": 5, "hd": 64, "page": 64, "rope": True},
        # the keys and values of 64 prompts, some going on in pages that earlier turns left part-filled
        {"name": "append batch", "op": "append", "seqs": 64, "lo": 113, "hi": 305, "old": 100, "kv": 5, "hd": 64, "page": 64, "rope": True},
        # one token of one sequence: latency
        {"name": "pages one", "op": "pages", "seqs": 1, "lo": 242, "hi": 242, "rows": 1, "causal": True, "heads": 15, "kv": 5, "hd": 64, "page": 64, "rope": True},
        # one token of 64 sequences at different points of their lives
        {"name": "pages batch", "op": "pages", "seqs": 64, "lo": 200, "hi": 8000, "rows": 1, "causal": True, "heads": 15, "kv": 5, "hd": 64, "page": 64, "rope": True},
        # a chunk of 50 action tokens of 64 robots, each token seeing all of them and the prompt
        {"name": "pages chunk", "op": "pages", "seqs": 64, "lo": 291, "hi": 291, "rows": 50, "causal": False, "heads": 15, "kv": 5, "hd": 64, "page": 32, "rope": True},
        # one token over a very long context on the larger heads
        {"name": "pages long", "op": "pages", "seqs": 1, "lo": 131071, "hi": 131071, "rows": 1, "causal": True, "heads": 32, "kv": 8, "hd": 128, "page": 64, "rope": False},
        # eight observations, each sampled eight ways: last step's samples go, new ones fork
        {"name": "fork", "op": "fork", "parents": 8, "children": 8, "length": 241, "layers": 16, "pool": 256, "kv": 5, "hd": 64, "page": 64},
        # a small cache after some sequences ended
        {"name": "compact small", "op": "compact", "seqs": 24, "length": 241, "live": 0.5, "layers": 16, "pool": 128, "kv": 5, "hd": 64, "page": 64},
        # the cache of a busy server after half of its sequences ended
        {"name": "compact large", "op": "compact", "seqs": 500, "length": 241, "live": 0.5, "layers": 16, "pool": 2048, "kv": 5, "hd": 64, "page": 64},
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["prompt", "append", "pages", "pages", "fork", "compact"])
    hd = rng.choice([64, 64, 128])
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 32, 64])
    if op == "prompt":
        hi = _log(rng, 1, 8000)
        lo = max(1, int(hi * rng.random()))
        # rows x rows x heads stays under the largest case's
        seqs = min(_log(rng, 1, 128), max(1, int(32 * 8191**2 / (hi * hi * kv * group))))
        return {"op": op, "seqs": seqs, "lo": lo, "hi": hi, "heads": kv * group, "kv": kv, "hd": hd, "rope": rng.random() < 0.5}
    if op == "append":
        hi = _log(rng, 1, 600)
        seqs = _log(rng, 1, 100)
        return {"op": op, "seqs": seqs, "lo": max(1, int(hi * rng.random())), "hi": hi, "old": _log(rng, 1, 400), "kv": kv, "hd": hd,
                "page": page, "rope": rng.random() < 0.5}  # fmt: skip
    if op == "pages":
        hi = _log(rng, 1, 131000)
        rows = rng.choice([1, 1, 2, 5, _log(rng, 1, 64)])
        room = 131071 * 8 * 128
        seqs = max(1, min(_log(rng, 1, 128), room // (hi * kv * hd), int(4e8 / (hi * kv * group * rows))))
        return {"op": op, "seqs": seqs, "lo": max(1, int(hi * rng.random())), "hi": hi, "rows": rows, "causal": rng.random() < 0.6,
                "heads": kv * group, "kv": kv, "hd": hd, "page": page, "rope": rng.random() < 0.5}  # fmt: skip
    layers = _log(rng, 1, 16)
    length = _log(rng, 1, 700)
    each = -(-length // page)
    room = min(1_300_000_000 // (layers * kv * page * hd * 2), 4096)  # pages that the largest pool has bytes for
    if op == "fork":
        parents, children = _log(rng, 1, 16), _log(rng, 1, 16)
        while parents * (each + children) + 1 > room and parents > 1:
            parents //= 2
        return {"op": op, "parents": parents, "children": children, "length": length, "layers": layers,
                "pool": parents * (each + children) + rng.randint(1, 40), "kv": kv, "hd": hd, "page": page}  # fmt: skip
    seqs = max(2, min(_log(rng, 2, 500), room // each))
    return {"op": op, "seqs": seqs, "length": length, "live": round(0.2 + 0.6 * rng.random(), 2), "layers": layers,
            "pool": seqs * each + rng.randint(0, 40), "kv": kv, "hd": hd, "page": page}  # fmt: skip


# ------------------------------------------------------------------------------------------------- inputs


def _lens(case: dict) -> list[int]:
    """The case's sequence lengths: the same for every seed."""
    rng = random.Random(case["seqs"] * 1000003 + case["hi"])
    got = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    got[-1] = case["hi"]
    return got


def _old(case: dict) -> list[int]:
    """Tokens that each sequence of an append case holds already: some none, some whole pages."""
    rng = random.Random(case["seqs"] * 7919 + case["old"])
    page = case["page"]
    if case["hi"] == 1:
        return [case["old"] + rng.randint(0, 2 * page) for _ in range(case["seqs"])]
    return [rng.choice([0, 0, page, rng.randint(1, case["old"])]) for _ in range(case["seqs"])]


def _starts(lens: list[int]) -> torch.Tensor:
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device="cuda")


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _rope(pos: torch.Tensor, hd: int) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 10000.0 ** (-torch.arange(0, hd // 2, device="cuda", dtype=torch.float32) * 2 / hd)
    ang = pos.float()[:, None] * inv[None]
    return torch.cos(ang), torch.sin(ang)


def _rows(g: torch.Generator, rows: int, heads: int, kv: int, hd: int) -> torch.Tensor:
    """Fused q | k | v rows as a projection leaves them: a few key channels are much larger than the rest."""
    x = torch.randn(rows, (heads + 2 * kv) * hd, device="cuda", generator=g)
    big = torch.rand((heads + 2 * kv) * hd, device="cuda", generator=g) < 0.03
    x = torch.where(big[None], 4.0 * x, x)
    return x.to(torch.bfloat16)


def _cache(g: torch.Generator, case: dict, layers: int, pages_of: list[int], lens: list[int], width: int, pool: int) -> dict:
    """A cache in use: sequence i has pages_of[i] pages, scattered over the pool as after hours of service."""
    kv, hd, page = case["kv"], case["hd"], case["page"]
    shape = (layers, pool, kv, page, hd)
    order = torch.randperm(pool, device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    used = torch.tensor(pages_of, device="cuda")
    at = torch.arange(width, device="cuda")[None] < used[:, None]
    table[at] = order[: int(used.sum())]
    refs = torch.zeros(pool, dtype=torch.int32, device="cuda")
    refs[table[at].long()] = 1
    codes = [torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
    # codes of bell-shaped values: the mean of two draws, and steps of 1/32 to 1/16 of a value's size
    codes = [((c // 2) + (torch.roll(c, 1, -1) // 2)).clamp_(min=-127) for c in codes]
    scales = [2.0 ** torch.randint(-6, -4, (layers, pool, kv), device="cuda", generator=g).float() for _ in range(2)]
    return {"k": codes[0], "v": codes[1], "k_scale": scales[0], "v_scale": scales[1], "table": table,
            "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"), "refs": refs}  # fmt: skip


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    op = case["op"]
    st: dict = {"case": case, "op": op}
    if op == "prompt":
        lens = _lens(case)
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        st["starts"], st["max_len"] = _starts(lens), max(lens)
        x = _rows(g, sum(lens), heads, kv, hd)
        st["q"], st["k"], st["v"] = x[:, : heads * hd], x[:, heads * hd : (heads + kv) * hd], x[:, (heads + kv) * hd :]
        if case["rope"]:
            st["cos"], st["sin"] = _rope(torch.cat([torch.arange(n, device="cuda") for n in lens]), hd)
        return st
    if op == "append":
        new, old, page = _lens(case), _old(case), case["page"]
        total = [a + b for a, b in zip(old, new)]
        pages_of = [-(-t // page) for t in total]
        st["cache"] = _cache(g, case, 1, pages_of, total, max(pages_of), sum(pages_of) + 7)
        st["starts"], st["max_new"] = _starts(new), max(new)
        first = [(o // page) * page for o in old]
        st["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        st["read_starts"], st["max_read"] = _starts([t - f for t, f in zip(total, first)]), max(t - f for t, f in zip(total, first))
        st["read_rows"] = sum(total) - sum(first)
        kv, hd = case["kv"], case["hd"]
        x = _rows(g, sum(new), 0, kv, hd)
        st["k_new"], st["v_new"] = x[:, : kv * hd], x[:, kv * hd :]
        if case["rope"]:
            st["cos"], st["sin"] = _rope(torch.cat([torch.arange(o, t, device="cuda") for o, t in zip(old, total)]), hd)
    elif op == "pages":
        lens, page, rows = _lens(case), case["page"], case["rows"]
        pages_of = [-(-n // page) for n in lens]
        st["cache"] = _cache(g, case, 1, pages_of, lens, max(pages_of), sum(pages_of) + 7)
        st["max_len"] = max(lens)
        heads, kv, hd = case["heads"], case["kv"], case["hd"]
        st["starts"] = _starts([rows] * len(lens))
        st["q"] = _rows(g, rows * len(lens), heads, 0, hd)
        if case["rope"]:
            st["cos"], st["sin"] = _rope(torch.cat([torch.arange(n - rows, n, device="cuda").clamp(min=0) for n in lens]), hd)
    elif op == "fork":
        n, m, page = case["parents"], case["children"], case["page"]
        each = -(-case["length"] // page)
        lens = [case["length"]] * n + [0] * (n * m)
        st["cache"] = _cache(g, case, case["layers"], [each] * n + [0] * (n * m), lens, each + 1, case["pool"])
        st["parents"] = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(m)
        st["children"] = torch.arange(n, n + n * m, device="cuda", dtype=torch.int32)
    else:
        n, page = case["seqs"], case["page"]
        each = -(-case["length"] // page)
        rng = random.Random(seed)
        gone = set(rng.sample(range(n), n - max(1, round(case["live"] * n))))
        lens = [0 if i in gone else case["length"] for i in range(n)]
        # every sequence had its pages in order of arrival; those that ended left holes
        st["cache"] = _cache(g, case, case["layers"], [0 if i in gone else each for i in range(n)], lens, each, case["pool"])
        # compaction moves the pages in place: the tables before it, so that each pass has the same work
        st["snapshot"] = {k: st["cache"][k].clone() for k in ("table", "refs")}
    if own:
        from so101_smolvla_edge_b200.pages import KvPages

        st["pages"] = KvPages.adopt(**st["cache"])
    return st


# ------------------------------------------------------------------------------------------- plain forms


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x (rows, heads, hd), the halves of each head turned by the row's angles."""
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _heads(x: torch.Tensor, hd: int, st: dict, rope: bool) -> torch.Tensor:
    y = x.float().reshape(x.shape[0], -1, hd)
    return _rotate(y, st["cos"], st["sin"]) if rope and "cos" in st else y


def _where(starts: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Each packed row's sequence and its place in it."""
    r = torch.arange(rows, device=starts.device)
    s = torch.searchsorted(starts, r.to(starts.dtype), right=True) - 1
    return s, r - starts[s]


def _softmax_v(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """q (b, kv, group * n, hd), k and v (b, kv, keys, hd), seen broadcast to the scores; rows that see nothing: 0."""
    s = torch.matmul(q, k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    s = s.masked_fill_(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(m == float("-inf"), torch.zeros_like(m), m)))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _grouped(q: torch.Tensor, kv: int) -> torch.Tensor:
    """(b, n, heads, hd) to (b, kv, group * n, hd)."""
    b, n, h, hd = q.shape
    return q.reshape(b, n, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, h // kv * n, hd)


def _plain_prompt(st: dict) -> torch.Tensor:
    c = st["case"]
    kv, hd, heads, most = c["kv"], c["hd"], c["heads"], st["max_len"]
    starts = st["starts"].long()
    rows = st["q"].shape[0]
    q, k, v = _heads(st["q"], hd, st, True), _heads(st["k"], hd, st, False), _heads(st["v"], hd, st, False)
    at = (starts[:-1, None] + torch.arange(most, device=q.device)).clamp(max=rows - 1)
    i = torch.arange(most, device=q.device)
    seen = i[None, :] <= i[:, None]  # keys past a sequence's end lie past all of its rows
    seen = seen.repeat(heads // kv, 1)[None, None]
    o = _softmax_v(_grouped(q[at], kv), k[at].transpose(1, 2), v[at].transpose(1, 2), seen)
    o = o.reshape(len(starts) - 1, kv, heads // kv, most, hd).permute(0, 3, 1, 2, 4)
    s, p = _where(starts, rows)
    return o[s, p].reshape(rows, heads * hd).to(torch.bfloat16)


def _step(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two s with amax <= 127 s (from 2^-126 to 2^121)."""
    m, e = torch.frexp(amax)
    s = torch.ldexp(torch.ones_like(amax), (e - 7 + (m > 127 / 128).to(e.dtype)).clamp(-126, 121))
    s = torch.where(amax == 0, torch.full_like(s, 2.0**-126), s)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


def _plain_append(st: dict) -> dict:
    c, cache = st["case"], st["cache"]
    kv, hd, page = c["kv"], c["hd"], c["page"]
    starts, lengths = st["starts"].long(), cache["lengths"].long()
    new = starts[1:] - starts[:-1]
    old = lengths - new
    touched = -(-st["max_read"] // page)
    at = torch.arange(touched, device="cuda")[None] + (old // page)[:, None]  # the pages that take new tokens
    live = at * page < lengths[:, None]
    ids = torch.where(live, cache["table"].long().gather(1, at.clamp(max=cache["table"].shape[1] - 1)), -1)
    token = at[..., None] * page + torch.arange(page, device="cuda")  # (seq, touched, page)
    row = (starts[:-1, None, None] + token - old[:, None, None]).clamp(0, st["k_new"].shape[0] - 1)
    fresh = ((token >= old[:, None, None]) & (token < lengths[:, None, None]))[:, :, None, :, None]
    kept = (token < old[:, None, None])[:, :, None, :, None]
    for name, x in (("k", _heads(st["k_new"], hd, st, True)), ("v", _heads(st["v_new"], hd, st, False))):
        codes, scale = cache[name][0], cache[name + "_scale"][0]
        safe = ids.clamp(min=0)
        x = x[row].transpose(2, 3)  # (seq, touched, kv, page, hd)
        x = torch.where(fresh, x, torch.zeros_like(x))
        was = codes[safe]
        had = (at * page < old[:, None])[..., None]
        s_old = torch.where(had, scale[safe], torch.full_like(scale[safe], 2.0**-126))
        s = torch.maximum(s_old, _step(x.abs().amax((-1, -2))))
        sx = s[..., None, None]
        got = torch.where(fresh, torch.round(x / sx).clamp(-127, 127), torch.round(was.float() * (s_old[..., None, None] / sx)))
        got = torch.where(fresh | kept, got, was.float()).to(torch.int8)
        # pages that no sequence touches here are written back to the page of the same name only
        codes.index_copy_(0, torch.where(live, safe, safe[:1, :1]).reshape(-1), torch.where(live[..., None, None, None], got, got[:1, :1]).flatten(0, 1))
        scale.index_copy_(0, torch.where(live, safe, safe[:1, :1]).reshape(-1), torch.where(live[..., None], s, s[:1, :1]).flatten(0, 1))
    s, p = _where(st["read_starts"].long(), st["read_rows"])
    tok = p + st["first"].long()[s]
    ids = cache["table"].long()[s, tok // page]
    read = [cache[n][0][ids, :, tok % page].float() * cache[n + "_scale"][0][ids][..., None] for n in ("k", "v")]
    return {"k": read[0].flatten(1).to(torch.bfloat16), "v": read[1].flatten(1).to(torch.bfloat16)}


def _plain_pages(st: dict) -> torch.Tensor:
    c, cache = st["case"], st["cache"]
    kv, hd, page, heads, rows = c["kv"], c["hd"], c["page"], c["heads"], c["rows"]
    lengths = cache["lengths"].long()
    b = lengths.shape[0]
    ids = cache["table"].long().clamp(min=0)
    k, v = (
        (cache[n][0][ids].float() * cache[n + "_scale"][0][ids][..., None, None]).transpose(1, 2).reshape(b, kv, -1, hd)
        for n in ("k", "v")
    )
    q = _heads(st["q"], hd, st, True).reshape(b, rows, heads, hd)
    j, i = torch.arange(k.shape[2], device="cuda"), torch.arange(rows, device="cuda")
    seen = j[None, None] < lengths[:, None, None]
    if c["causal"]:
        seen = seen & (j[None, None] <= (lengths[:, None] - rows + i[None])[:, :, None])
    seen = seen.expand(b, rows, -1)[:, None, None].expand(-1, 1, heads // kv, -1, -1).reshape(b, 1, heads // kv * rows, -1)
    o = _softmax_v(_grouped(q, kv), k, v, seen)
    o = o.reshape(b, kv, heads // kv, rows, hd).permute(0, 3, 1, 2, 4)
    return o.reshape(b * rows, heads * hd).to(torch.bfloat16)


def _state(cache: dict) -> dict:
    """Pages move as bytes: codes and scales come back as they are held."""
    return {k: cache[k] for k in ("k", "v", "k_scale", "v_scale", "table", "lengths", "refs")}


def _plain_fork(st: dict) -> dict:
    cache, page = st["cache"], st["case"]["page"]
    table, lengths, refs = cache["table"], cache["lengths"], cache["refs"]
    par, chi = st["parents"].long(), st["children"].long()
    at = torch.arange(table.shape[1], device="cuda")[None]
    # the children's pages go back first
    held = at < ((lengths[chi] + page - 1) // page)[:, None]
    refs.index_add_(0, table[chi].long().clamp(min=0).flatten(), -held.to(refs.dtype).flatten())
    # whole pages are shared, a part-filled one is copied into the lowest free pages in order
    length = lengths[par]
    whole, part = (length // page)[:, None], (length % page > 0)[:, None]
    shared = at < whole
    rows = table[par]
    refs.index_add_(0, rows.long().clamp(min=0).flatten(), shared.to(refs.dtype).flatten())
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    fresh = free[(part[:, 0].long().cumsum(0) - 1).clamp(min=0)]
    table[chi] = torch.where(shared, rows, torch.where((at == whole) & part, fresh[:, None].to(table.dtype), torch.full_like(rows, -1)))
    refs.index_add_(0, fresh, part[:, 0].to(refs.dtype))
    lengths[chi] = length
    src = rows.gather(1, whole.long().clamp(max=table.shape[1] - 1))[:, 0].long().clamp(min=0)
    dst = torch.where(part[:, 0], fresh, src)
    for n in ("k", "v", "k_scale", "v_scale"):
        cache[n].index_copy_(1, dst, cache[n].index_select(1, src))
    return _state(cache)


def _plain_compact(st: dict) -> dict:
    cache = st["cache"]
    refs = cache["refs"]
    n = refs.shape[0]
    at = torch.arange(n, device="cuda")
    live = refs > 0
    count = live.sum()
    high, hole = live & (at >= count), ~live & (at < count)
    moves = at < high.sum()
    src, dst = torch.argsort((~high).to(torch.int8), stable=True), torch.argsort((~hole).to(torch.int8), stable=True)
    to = at.clone().scatter_(0, src, torch.where(moves, dst, src))  # a page's new number
    take = at.clone().scatter_(0, dst, torch.where(moves, src, dst))  # what a page's bytes come from
    for k in ("k", "v", "k_scale", "v_scale"):
        cache[k].copy_(cache[k].index_select(1, take))
    refs.copy_(torch.where(at < count, refs[take], torch.zeros_like(refs)))
    t = cache["table"]
    t.copy_(torch.where(t >= 0, to[t.long().clamp(min=0)].to(t.dtype), t))
    return _state(cache)


# -------------------------------------------------------------------------------------------------- runs


def _own(st: dict):
    from so101_smolvla_edge_b200 import ops

    c, op = st["case"], st["op"]
    cos, sin = st.get("cos"), st.get("sin")
    if op == "prompt":
        return ops.attention_packed(st["q"], st["k"], st["v"], st["starts"], st["max_len"], c["heads"], c["kv"], cos=cos, sin=sin)
    pages = st["pages"]
    if op == "append":
        ops.kv_append(pages, 0, st["k_new"], st["v_new"], st["starts"], max_new=st["max_new"], cos=cos, sin=sin)
        k, v = ops.kv_read(pages, 0, st["read_starts"], st["read_rows"], first=st["first"])
        return {"k": k, "v": v}
    if op == "pages":
        starts = None if c["rows"] == 1 else st["starts"]
        return ops.attention_pages(st["q"], pages, 0, c["heads"], starts, max_q=c["rows"], causal=c["causal"], cos=cos, sin=sin)
    if op == "fork":
        ops.kv_free(pages, st["children"])
        ops.kv_fork(pages, st["parents"], st["children"])
    else:
        ops.kv_compact(pages)
    return _state(st["cache"])


def run(st: dict):
    if st["op"] == "compact":
        for k, t in st["snapshot"].items():
            st["cache"][k].copy_(t)
    if own:
        return _own(st)
    return {"prompt": _plain_prompt, "append": _plain_append, "pages": _plain_pages, "fork": _plain_fork, "compact": _plain_compact}[st["op"]](st)


def work(case: dict) -> dict:
    op, hd, kv = case["op"], case["hd"], case["kv"]
    if op == "prompt":
        lens, heads = _lens(case), case["heads"]
        rows = sum(lens)
        byte = rows * (2 * heads + 2 * kv) * hd * 2 + (rows * hd * 4 if case["rope"] else 0) + 4 * (len(lens) + 1)
        return {"bytes": byte, "flops": 4 * hd * heads * sum(n * (n + 1) // 2 for n in lens)}
    if op == "append":
        new, old, page = _lens(case), _old(case), case["page"]
        rows, kept = sum(new), sum(o % page for o in old)
        one = 2 * kv * hd
        # new rows in, their codes out, codes of part-filled pages in and out, and the touched pages as rows
        return {"bytes": rows * one * 3 + kept * one * 2 + (rows + kept) * one * 2 + (rows * hd * 4 if case["rope"] else 0), "flops": 8 * rows * one}
    if op == "pages":
        lens, rows, heads = _lens(case), case["rows"], case["heads"]
        pages_of = [-(-n // case["page"]) for n in lens]
        q = len(lens) * rows * heads * hd * 4 + (len(lens) * rows * hd * 4 if case["rope"] else 0)
        return {"bytes": 2 * sum(lens) * kv * hd + sum(pages_of) * (8 * kv + 4) + q, "flops": 4 * hd * heads * rows * sum(lens)}
    each = -(-case["length"] // case["page"])
    page_bytes = case["layers"] * kv * (2 * case["page"] * hd + 8)
    if op == "fork":
        n = case["parents"] * case["children"]
        return {"bytes": (2 * page_bytes * n if case["length"] % case["page"] else 0) + 12 * n * (each + 1) + 4 * case["pool"], "flops": 0}
    live = max(1, round(case["live"] * case["seqs"])) * each
    # of the live pages, scattered evenly, those past the live count move
    return {"bytes": 2 * page_bytes * max(1, round(live * (1 - live / case["pool"]))) + 8 * case["pool"] + 8 * case["seqs"] * each, "flops": 0}


# ------------------------------------------------------------------------------------- values in 64 bits


def _attend64(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, last: torch.Tensor) -> torch.Tensor:
    """One head in 64 bits: row i of q sees keys 0 .. last[i]."""
    out = torch.zeros_like(q)
    for r in range(0, q.shape[0], 2048):
        s = q[r : r + 2048] @ k.T / q.shape[1] ** 0.5
        hide = torch.arange(k.shape[0], device=q.device)[None] > last[r : r + 2048, None]
        s[hide] = -torch.inf
        p = torch.softmax(s, -1)
        p[last[r : r + 2048] < 0] = 0
        out[r : r + 2048] = p @ v
    return out


def _turn64(x: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None) -> torch.Tensor:
    x = x.double()
    if cos is None:
        return x
    h = x.shape[-1] // 2
    y = x.clone()
    y[..., :h] = x[..., :h] * cos.double() - x[..., h:] * sin.double()
    y[..., h:] = x[..., h:] * cos.double() + x[..., :h] * sin.double()
    return y


def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op, hd, kv = case["op"], case["hd"], case["kv"]
    cos, sin = st.get("cos"), st.get("sin")
    if op == "prompt":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        starts, group = st["starts"].tolist(), case["heads"] // kv
        for a, b in zip(starts, starts[1:]):
            for h in range(case["heads"]):
                q = _turn64(st["q"][a:b, h * hd : (h + 1) * hd], *(None if t is None else t[a:b] for t in (cos, sin)))
                g = h // group
                k, v = (st[n][a:b, g * hd : (g + 1) * hd].double() for n in ("k", "v"))
                out[a:b, h * hd : (h + 1) * hd] = _attend64(q, k, v, torch.arange(b - a, device="cuda"))
        return out
    cache = st["cache"]
    if op == "pages":
        rows, page, group = case["rows"], case["page"], case["heads"] // kv
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(cache["lengths"].tolist()):
            ids = cache["table"][i, : -(-n // page)].long()
            a, b = i * rows, (i + 1) * rows
            last = torch.arange(n - rows, n, device="cuda") if case["causal"] else torch.full((rows,), n - 1, device="cuda")
            for g in range(kv):
                k, v = (
                    (cache[t][0][ids, g].double() * cache[t + "_scale"][0][ids, g].double()[:, None, None]).reshape(-1, hd)[:n]
                    for t in ("k", "v")
                )
                for h in range(g * group, (g + 1) * group):
                    q = _turn64(st["q"][a:b, h * hd : (h + 1) * hd], *(None if t is None else t[a:b] for t in (cos, sin)))
                    out[a:b, h * hd : (h + 1) * hd] = _attend64(q, k, v, last)
        return out
    if op == "append":
        page = case["page"]
        starts, first = st["starts"].tolist(), st["first"].tolist()
        lengths, table = cache["lengths"].tolist(), cache["table"].tolist()
        got = {}
        for name in ("k", "v"):
            rows = []
            x = st[name + "_new"].reshape(-1, kv, hd)
            turn = (cos[:, None], sin[:, None]) if name == "k" and cos is not None else (None, None)
            x = _turn64(x, *turn).cpu()
            codes, scale = cache[name][0].cpu(), cache[name + "_scale"][0].double().cpu()
            for i, n in enumerate(lengths):
                old = n - (starts[i + 1] - starts[i])
                for p in range(first[i] // page, -(-n // page)):
                    lo, hi = p * page, min(n, (p + 1) * page)
                    held = max(0, old - lo)
                    fresh = x[starts[i] + lo + held - old : starts[i] + hi - old]
                    big = fresh.abs().amax((0, 2))
                    s = 2.0 ** torch.ceil(torch.log2(big.clamp(min=1e-300) / 127)).clamp(-126, 121)
                    before = codes[table[i][p], :, :held].double().transpose(0, 1) * scale[table[i][p]][None, :, None]
                    if held:
                        s = torch.maximum(s, scale[table[i][p]])
                    both = torch.cat([before, fresh])
                    rows.append((torch.round(both / s[None, :, None]).clamp(-127, 127) * s[None, :, None]).flatten(1))
            got[name] = torch.cat(rows)
        return got
    page = case["page"]
    table, lengths, refs = cache["table"].tolist(), cache["lengths"].tolist(), cache["refs"].tolist()
    moves = []
    if op == "fork":
        for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
            for t in range(lengths[p] // page):
                refs[table[p][t]] += 1
        for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
            whole = lengths[p] // page
            table[c] = [table[p][t] if t < whole else -1 for t in range(len(table[p]))]
            if lengths[p] % page:
                new = refs.index(0)
                refs[new] = 1
                table[c][whole] = new
                moves.append((table[p][whole], new))
            lengths[c] = lengths[p]
    else:
        live = sum(r > 0 for r in refs)
        high = [i for i, r in enumerate(refs) if r > 0 and i >= live]
        holes = [i for i, r in enumerate(refs) if r == 0 and i < live]
        to = dict(zip(high, holes))
        for s, d in to.items():
            refs[d], refs[s] = refs[s], 0
        table = [[to.get(t, t) for t in row] for row in table]
        moves = list(to.items())
    out = {k: cache[k] for k in ("k", "v", "k_scale", "v_scale")}
    if moves:
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*moves))
        for t in out.values():
            t[:, dst] = t[:, src]
    for n in ("k_scale", "v_scale"):
        out[n] = out[n].double()
    return out | {"table": torch.tensor(table), "lengths": torch.tensor(lengths), "refs": torch.tensor(refs)}
