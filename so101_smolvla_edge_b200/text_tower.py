"""The bundle's text tower as a serving loop: packed prompts, an 8-bit paged cache, forks, single tokens.

    python -m so101_smolvla_edge_b200.text_tower [BUNDLE]

`Engine` runs the tower once per chunk, over prefix rows of one fixed length, into caches of its own. `TextTower`
runs the same layers over prompts of any lengths packed end to end, causally, and keeps their keys and
values in `pages.KvPages`, so that sequences can go on token by token, share a prompt (several
continuations or noise samples of one observation) and give their memory back:

    tower = TextTower(bundle, n_pages=512, max_seqs=64, max_len=1024)
    rows = tower.prompt(embedded_rows, lengths=[241, 177], seqs=[0, 1])     # all rows' hidden states
    tower.fork([0, 0, 1], [2, 3, 4])                                        # continuations share pages
    rows = tower.step(next_rows, seqs=[2, 3, 4])                            # one token each
    tower.free([2, 3]); tower.compact()

The layers are the reference's prefix layers (pkg/model/smolvla_triton.py:78-103: RMSNorm, fused q|k|v, RoPE, attention,
output projection, SwiGLU), but under a causal mask, as a language model runs them; in the policy's prefix images
and task tokens see each other. From the second layer on the hidden states, keys and values are therefore not those
that the policy's action expert was trained on: its chunks come from `Engine`. A bundle holds neither a token embedding nor an output
head, so rows come in embedded and go out as hidden states. The cache and its sharing have no counterpart in the reference.
"""

from __future__ import annotations

import argparse
import functools
import time

import torch

from . import _lib as L
from . import ops
from .bundle import Bundle, load_bundle, seeded_bundle
from .pages import HEAD_DIMS, KvPages
from .path import Packed, _rope
from .spec import ModelSpec


def _here(method):
    """A method with its tower's device current, which is where the library launches."""

    @functools.wraps(method)
    def run(self, *args, **kwargs):
        with torch.cuda.device(self.dev):
            return method(self, *args, **kwargs)

    return run


class TextTower:
    """The text layers of a bundle over a cache of `n_pages` pages for `max_seqs` sequences."""

    def __init__(self, bundle, n_pages: int, max_seqs: int, max_len: int, page: int = 64, device: str = "cuda"):
        self.b: Bundle = load_bundle(bundle)
        self.spec: ModelSpec = self.b.spec
        if self.spec.head_dim not in HEAD_DIMS:
            raise ValueError(f"the paged cache takes head_dim {HEAD_DIMS}, not {self.spec.head_dim}")
        self.dev = torch.device(device)
        if self.dev.index is None:
            self.dev = torch.device("cuda", torch.cuda.current_device())
        with torch.cuda.device(self.dev):
            self.packed = Packed.get(self.b, self.dev, (), L.lib())
            self.w = self.packed.w
            s = self.spec
            self.pages = KvPages(s.n_layers, n_pages, s.n_kv, s.head_dim, max_seqs, max_len, page, self.dev)
            self.cos, self.sin = (t.to(self.dev) for t in _rope(torch.arange(self.pages.max_len), s.head_dim, s.rope_wavelength))
        self.lengths = [0] * max_seqs  # the host's own count: what the next positions are

    def _put(self, *lists) -> tuple[torch.Tensor, ...]:
        """Lists of integers on the device, in one copy from pinned memory that the host does not wait for."""
        parts = [torch.as_tensor(x, dtype=torch.int32) for x in lists]
        sizes = [x.numel() for x in parts]
        host = torch.cat(parts, out=torch.empty(sum(sizes), dtype=torch.int32, pin_memory=True))
        return host.to(self.dev, non_blocking=True).split(sizes)

    def _grow(self, seqs: list[int], counts: list[int]) -> tuple[torch.Tensor, ...]:
        """Pages for `counts` more tokens. Returns the sequences' numbers, the packed starts and the new tokens' angles, on
        the device. A sequence that a refused call (of which only `check` tells the host) left shorter than this object
        counts asks for more than there can be, so that the calls after it are refused too, and nothing is cached at a place
        that is not its own."""
        held = [self.lengths[s] for s in seqs]
        starts = [0, *torch.tensor(counts).cumsum(0).tolist()]
        at = torch.cat([torch.arange(h, h + n, dtype=torch.int32) for h, n in zip(held, counts)])
        ids, more, held, starts, at = self._put(seqs, counts, held, starts, at)
        behind = self.pages.lengths[ids] != held
        ops.kv_reserve(self.pages, ids, torch.add(more, behind, alpha=1 << 30))
        for s, n in zip(seqs, counts):
            self.lengths[s] += n
        return ids, starts, self.cos[at], self.sin[at]

    def _check_seqs(self, what: str, seqs: list[int]) -> None:
        if not all(0 <= s < len(self.lengths) for s in seqs):
            raise ValueError(f"{what} must be sequences of the cache, 0 to {len(self.lengths) - 1}")

    def _check(self, seqs: list[int], counts: list[int], rows: torch.Tensor) -> None:
        self._check_seqs("seqs", seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("seqs must be distinct")
        if len(counts) != len(seqs) or min(counts, default=1) < 1 or rows.shape != (sum(counts), self.spec.text_dim):
            raise ValueError(f"rows must be ({sum(counts)}, {self.spec.text_dim}), at least one per sequence")
        if any(self.lengths[s] + n > self.pages.max_len for s, n in zip(seqs, counts)):
            raise ValueError(f"a sequence would pass {self.pages.max_len} tokens")

    def _mlp(self, i: int, x: torch.Tensor) -> torch.Tensor:
        h = ops.rms_norm(x, self.w[f"txt.{i}.ln_post"], self.spec.rms_eps)
        h = ops.linear(h, self.w[f"txt.{i}.gate_up"], silu_gate=True)
        return ops.linear(h, self.w[f"txt.{i}.down"], residual=x)

    @_here
    def prompt(self, rows: torch.Tensor, lengths: list[int], seqs: list[int]) -> torch.Tensor:
        """Whole prompts of empty sequences, packed end to end: rows (sum(lengths), text_dim), embedded.
        Returns every row's hidden state (float32)."""
        s = self.spec
        self._check(seqs, lengths, rows)
        if not seqs:
            return rows.float()
        if any(self.lengths[q] for q in seqs):
            raise ValueError("a prompt starts an empty sequence")
        ids, starts, cos, sin = self._grow(seqs, lengths)
        most, q_dim = max(lengths), s.q_dim
        x = rows.float()
        k = torch.empty(x.shape[0], s.kv_dim, dtype=torch.bfloat16, device=self.dev)
        for i in range(s.n_layers):
            qkv = ops.linear(ops.rms_norm(x, self.w[f"txt.{i}.ln_in"], s.rms_eps), self.w[f"txt.{i}.qkv"])
            ops.rope_kv(qkv, s.n_heads, s.n_kv, cos, sin, k)
            v = qkv[:, q_dim + s.kv_dim :]
            ops.kv_append(self.pages, i, qkv[:, q_dim : q_dim + s.kv_dim], v, starts, ids, max_new=most, cos=cos, sin=sin)
            a = ops.attention_packed(qkv[:, :q_dim], k, v, starts, most, s.n_heads, s.n_kv, cos=cos, sin=sin)
            x = self._mlp(i, ops.linear(a, self.w[f"txt.{i}.o"], residual=x))
        return x

    @_here
    def step(self, rows: torch.Tensor, seqs: list[int], counts: list[int] | None = None) -> torch.Tensor:
        """The next tokens of sequences that hold some: one row each, or `counts` (drafted tokens, the rest of a
        prompt). Returns their hidden states (float32)."""
        s = self.spec
        single = counts is None
        counts = [1] * len(seqs) if single else counts
        self._check(seqs, counts, rows)
        if not seqs:
            return rows.float()
        ids, starts, cos, sin = self._grow(seqs, counts)
        starts = None if single else starts
        most, q_dim = max(counts), s.q_dim
        x = rows.float()
        for i in range(s.n_layers):
            qkv = ops.linear(ops.rms_norm(x, self.w[f"txt.{i}.ln_in"], s.rms_eps), self.w[f"txt.{i}.qkv"])
            ops.kv_append(self.pages, i, qkv[:, q_dim : q_dim + s.kv_dim], qkv[:, q_dim + s.kv_dim :], starts, ids,
                          max_new=most, cos=cos, sin=sin)  # fmt: skip
            a = ops.attention_pages(qkv[:, :q_dim], self.pages, i, s.n_heads, starts, ids, max_q=most, cos=cos, sin=sin)
            x = self._mlp(i, ops.linear(a, self.w[f"txt.{i}.o"], residual=x))
        return x

    @_here
    def fork(self, parents: list[int], children: list[int]) -> None:
        """children[i] (empty) goes on from where parents[i] stands."""
        self._check_seqs("parents", parents)
        self._check_seqs("children", children)
        if len(parents) != len(children):
            raise ValueError("there is one parent per child")
        if len(set(children)) != len(children) or any(self.lengths[c] for c in children) or set(parents) & set(children):
            raise ValueError("children must be distinct, empty and no parents")
        ops.kv_fork(self.pages, *self._put(parents, children))
        for p, c in zip(parents, children):
            self.lengths[c] = self.lengths[p]

    @_here
    def free(self, seqs: list[int]) -> None:
        """The sequences give their pages back and are empty."""
        self._check_seqs("seqs", seqs)
        ops.kv_free(self.pages, *self._put(seqs))
        for q in seqs:
            self.lengths[q] = 0

    @_here
    def compact(self) -> None:
        ops.kv_compact(self.pages)

    @_here
    def check(self) -> None:
        """Raise if a call since the last check could not be met (too few free pages). The cache then stands as before
        that call, later calls of its sequences were refused with it (what all of them returned is void), and this
        object counts the lengths that the cache has. Waits for the device: not once per token."""
        torch.cuda.current_stream(self.dev).synchronize()
        status = ops.device_status()
        if status != L.OK:
            ops.clear_device_status()
            self.lengths = self.pages.lengths.tolist()
            L.check(status, "TextTower")

    @_here
    def cached(self, layer: int, seq: int) -> tuple[torch.Tensor, torch.Tensor]:
        """A sequence's cached keys (rotated) and values of one layer, as bf16 rows (of a causal pass: see the top)."""
        self._check_seqs("seq", [seq])
        n = self.lengths[seq]
        starts, ids = self._put([0, n], [seq])
        return ops.kv_read(self.pages, layer, starts, n, ids)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("bundle", nargs="?", help="a bundle directory (default: seeded weights of the default model's text tower)")
    a = ap.parse_args()
    bundle = a.bundle or seeded_bundle(ModelSpec(lang_len=48), seed=7, image_hw=(480, 640), state_dim=6, action_dim=6)
    tower = TextTower(bundle, n_pages=256, max_seqs=32, max_len=512)
    g = torch.Generator(device="cuda").manual_seed(0)
    lengths = [241, 177, 113, 305]
    rows = lambda n: torch.randn(n, tower.spec.text_dim, device="cuda", generator=g)  # noqa: E731

    def timed(what: str, fn, reps: int = 1):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(reps):
            out = fn()
        torch.cuda.synchronize()
        print(f"{what}: {(time.perf_counter() - t) / reps * 1e3:.3f} ms")
        return out

    for _ in range(2):  # the first turn builds what later ones keep
        tower.prompt(rows(sum(lengths)), lengths, [0, 1, 2, 3])
        tower.free([0, 1, 2, 3])
    timed(f"prompts of {lengths} tokens", lambda: tower.prompt(rows(sum(lengths)), lengths, [0, 1, 2, 3]))
    children = list(range(4, 20))
    timed("16 forks", lambda: tower.fork([c % 4 for c in children], children))
    x = timed("a token of each of 16", lambda: tower.step(rows(16), children), reps=20)
    timed("free and compact", lambda: (tower.free(children), tower.compact()))
    tower.check()
    print(f"hidden state {tuple(x.shape)}, finite {bool(x.isfinite().all())}")


if __name__ == "__main__":
    main()
