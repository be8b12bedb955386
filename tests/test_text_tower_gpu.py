"""The text tower over the paged cache against the same layers in float32, recomputed whole for every sequence.

Tolerances are relative 2-norms of the hidden states. Prompts: bf16 activations, rounded about six times per layer by at
most 2^-8 each, independent, over 4 layers: sqrt(24) 2^-8 = 1.9e-2. Tokens over the 8-bit cache: a step of
the codes is at most amax / 63.5, its rounding error 1 / sqrt(12) of that, with amax about four deviations 1.8e-2 of the
cached values, in keys and values of every layer: sqrt(1.9^2 + 8 * 1.8^2) e-2 = 5.4e-2 if nothing averaged out.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.smolvla_fp32 import gqa, rms_norm, rope, rope_tables

pytestmark = pytest.mark.gpu
PROMPT, TOKEN = 1.9e-2, 5.4e-2


@pytest.fixture(scope="module")
def bundle():
    from so101_smolvla_edge_b200.bundle import seeded_bundle
    from so101_smolvla_edge_b200.spec import ModelSpec

    spec = ModelSpec(n_cams=2, image_size=128, vis_dim=128, vis_layers=1, vis_heads=2, vis_mlp=256, text_dim=384,
                     n_layers=4, n_heads=6, n_kv=2, head_dim=64, text_mlp=256, exp_dim=96, exp_mlp=256, chunk=10,
                     max_state=8, max_action=8, n_steps=3, lang_len=5)  # fmt: skip
    return seeded_bundle(spec, seed=7, image_hw=(120, 160), state_dim=6, action_dim=6, style="test")


def plain(b, rows):
    """The layers over one sequence's rows (n, text_dim), causal, float32."""
    s, w = b.spec, {k: torch.from_numpy(np.ascontiguousarray(v)) for k, v in b.tensors.items()}
    n = rows.shape[0]
    cos, sin = rope_tables(torch.arange(n), s.head_dim, s.rope_wavelength)
    seen = torch.tril(torch.ones(n, n, dtype=torch.bool))
    x = rows.clone()
    for i in range(s.n_layers):
        t = f"txt.{i}."
        q, k, v = (rms_norm(x, w[t + "ln_in"], s.rms_eps) @ w[t + "qkv"].T).split([s.q_dim, s.kv_dim, s.kv_dim], -1)
        q = rope(q.reshape(n, s.n_heads, -1), cos, sin)
        k = rope(k.reshape(n, s.n_kv, -1), cos, sin)
        x = x + gqa(q, k, v.reshape(n, s.n_kv, -1), seen) @ w[t + "o"].T
        g, u = (rms_norm(x, w[t + "ln_post"], s.rms_eps) @ w[t + "gate_up"].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ w[t + "down"].T
    return x


def off(got, want):
    return float((got.cpu().float() - want).norm() / want.norm())


def test_prompts_forks_and_tokens(bundle):
    from so101_smolvla_edge_b200 import ops
    from so101_smolvla_edge_b200.text_tower import TextTower

    g = torch.Generator().manual_seed(1)
    tower = TextTower(bundle, n_pages=24, max_seqs=8, max_len=256, page=32)
    dim = bundle.spec.text_dim
    lens = [70, 1, 32]
    text = {q: torch.randn(n, dim, generator=g) for q, n in zip((5, 0, 2), lens)}
    got = tower.prompt(torch.cat(list(text.values())).cuda(), lens, [5, 0, 2])
    want = torch.cat([plain(bundle, x) for x in text.values()])
    assert off(got, want) <= PROMPT
    # two continuations of one prompt, one of another; the parents go on too
    tower.fork([5, 5, 2], [1, 3, 4])
    for c, p in ((1, 5), (3, 5), (4, 2)):
        text[c] = text[p]
    for turn in range(3):
        seqs = [3, 0, 1, 5, 4] if turn else [5, 1, 2]
        rows = torch.randn(len(seqs), dim, generator=g)
        got = tower.step(rows.cuda(), seqs)
        for i, q in enumerate(seqs):
            text[q] = torch.cat([text[q], rows[i : i + 1]])
            assert off(got[i], plain(bundle, text[q])[-1]) <= TOKEN, (turn, q)
    # some end, the rest move together; several tokens at once after that
    tower.free([5, 0])
    tower.compact()
    seqs, counts = [4, 1, 2], [3, 7, 1]
    rows = torch.randn(sum(counts), dim, generator=g)
    got = tower.step(rows.cuda(), seqs, counts)
    at = 0
    for q, n in zip(seqs, counts):
        text[q] = torch.cat([text[q], rows[at : at + n]])
        assert off(got[at : at + n], plain(bundle, text[q])[-n:]) <= TOKEN, q
        at += n
    tower.check()
    live = [q for q in range(8) if tower.lengths[q]]
    assert tower.pages.lengths.tolist() == tower.lengths and live == [1, 2, 3, 4]
    refs = tower.pages.refs.tolist()
    assert 0 not in refs[: sum(r > 0 for r in refs)]
    k, v = tower.cached(1, 4)
    assert k.shape == v.shape == (tower.lengths[4], bundle.spec.kv_dim)
    assert ops.device_status() == 0


def test_refusals(bundle):
    from so101_smolvla_edge_b200 import _lib as L
    from so101_smolvla_edge_b200.text_tower import TextTower

    tower = TextTower(bundle, n_pages=2, max_seqs=3, max_len=64, page=32)
    dim = bundle.spec.text_dim
    x = torch.zeros(70, dim, device="cuda")
    with pytest.raises(ValueError):
        tower.prompt(x, [70], [0])  # past max_len
    with pytest.raises(ValueError):
        tower.prompt(x[:4], [2, 1], [0, 1])
    with pytest.raises(ValueError):
        tower.prompt(x[:4], [2, 2], [0, 0])
    tower.prompt(x[:33], [33], [0])
    with pytest.raises(ValueError):
        tower.prompt(x[:1], [1], [0])
    with pytest.raises(ValueError):
        tower.fork([0], [0])
    tower.check()
    tower.step(x[:1], [1])  # both pages are taken
    with pytest.raises(L.KernelError):
        tower.check()
    L.lib().so101_clear_device_status()
