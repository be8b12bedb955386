"""The paged 8-bit K/V cache: the handle that `ops.kv_*` and `ops.attention_pages` work on.

Token t of sequence s lies in page `table[s, t // page]`, slot `t % page`; one page number serves every
layer. Codes are int8, `k[layer, page, head, slot, dim]`, and every (layer, page, kv head) has one
power-of-two scale for its keys and one for its values, so a value is `code * scale` exactly.
`refs[p]` counts the sequences that hold page p: forked sequences share their whole pages. Everything
lives on the device and nothing here reads it back, so a serving loop never waits for the GPU.

The reference (so101-smolvla-edge) keeps one bf16 buffer of a fixed size per engine
(model/smolvla_triton.py:9-17); it has no counterpart.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

PAGE_SIZES = (16, 32, 64)
HEAD_DIMS = (64, 128)


class KvPages:
    """Cache arrays and their C descriptor. `KvPages(...)` allocates; `KvPages.adopt(...)` takes arrays."""

    def __init__(self, n_layers: int, n_pages: int, n_kv: int, head_dim: int, max_seqs: int, max_len: int,
                 page: int = 64, device: torch.device | str = "cuda"):  # fmt: skip
        if page not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, not {page}, {head_dim}")
        if min(n_layers, n_pages, n_kv, max_seqs, max_len) < 1:
            raise ValueError("n_layers, n_pages, n_kv, max_seqs and max_len must be positive")
        codes = (n_layers, n_pages, n_kv, page, head_dim)
        self._take(
            torch.zeros(codes, dtype=torch.int8, device=device), torch.zeros(codes, dtype=torch.int8, device=device),
            torch.zeros(codes[:3], dtype=torch.float32, device=device),
            torch.zeros(codes[:3], dtype=torch.float32, device=device),
            torch.full((max_seqs, -(-max_len // page)), -1, dtype=torch.int32, device=device),
            torch.zeros(max_seqs, dtype=torch.int32, device=device),
            torch.zeros(n_pages, dtype=torch.int32, device=device),
        )  # fmt: skip

    @classmethod
    def adopt(cls, k, v, k_scale, v_scale, table, lengths, refs) -> "KvPages":
        """A handle on existing arrays (they stay the caller's, and are updated in place)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale, table, lengths, refs)
        return self

    def _take(self, k, v, k_scale, v_scale, table, lengths, refs) -> None:
        if k.dim() != 5 or k.shape[3] not in PAGE_SIZES or k.shape[4] not in HEAD_DIMS:
            raise ValueError(f"k must be (layers, pages, heads, slots, dims) with {PAGE_SIZES} slots and {HEAD_DIMS} dims")
        for name, t, dtype, shape in (
            ("k", k, torch.int8, k.shape), ("v", v, torch.int8, k.shape),
            ("k_scale", k_scale, torch.float32, k.shape[:3]), ("v_scale", v_scale, torch.float32, k.shape[:3]),
            ("table", table, torch.int32, (lengths.numel(), table.shape[-1])),
            ("lengths", lengths, torch.int32, (lengths.numel(),)), ("refs", refs, torch.int32, (k.shape[1],)),
        ):  # fmt: skip
            if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} of shape {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
            if t.device != k.device or t.device.type != "cuda":
                raise ValueError("the cache's arrays must lie on one CUDA device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.lengths, self.refs = table, lengths, refs
        self.device = k.device
        self.n_layers, self.n_pages, self.n_kv, self.page, self.head_dim = k.shape
        self.max_seqs, self.max_pages = table.shape
        self.desc = L.KvPages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), table.data_ptr(),
                              lengths.data_ptr(), refs.data_ptr(), None, *k.shape, *table.shape)  # fmt: skip
        ints = C.c_int64()
        L.check(L.lib().so101_kv_scratch(C.byref(self.desc), C.byref(ints)), "so101_kv_scratch")
        self.scratch = torch.zeros(ints.value, dtype=torch.int32, device=k.device)
        self.desc.scratch = self.scratch.data_ptr()
        # what the calls take: the descriptor's address and the device
        self.handle = (C.addressof(self.desc), k.device.index)

    @property
    def max_len(self) -> int:
        """The most tokens that a sequence can hold."""
        return self.max_pages * self.page
