"""The serving operators' C ABI without a GPU: exports, bindings and what is refused before the device is touched."""

from __future__ import annotations

import ctypes as C
import math

import pytest

from so101_smolvla_edge_b200 import _lib as L

FAKE = 1 << 20  # never dereferenced: every call below fails its host-side checks, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def pages(**kw):
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, table=FAKE, lengths=FAKE, refs=FAKE, scratch=FAKE, n_layers=2,
             n_pages=8, n_kv=2, page=16, hd=64, max_seqs=4, max_pages=4)  # fmt: skip
    a.update(kw)
    return C.byref(L.KvPages(*a.values()))


def test_header_is_exported_and_bound(lib):
    names = L.header_symbols(L.TEXT_HEADER)
    assert len(names) == 10 and all(hasattr(lib, n) for n in names)
    assert set(names) <= set(L.SIGNATURES)
    assert f"#define SO101_ERR_PAGES {L.ERR_PAGES}" in L.TEXT_HEADER.read_text()


def test_call_module_loads():
    calls = L.calls()
    assert {"attention_packed", "attention_pages", "kv_append", "kv_read", "kv_compact"} <= set(dir(calls))
    with pytest.raises(TypeError):
        calls.kv_compact()
    with pytest.raises(ValueError):
        calls.kv_free((0, 0), None)


BAD_PAGES = [dict(k=None), dict(scratch=None), dict(v=FAKE + 8), dict(k_scale=FAKE + 4), dict(page=48), dict(page=128), dict(hd=96),
             dict(hd=32), dict(n_kv=0), dict(n_pages=0), dict(n_pages=(1 << 20) + 1), dict(max_pages=1 << 27)]  # fmt: skip


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_cache_handles_are_checked(lib, bad):
    c = pages(**bad)
    assert lib.so101_kv_append(c, 0, FAKE, 128, FAKE, 128, 4, FAKE, None, 1, 4, None, None, None) == L.ERR_ARG
    assert lib.so101_kv_read(c, 0, FAKE, None, None, 1, 4, FAKE, 128, FAKE, 128, None) == L.ERR_ARG
    assert lib.so101_attention_pages(FAKE, 256, FAKE, 256, 4, c, 0, 4, FAKE, None, 1, 4, 1, 0.1, None, None, FAKE, 1 << 20, FAKE,
                                     1 << 10, None) == L.ERR_ARG  # fmt: skip
    assert lib.so101_kv_reserve(c, FAKE, FAKE, 1, None) == L.ERR_ARG
    assert lib.so101_kv_free(c, FAKE, 1, None) == L.ERR_ARG
    assert lib.so101_kv_fork(c, FAKE, FAKE, 1, None) == L.ERR_ARG
    assert lib.so101_kv_copy(c, FAKE, FAKE, 1, None) == L.ERR_ARG
    assert lib.so101_kv_compact(c, None) == L.ERR_ARG


def test_attention_packed_arguments(lib):
    def call(**kw):
        a = dict(q=FAKE, ldq=640, k=FAKE, ldk=640, v=FAKE, ldv=640, o=FAKE, ldo=256, rows=10, starts=FAKE, n=1, most=10, nq=4,
                 nkv=2, hd=64, scale=0.125, cos=None, sin=None)  # fmt: skip
        a.update(kw)
        return lib.so101_attention_packed(*a.values(), None)

    for bad in (dict(q=None), dict(starts=None), dict(hd=32), dict(hd=80), dict(nq=3), dict(nkv=0), dict(q=FAKE + 8), dict(ldk=641),
                dict(ldo=128), dict(ldq=128), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
                dict(cos=FAKE), dict(cos=FAKE + 4, sin=FAKE), dict(rows=-1), dict(n=-1), dict(rows=1 << 30, nq=4)):  # fmt: skip
        assert call(**bad) == L.ERR_ARG, bad
    assert call(rows=0) == L.OK and call(n=0) == L.OK


def test_attention_pages_arguments(lib):
    def call(**kw):
        a = dict(q=FAKE, ldq=256, o=FAKE, ldo=256, rows=4, c=pages(), layer=1, nq=4, starts=FAKE, seqs=None, n=2, most=3, causal=1,
                 scale=0.125, cos=None, sin=None, ws=FAKE, ws_bytes=1 << 22, tick=FAKE, n_tick=1 << 10)  # fmt: skip
        a.update(kw)
        return lib.so101_attention_pages(*a.values(), None)

    for bad in (dict(q=None), dict(layer=2), dict(layer=-1), dict(nq=3), dict(q=FAKE + 8), dict(ldq=252), dict(ldo=128),
                dict(o=FAKE + 2), dict(starts=None), dict(most=0), dict(scale=0.0), dict(sin=FAKE), dict(n=-1)):  # fmt: skip
        assert call(**bad) == L.ERR_ARG, bad
    assert call(ws=None) == L.ERR_WORKSPACE and call(tick=None) == L.ERR_WORKSPACE
    assert call(rows=0, n=0) == L.OK
    assert call(starts=None, rows=2, most=2) == L.ERR_ARG  # one row per sequence, so max_q is 1


def test_append_read_and_lists_arguments(lib):
    c = pages()
    append = lambda **kw: lib.so101_kv_append(*{**dict(c=c, layer=0, k=FAKE, ldk=256, v=FAKE, ldv=256, rows=4, starts=FAKE, seqs=None,  # noqa: E731
                                                       n=2, most=3, cos=None, sin=None), **kw}.values(), None)  # fmt: skip
    for bad in (dict(k=None), dict(layer=2), dict(ldk=120), dict(ldv=250), dict(k=FAKE + 2), dict(most=0), dict(starts=None),
                dict(cos=FAKE), dict(cos=FAKE + 8, sin=FAKE), dict(n=70000)):  # fmt: skip
        assert append(**bad) == L.ERR_ARG, bad
    assert append(rows=0) == L.OK
    read = lambda **kw: lib.so101_kv_read(*{**dict(c=c, layer=0, starts=FAKE, seqs=None, first=None, n=2, rows=4, k=FAKE, ldk=128,  # noqa: E731
                                                   v=FAKE, ldv=128), **kw}.values(), None)  # fmt: skip
    for bad in (dict(starts=None), dict(layer=-1), dict(k=FAKE + 8), dict(ldk=64), dict(ldv=132), dict(rows=-1)):
        assert read(**bad) == L.ERR_ARG, bad
    assert read(rows=0) == L.OK
    for fn in (lib.so101_kv_reserve, lib.so101_kv_fork):
        assert fn(c, None, FAKE, 1, None) == L.ERR_ARG and fn(c, FAKE, FAKE, 5, None) == L.ERR_ARG  # more than max_seqs
        assert fn(c, FAKE, FAKE, -1, None) == L.ERR_ARG and fn(c, None, None, 0, None) == L.OK
    assert lib.so101_kv_copy(c, FAKE, FAKE, 9, None) == L.ERR_ARG  # more than n_pages
    assert lib.so101_kv_free(c, None, 1, None) == L.ERR_ARG and lib.so101_kv_free(c, None, 0, None) == L.OK
    got = C.c_int64()
    assert lib.so101_kv_scratch(c, C.byref(got)) == L.OK and got.value >= 3 * 8
    assert lib.so101_kv_scratch(c, None) == L.ERR_ARG
