"""The entries around the K/V cache without a GPU: every contract violation is refused with its code before any HIP
call, empty calls touch nothing, and the workspace queries fit the calls."""
from __future__ import annotations

import ctypes

import pytest

from v7multiplikator_amd import _lib

NULL, SHAPE, ALIGN, ALIAS = _lib.V7G_ERR_NULL, _lib.V7G_ERR_SHAPE, _lib.V7G_ERR_ALIGN, _lib.V7G_ERR_ALIAS
MB = 1 << 20


def at(i):
    """Addresses a gigabyte apart, never dereferenced: validation fails first."""
    return (i + 1) << 30


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def refused(L, want, fn, *args):
    L.v7g_clear_last_error()
    rc = fn(*args)
    assert (rc, L.v7g_get_last_error()) == (want, want)
    L.v7g_clear_last_error()


# ------------------------------------------------------------------------------------------------ attention_prefill

PREFILL = dict(out=at(0), out_stride=512, q=at(1), q_stride=512, k=at(2), k_stride=128, v=at(3), v_stride=128, cu=at(4),
               cuk=None, n_seqs=2, T=600, S=600, Hq=8, Hk=2, D=64, scale=0.1, ws=at(5), ws_bytes=256 * MB)


@pytest.mark.parametrize("change,want", [
    (dict(n_seqs=-1), SHAPE), (dict(T=-1), SHAPE), (dict(S=-1, cuk=at(6)), SHAPE), (dict(S=599), SHAPE),
    (dict(Hq=7), SHAPE), (dict(Hq=0), SHAPE), (dict(Hk=0), SHAPE), (dict(D=48), SHAPE), (dict(D=32), SHAPE),
    (dict(D=544), SHAPE), (dict(q_stride=510), SHAPE), (dict(q_stride=508), SHAPE), (dict(out_stride=500), SHAPE),
    (dict(k_stride=126), SHAPE), (dict(v_stride=124), SHAPE), (dict(T=1 << 22, S=1 << 22), SHAPE), (dict(n_seqs=1 << 22), SHAPE),
    (dict(out=None), NULL), (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(cu=None), NULL),
    (dict(out=at(0) + 4), ALIGN), (dict(q=at(1) + 8), ALIGN), (dict(k=at(2) + 4), ALIGN), (dict(v=at(3) + 2), ALIGN),
    (dict(cu=at(4) + 1), ALIGN), (dict(cuk=at(6) + 2), ALIGN),
    (dict(out=at(1)), ALIAS), (dict(out=at(1) + 599 * 2048), ALIAS), (dict(out=at(2)), ALIAS), (dict(out=at(3)), ALIAS),
    (dict(out=at(4)), ALIAS),
])
def test_prefill_refuses(L, change, want):
    refused(L, want, L.v7g_attention_prefill, *{**PREFILL, **change}.values())


def test_prefill_workspace(L):
    """A call whose tiles leave the chip idle wants scratch: too little, none, misaligned or overlapping is refused."""
    few = {**PREFILL, "T": 3, "S": 5000, "cuk": at(6)}
    need = L.v7g_attention_prefill_workspace(2, 3, 5000, 8, 2, 64)
    assert need > 0
    f = lambda **c: {**few, "ws_bytes": need, **c}.values()  # noqa: E731
    refused(L, SHAPE, L.v7g_attention_prefill, *f(ws_bytes=need - 1))
    refused(L, NULL, L.v7g_attention_prefill, *f(ws=None))
    refused(L, ALIGN, L.v7g_attention_prefill, *f(ws=at(5) + 8))
    for other in ("q", "k", "v", "cu", "out"):
        refused(L, ALIAS, L.v7g_attention_prefill, *f(ws=PREFILL[other]))
    assert L.v7g_attention_prefill_workspace(1, 8192, 8192, 32, 8, 128) == 0  # whole tiles fill the chip
    assert L.v7g_attention_prefill_workspace(1, 8192, 8192, 32, 7, 128) == 0  # no such call


def test_prefill_empty(L):
    L.v7g_clear_last_error()
    none = {k: (None if k in ("out", "q", "k", "v", "cu", "ws") else v) for k, v in PREFILL.items()}
    assert L.v7g_attention_prefill(*{**none, "T": 0, "S": 0}.values()) == 0
    assert L.v7g_attention_prefill(*{**none, "n_seqs": 0}.values()) == 0
    assert L.v7g_get_last_error() == 0


# ------------------------------------------------------------------------------------------------ pages

def pages(**c):
    g = _lib.KvPages()
    d = dict(k=at(10), v=at(11), n_layers=1, n_pages=100, page_size=16, n_kv_heads=2, head_dim=64, layer_stride=0,
             page_stride=2048, token_stride=128)
    d.update(c)
    for k, v in d.items():
        setattr(g, k, v)
    return g


BAD_PAGES = [
    (dict(n_layers=0), SHAPE), (dict(n_layers=20000), SHAPE),
    (dict(n_layers=1 << 14, n_kv_heads=16, token_stride=1024, page_stride=16384, layer_stride=100 * 16384), SHAPE), (dict(n_pages=-1), SHAPE), (dict(page_size=8), SHAPE),
    (dict(page_size=24), SHAPE), (dict(page_size=1 << 17), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(head_dim=-64), SHAPE),
    (dict(token_stride=126), SHAPE), (dict(token_stride=124), SHAPE), (dict(page_stride=2044), SHAPE),
    (dict(page_stride=2046), SHAPE), (dict(n_layers=2, layer_stride=100 * 2048 - 4), SHAPE), (dict(layer_stride=2), SHAPE),
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(k=at(10) + 4), ALIGN), (dict(v=at(11) + 2), ALIGN),
]

TREE = dict(out=at(0), out_stride=512, q=at(1), q_stride=512, pages=None, table=at(2), width=8, lens=at(3), cu=at(4),
            mask=at(5), words=1, n_seqs=3, T=70, Hq=8, scale=0.1, ws=at(6), ws_bytes=64 * MB)


def tree(c, **p):
    g = pages(**p)
    return g, list({**TREE, "pages": ctypes.addressof(g), **c}.values())


@pytest.mark.parametrize("p,want", BAD_PAGES)
def test_every_entry_refuses_bad_pages(L, p, want):
    g, args = tree({}, **p)
    refused(L, want, L.v7g_attention_tree, *args)
    a = ctypes.addressof(g)
    refused(L, want, L.v7g_kv_pack_f16_pages, a, at(0), at(1), 128, at(2), 8, 3, at(3), None, 3)
    refused(L, want, L.v7g_kv_pages_compact, a, at(0), at(2), 8, at(3), at(4), 5, at(5), 3)
    refused(L, want, L.v7g_kv_pages_assign, a, at(0), at(1), at(2), at(3), at(4), at(5), at(6), at(7), None, 3, 8, at(8),
            MB)


@pytest.mark.parametrize("c,want", [
    (dict(pages=None), NULL), (dict(width=-1), SHAPE), (dict(width=1 << 27), SHAPE), (dict(cu=None), SHAPE),
    (dict(words=0), SHAPE), (dict(mask=None), SHAPE), (dict(words=-1), SHAPE), (dict(Hq=7), SHAPE), (dict(T=-1), SHAPE),
    (dict(n_seqs=-1), SHAPE), (dict(q_stride=256), SHAPE), (dict(out_stride=511), SHAPE), (dict(ws_bytes=16), SHAPE),
    (dict(out=None), NULL), (dict(q=None), NULL), (dict(table=None), NULL), (dict(lens=None), NULL), (dict(ws=None), NULL),
    (dict(out=at(0) + 8), ALIGN), (dict(q=at(1) + 4), ALIGN), (dict(table=at(2) + 2), ALIGN), (dict(lens=at(3) + 1), ALIGN),
    (dict(cu=at(4) + 2), ALIGN), (dict(mask=at(5) + 4), ALIGN), (dict(ws=at(6) + 8), ALIGN),
    (dict(out=at(1)), ALIAS), (dict(out=at(10)), ALIAS), (dict(out=at(11)), ALIAS), (dict(out=at(2)), ALIAS),
    (dict(out=at(3)), ALIAS), (dict(out=at(4)), ALIAS), (dict(out=at(5)), ALIAS), (dict(out=at(6)), ALIAS),
    (dict(ws=at(10)), ALIAS),
])
def test_tree_refuses(L, c, want):
    assert L.v7g_attention_tree_workspace(3, 70, 8, 16, 8, 2, 64) == 0
    wide = {"width": 64, **c}
    assert 16 < L.v7g_attention_tree_workspace(3, 70, 64, 16, 8, 2, 64) <= TREE["ws_bytes"]
    g, args = tree(wide)
    refused(L, want, L.v7g_attention_tree, *args)


def test_tree_refuses_head_dims_outside_the_contract(L):
    for D in (32, 80, 544):
        g, args = tree({}, head_dim=D, token_stride=2 * D, page_stride=32 * D)
        refused(L, SHAPE, L.v7g_attention_tree, *args)


def test_tree_empty(L):
    g, args = tree(dict(T=0, n_seqs=0, out=None, q=None, table=None, lens=None, cu=None, mask=None, words=0, ws=None))
    assert L.v7g_attention_tree(*args) == 0


@pytest.mark.parametrize("i,v,want", [
    (0, None, NULL), (1, None, NULL), (2, None, NULL), (4, None, NULL), (7, None, NULL), (3, 126, SHAPE), (3, 124, SHAPE),
    (5, -1, SHAPE), (5, 1 << 27, SHAPE), (6, -1, SHAPE), (9, -1, SHAPE), (9, 4, SHAPE), (1, at(0) + 8, ALIGN),
    (2, at(1) + 4, ALIGN), (4, at(2) + 1, ALIGN), (7, at(3) + 2, ALIGN), (8, at(4) + 2, ALIGN), (1, at(10), ALIAS),
    (2, at(11) + 16, ALIAS), (4, at(10) + 64, ALIAS), (7, at(11) + 4, ALIAS), (8, at(10) + 8, ALIAS),
])
def test_pack_refuses(L, i, v, want):
    g = pages()
    args = [ctypes.addressof(g), at(0), at(1), 128, at(2), 8, 3, at(3), None, 3]
    args[i] = v
    refused(L, want, L.v7g_kv_pack_f16_pages, *args)


def test_pages_of_k_and_v_apart(L):
    """K pages over V pages are refused; interleaved K and V pages and rows are not taken for an overlap."""
    n = 3
    for p, bad in ((dict(v=at(10)), True), (dict(v=at(10) + 99 * 4096), True), (dict(v=at(10) + 4096, page_stride=4096), False),
                   (dict(v=at(10) + 2048, page_stride=4096), True)):
        g = pages(**p)
        # a source over the table's memory is not what is tested: an unaligned one ends accepted layouts first
        args = [ctypes.addressof(g), at(0), at(1), 128, at(2), 8, n, at(3), None, n]
        if bad:
            refused(L, ALIAS, L.v7g_kv_pack_f16_pages, *args)
        else:
            args[1] = at(10)  # this overlap is found, the pages' own is not reported first
            refused(L, ALIAS, L.v7g_kv_pack_f16_pages, *args)


@pytest.mark.parametrize("i,v,want", [
    (0, None, NULL), (1, None, NULL), (2, None, NULL), (4, None, NULL), (5, None, NULL), (7, None, NULL), (3, -1, SHAPE),
    (6, -1, SHAPE), (8, -1, SHAPE), (1, at(0) + 2, ALIGN), (2, at(2) + 1, ALIGN), (4, at(3) + 2, ALIGN),
    (5, at(4) + 2, ALIGN), (7, at(5) + 2, ALIGN), (1, at(2), ALIAS), (1, at(3), ALIAS), (1, at(4), ALIAS),
    (1, at(5), ALIAS), (1, at(10), ALIAS), (4, at(11), ALIAS),
])
def test_compact_refuses(L, i, v, want):
    g = pages()
    args = [ctypes.addressof(g), at(0), at(2), 8, at(3), at(4), 5, at(5), 3]
    args[i] = v
    refused(L, want, L.v7g_kv_pages_compact, *args)


@pytest.mark.parametrize("i,v,want", [
    *[(i, None, NULL) for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 12)], (10, -1, SHAPE), (11, -1, SHAPE), (10, 1 << 30, SHAPE),
    (13, 16, SHAPE), *[(i, at(i - 1) + 2, ALIGN) for i in (1, 2, 3, 4, 5, 6, 7, 8)], (9, at(12) + 2, ALIGN),
    (12, at(8) + 8, ALIGN), (1, at(4), ALIAS), (2, at(5), ALIAS), (3, at(6), ALIAS), (4, at(7), ALIAS), (1, at(1), ALIAS),
    (12, at(0), ALIAS), (12, at(4), ALIAS), (9, at(2), ALIAS), (1, at(10), ALIAS), (5, at(11), ALIAS),
])
def test_assign_refuses(L, i, v, want):
    g = pages()
    args = [ctypes.addressof(g), *(at(j) for j in range(8)), None, 3, 8, at(8), MB]
    assert L.v7g_kv_pages_assign_workspace(3, 100) <= MB
    args[i] = v
    refused(L, want, L.v7g_kv_pages_assign, *args)


# ------------------------------------------------------------------------------------------------ token scores

LOGPROBS = dict(lp=at(0), ent=at(1), tl=at(2), ti=at(3), x=at(4), stride=5000, ids=at(5), T=3, V=5000, K=4, ws=at(6),
                ws_bytes=MB)


@pytest.mark.parametrize("c,want", [
    (dict(T=-1), SHAPE), (dict(T=1 << 24), SHAPE), (dict(V=0), SHAPE), (dict(V=(1 << 30) + 1), SHAPE), (dict(K=-1), SHAPE), (dict(K=65), SHAPE),
    (dict(V=3), SHAPE), (dict(stride=4999), SHAPE), (dict(ws_bytes=8), SHAPE), (dict(lp=None), NULL), (dict(ent=None), NULL),
    (dict(tl=None), NULL), (dict(ti=None), NULL), (dict(x=None), NULL), (dict(ids=None), NULL), (dict(ws=None), NULL),
    (dict(lp=at(0) + 2), ALIGN), (dict(ent=at(1) + 1), ALIGN), (dict(tl=at(2) + 2), ALIGN), (dict(ti=at(3) + 2), ALIGN),
    (dict(x=at(4) + 2), ALIGN), (dict(ids=at(5) + 2), ALIGN), (dict(ws=at(6) + 8), ALIGN), (dict(lp=at(4)), ALIAS),
    (dict(ent=at(0)), ALIAS), (dict(tl=at(5)), ALIAS), (dict(ti=at(4) + 400), ALIAS), (dict(ws=at(4)), ALIAS),
])
def test_logprobs_refuses(L, c, want):
    assert 8 < L.v7g_token_logprobs_workspace(3, 5000, 4) <= MB
    refused(L, want, L.v7g_token_logprobs, *{**LOGPROBS, **c}.values())


def test_logprobs_empty(L):
    assert L.v7g_token_logprobs(None, None, None, None, None, 0, None, 0, 100, 4, None, 0) == 0
