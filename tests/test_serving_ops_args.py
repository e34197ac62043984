"""The serving-loop operators' checks of their arguments, without a GPU: every refusal comes before any device call."""
import ctypes as C
import math

import pytest

from mosship import lib

P = 0x1000  # a 16-byte aligned address that no refused call may touch


def _cache(**kw):
    f = dict(k=P, v=P, k_scale=None, v_scale=None, kv_dtype=lib.F16, kv_heads=4, head_dim=64, page_size=64, n_pages=8,
             page_table=P, table_stride=4, streams=2)
    f.update(kw)
    return lib.KVCacheStruct(**f)


def _pages(**kw):
    f = dict(page_table=P, table_stride=4, streams=2, refs=P, n_pages=8, page_size=64)
    f.update(kw)
    return lib.KVPagesStruct(**f)


def _adapters(**kw):
    f = dict(a=P, b=P, scale=None, n_adapters=2, max_rank=16, cols=64, out=32)
    f.update(kw)
    return lib.AdaptersStruct(**f)


def _refused(rc, word):
    assert rc == lib.EINVAL
    assert word in lib.load().moss_hip_last_error().decode(), lib.load().moss_hip_last_error()


def _each(fn, ok, bad):
    for i, value, word in bad:
        a = list(ok)
        a[i] = value
        _refused(fn(*a), word)


def test_verify_refusals():
    L = lib.load()
    #     0  1    2        3     4  5  6    7  8  9     10 11 12 13   14   15 16 17 18 19 20       21
    ok = [P, 99999, lib.F32, None, 0, 8, 99999, P, P, None, 2, 4, P, 1.0, 1.0, 0, P, P, P, P, 1 << 20, None]
    _each(L.moss_hip_verify_tokens, ok, [
        (0, None, "null"), (7, None, "null"), (8, None, "null"), (16, None, "null"), (17, None, "null"), (18, None, "null"),
        (12, None, "uniforms"), (2, lib.I8, "dtype"), (1, -1, "negative"), (4, -1, "negative"), (1, (1 << 40) + 1, "2^40"), (5, -1, "rows"),
        (6, 0, "vocab"), (6, (1 << 20) + 1, "vocab"), (10, -1, "streams"), (10, 65537, "streams"), (11, 0, "max_rows"), (11, 65, "max_rows"),
        (13, 0.0, "temperatures"), (13, math.nan, "temperatures"), (14, math.inf, "temperatures"), (14, -1.0, "temperatures"),
        (15, 2, "greedy"), (15, 1, "greedy takes no"), (19, None, "workspace needs"), (20, 100, "workspace needs"), (19, P + 8, "aligned")])
    both = list(ok)
    both[3] = both[9] = P
    _refused(L.moss_hip_verify_tokens(*both), "chains")
    n = C.c_size_t()
    for a, word in [((-1, 1, 1, 0), "streams"), ((1, 0, 1, 0), "max_rows"), ((1, 1, 0, 0), "vocab"), ((65536, 64, 1 << 20, 0), "2^34")]:
        _refused(L.moss_hip_verify_tokens_workspace(*a, C.byref(n)), word)
    _refused(L.moss_hip_verify_tokens_workspace(1, 1, 1, 0, None), "null")
    assert L.moss_hip_verify_tokens_workspace(0, 1, 1, 0, C.byref(n)) == lib.OK and n.value == 0
    sizes = []
    for draft in (0, 1):
        assert L.moss_hip_verify_tokens_workspace(3, 5, 130001, draft, C.byref(n)) == lib.OK
        sizes.append(n.value)
    assert 0 < sizes[0] < sizes[1]
    assert L.moss_hip_verify_tokens_workspace(3, 5, 1024, 1, C.byref(n)) == lib.OK and n.value == 0  # (one launch holds all of it)
    nothing = list(ok)  # no streams: nothing to do
    nothing[10], nothing[19] = 0, None
    assert L.moss_hip_verify_tokens(*nothing) == lib.OK


BAD_PAGES = [(dict(streams=-1), "streams"), (dict(streams=65537), "streams"), (dict(table_stride=0), "table_stride"),
             (dict(streams=65536, table_stride=2048), "2^26"), (dict(page_size=0), "page_size"), (dict(page_size=40), "page_size"),
             (dict(page_size=65536), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_pages=(1 << 30) + 1), "n_pages")]


@pytest.mark.parametrize("kw,word", BAD_PAGES + [(dict(page_table=None), "null"), (dict(refs=None), "null")])
def test_bad_pages(kw, word):
    L, p, c, n = lib.load(), _pages(**kw), _cache(), C.c_size_t()
    r, l = C.addressof(p), C.addressof(c)
    _refused(L.moss_hip_kv_fork(r, P, P, P, 1 << 30, None), word)
    _refused(L.moss_hip_kv_reserve(r, l, 1, P, P, 4, P, P, 1 << 30, None), word)
    if word != "null":
        _refused(L.moss_hip_kv_fork_workspace(r, C.byref(n)), word)
        _refused(L.moss_hip_kv_reserve_workspace(r, 4, C.byref(n)), word)


def test_page_call_refusals():
    L, p, c, n = lib.load(), _pages(), _cache(), C.c_size_t()
    r, l = C.addressof(p), C.addressof(c)
    _each(L.moss_hip_kv_fork, [r, P, P, None, 0, None], [(0, None, "null"), (1, None, "null")])
    ok = [r, l, 1, P, P, 4, P, P, 1 << 20, None]
    _each(L.moss_hip_kv_reserve, ok, [
        (0, None, "null"), (1, None, "null"), (2, 0, "n_layers"), (2, 65, "n_layers"), (3, None, "null"), (4, None, "null"), (6, None, "null"),
        (5, 0, "max_rows"), (5, 257, "max_rows"), (7, None, "workspace needs"), (8, 8, "workspace needs"), (7, P + 4, "aligned")])
    for kw in (dict(page_table=P + 64), dict(table_stride=5), dict(streams=3), dict(n_pages=9), dict(page_size=32)):
        a = list(ok)
        other = _cache(**kw)
        a[1] = C.addressof(other)
        _refused(L.moss_hip_kv_reserve(*a), "those of the pages")
    for out in (L.moss_hip_kv_fork_workspace(r, None), L.moss_hip_kv_reserve_workspace(r, 4, None)):
        _refused(out, "null")
    _refused(L.moss_hip_kv_reserve_workspace(r, 0, C.byref(n)), "max_rows")
    # small tables are forked without a workspace, large ones with one
    assert L.moss_hip_kv_fork_workspace(r, C.byref(n)) == lib.OK and n.value == 0
    big = _pages(streams=1024, table_stride=64)
    assert L.moss_hip_kv_fork_workspace(C.addressof(big), C.byref(n)) == lib.OK and n.value == 4 * 65536
    _refused(L.moss_hip_kv_fork(C.addressof(big), P, P, None, 0, None), "workspace needs")
    none = _pages(streams=0, page_table=None)
    assert L.moss_hip_kv_fork(C.addressof(none), P, P, None, 0, None) == lib.OK


def test_layers_of_one_shape():
    L = lib.load()
    ok = [P, P, P, 4, 4, None]
    base = [None, 1, *ok]
    _refused(L.moss_hip_kv_compact(*base), "null")
    for kw in (dict(kv_dtype=lib.F32), dict(kv_heads=2), dict(head_dim=128), dict(page_size=32), dict(n_pages=9), dict(page_table=P + 64),
               dict(table_stride=5), dict(streams=3)):
        two = (lib.KVCacheStruct * 2)(_cache(), _cache(**kw))
        _refused(L.moss_hip_kv_compact(C.addressof(two), 2, *ok), "one shape")
    two = (lib.KVCacheStruct * 2)(_cache(), _cache(v=P + 8))
    _refused(L.moss_hip_kv_compact(C.addressof(two), 2, *ok), "aligned")
    c = _cache()
    _each(L.moss_hip_kv_compact, [C.addressof(c), 1, *ok], [
        (1, 0, "n_layers"), (1, 65, "n_layers"), (2, None, "null"), (3, None, "null"), (4, None, "null"), (5, -1, "rows"), (6, 0, "max_rows"),
        (6, 65, "max_rows")])
    assert L.moss_hip_kv_compact(C.addressof(c), 1, P, P, None, 0, 4, None) == lib.OK


@pytest.mark.parametrize("kw,word", [
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(a=P + 8), "aligned"), (dict(b=P + 2), "aligned"), (dict(n_adapters=0), "n_adapters"),
    (dict(n_adapters=(1 << 20) + 1), "n_adapters"), (dict(max_rank=0), "max_rank"), (dict(max_rank=24), "max_rank"), (dict(max_rank=144), "max_rank"),
    (dict(cols=0), "cols"), (dict(cols=48), "cols"), (dict(cols=65568), "cols"), (dict(out=0), "out"), (dict(out=24), "out"), (dict(out=65552), "out")])
def test_bad_adapters(kw, word):
    L, a = lib.load(), _adapters(**kw)
    _refused(L.moss_hip_adapter_rows(P, 64, lib.F32, C.addressof(a), P, 1, P, 32, P, 32, lib.F32, None), word)
    _refused(L.moss_hip_adapter_pack(C.addressof(a), 0, 1, P, P, None, None), word)
    n = C.c_size_t()
    if word not in ("null", "aligned"):
        _refused(L.moss_hip_adapter_sizes(C.addressof(a), C.byref(n), C.byref(n)), word)


def test_adapter_pack_refusals():
    L, a = lib.load(), _adapters()
    _each(L.moss_hip_adapter_pack, [C.addressof(a), 0, 2, P, P, None, None], [
        (0, None, "null"), (1, -1, "first"), (1, 1, "first"), (1, 1 << 31 - 1, "first"), (2, -1, "count"), (2, 3, "count"), (3, None, "null"),
        (4, None, "null"), (3, P + 8, "aligned"), (4, P + 2, "aligned")])
    assert L.moss_hip_adapter_pack(C.addressof(a), 2, 0, P, P, None, None) == lib.OK
    x, y = C.c_size_t(), C.c_size_t()
    for kw, sizes in ((dict(), (2 * 16 * 64 * 2, 2 * 64 * 16 * 2)), (dict(max_rank=48, out=80), (2 * 64 * 64 * 2, 2 * 128 * 64 * 2))):
        b = _adapters(**kw)
        assert L.moss_hip_adapter_sizes(C.addressof(b), C.byref(x), C.byref(y)) == lib.OK and (x.value, y.value) == sizes
    _refused(L.moss_hip_adapter_sizes(C.addressof(a), None, C.byref(y)), "null")


def test_adapter_rows_refusals():
    L, a = lib.load(), _adapters()
    Q = P + (1 << 20)
    ok = [P, 64, lib.F32, C.addressof(a), P, 4, Q, 32, Q, 32, lib.F32, None]
    _each(L.moss_hip_adapter_rows, ok, [
        (0, None, "null"), (3, None, "null"), (4, None, "null"), (6, None, "null"), (8, None, "null"), (2, lib.I8, "dtype"), (10, lib.E4M3, "dtype"),
        (5, -1, "rows"), (1, -1, "negative"), (7, -1, "negative"), (9, 31, "overlap"), (7, 64, "same stride"), (8, P, "must not be x")])
    none = list(ok)
    none[5] = 0
    assert L.moss_hip_adapter_rows(*none) == lib.OK
