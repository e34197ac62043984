"""The decoding-loop operators' checks of their arguments, and the rotation frequencies, without a GPU:
every refusal comes before any device call."""
import ctypes as C
import math

import numpy as np
import pytest

from mosship import lib

P = 0x1000  # a 16-byte aligned address that no refused call may touch


def _cache(**kw):
    f = dict(k=P, v=P, k_scale=None, v_scale=None, kv_dtype=lib.F16, kv_heads=4, head_dim=64, page_size=64, n_pages=8,
             page_table=P, table_stride=4, streams=2)
    f.update(kw)
    return lib.KVCacheStruct(**f)


def _rope(**kw):
    f = dict(freqs=P, rot_dim=64, halves=0, mscale=1.0)
    f.update(kw)
    return lib.RopeStruct(**f)


def _refused(rc, word):
    assert rc == lib.EINVAL
    assert word in lib.load().moss_hip_last_error().decode(), lib.load().moss_hip_last_error()


BAD_CACHES = [
    (dict(kv_dtype=4), "kv_dtype"), (dict(kv_dtype=-1), "kv_dtype"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1025), "kv_heads"), (dict(page_size=0), "page_size"), (dict(page_size=40), "page_size"),
    (dict(page_size=65536), "page_size"), (dict(streams=-1), "streams"), (dict(k=None), "null"), (dict(page_table=None), "null"),
    (dict(n_pages=0), "n_pages"), (dict(table_stride=0), "table_stride"), (dict(kv_dtype=lib.I8), "scales"),
    (dict(k_scale=P, v_scale=P), "scales"), (dict(kv_dtype=lib.E4M3, k_scale=P), "scales"), (dict(v=P + 8), "aligned"),
    (dict(kv_dtype=lib.I8, k_scale=P + 4, v_scale=P), "aligned"),
]


@pytest.mark.parametrize("kw,word", BAD_CACHES)
def test_bad_caches(kw, word):
    L, c = lib.load(), _cache(**kw)
    r = C.addressof(c)
    _refused(L.moss_hip_kv_write(r, P, 256, P, 256, lib.F32, 1, P, P, None, None, None), word)
    _refused(L.moss_hip_kv_read(r, P, P, 1, P, 256, P, 256, lib.F32, None), word)
    _refused(L.moss_hip_attn_tree(P, 256, lib.F32, 4, r, P, P, None, 1, 1, 64, 0.125, P, 256, lib.F32, None, P, 1 << 30, None), word)


def test_null_structs():
    L, c = lib.load(), _cache()
    r = C.addressof(c)
    _refused(L.moss_hip_kv_write(None, P, 256, P, 256, lib.F32, 1, P, P, None, None, None), "null")
    _refused(L.moss_hip_kv_read(None, P, P, 1, P, 256, P, 256, lib.F32, None), "null")
    _refused(L.moss_hip_attn_tree_workspace(None, 4, 1, 1, 64, C.byref(C.c_size_t())), "null")
    _refused(L.moss_hip_attn_tree_workspace(r, 4, 1, 1, 64, None), "null")
    _refused(L.moss_hip_rope_rows(P, 64, 64, P, 64, 64, lib.F32, 1, 1, 64, P, None, None), "null")
    _refused(L.moss_hip_rope_freqs(None, None, None), "null")


@pytest.mark.parametrize("i,value,word", [
    (0, None, "null"), (3, None, "null"), (10, None, "null"), (6, lib.I8, "dtype"), (7, -1, "rows"), (7, (1 << 22) + 1, "rows"),
    (8, 0, "heads"), (9, 0, "head_dim"), (9, 65, "even"), (1, -1, "negative"), (4, 768, "same strides"), (5, 32, "overlap"), (4, 700, "overlap"),
    (4, 0, "overlap"), (4, 32, "overlap")])
def test_rope_rows_refusals(i, value, word):
    a = [P, 1024, 64, P, 1024, 64, lib.F32, 4, 12, 64, P]
    a[i] = value
    if word == "overlap":
        a[3] = P + 0x10000
    _refused(lib.load().moss_hip_rope_rows(*a, C.addressof(_rope()), None), word)


@pytest.mark.parametrize("kw,word", [(dict(freqs=None), "freqs"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=63), "rot_dim"),
                                     (dict(rot_dim=66), "rot_dim"), (dict(halves=2), "halves")])
def test_rope_struct_refusals(kw, word):
    L, rope, c = lib.load(), _rope(**kw), _cache()
    _refused(L.moss_hip_rope_rows(P, 64, 64, P, 64, 64, lib.F32, 1, 1, 64, P, C.addressof(rope), None), word)
    _refused(L.moss_hip_kv_write(C.addressof(c), P, 256, P, 256, lib.F32, 1, P, P, C.addressof(rope), None, None), word)


def test_kv_refusals():
    L, c = lib.load(), _cache()
    r = C.addressof(c)
    ok = [r, P, 256, P, 256, lib.F32, 4, P, P, None, None, None]
    for i, value, word in [(1, None, "null"), (3, None, "null"), (7, None, "null"), (8, None, "null"), (5, lib.I8, "dtype"), (6, -1, "rows"),
                           (2, -1, "negative"), (10, P, "rope_pos without rope")]:
        a = list(ok)
        a[i] = value
        _refused(L.moss_hip_kv_write(*a), word)
    ok = [r, P, P, 4, P, 256, P, 256, lib.F32, None]
    for i, value, word in [(1, None, "null"), (2, None, "null"), (4, None, "null"), (6, None, "null"), (3, -1, "rows"), (5, 255, "overlap"),
                           (8, lib.E4M3, "dtype")]:
        a = list(ok)
        a[i] = value
        _refused(L.moss_hip_kv_read(*a), word)


def test_attn_tree_refusals():
    L, c = lib.load(), _cache(streams=1)
    ok = [P, 1024, lib.F32, 16, C.addressof(c), P, P, None, 4, 4, 256, 0.125, P, 1024, lib.F32, None, P, 1 << 30, None]
    for i, value, word in [(0, None, "null"), (5, None, "null"), (6, None, "null"), (12, None, "null"), (2, lib.I8, "dtype"), (14, 7, "dtype"),
                           (3, 0, "heads"), (3, 6, "heads"), (3, 2048, "heads"), (8, -1, "rows"), (9, 0, "max_rows"), (9, 65, "max_rows"),
                           (10, 0, "max_keys"), (10, (1 << 28) + 1, "max_keys"), (11, math.nan, "scale"), (11, math.inf, "scale"),
                           (1, -1, "negative"), (13, 1023, "overlap")]:
        a = list(ok)
        a[i] = value
        _refused(L.moss_hip_attn_tree(*a), word)
    n = C.c_size_t()
    assert L.moss_hip_attn_tree_workspace(C.addressof(c), 16, 4, 4, 8192, C.byref(n)) == lib.OK and n.value > 0
    a = list(ok)
    a[10] = 8192
    for i, value, word in [(16, None, "workspace needs"), (17, n.value - 1, "workspace needs"), (16, P + 4, "aligned")]:
        b = list(a)
        b[i] = value
        _refused(L.moss_hip_attn_tree(*b), word)
    assert L.moss_hip_attn_tree_workspace(C.addressof(c), 16, 0, 4, 8192, C.byref(n)) == lib.OK and n.value == 0


def test_token_logprobs_refusals():
    L = lib.load()
    ok = [P, 1024, lib.F32, 4, 1024, P, 1.0, P, P, 5, P, P, P, 1 << 30, None]
    for i, value, word in [(0, None, "null"), (5, None, "null"), (7, None, "null"), (10, None, "null"), (11, None, "null"), (2, lib.I8, "dtype"),
                           (3, -1, "rows"), (4, 0, "vocab"), (4, (1 << 20) + 1, "vocab"), (9, -1, "top_k"), (9, 33, "top_k"), (6, 0.0, "inv_temperature"),
                           (6, -1.0, "inv_temperature"), (6, math.nan, "inv_temperature"), (6, math.inf, "inv_temperature"), (1, -1, "negative")]:
        a = list(ok)
        a[i] = value
        _refused(L.moss_hip_token_logprobs(*a), word)
    n = C.c_size_t()
    assert L.moss_hip_token_logprobs_workspace(4, 100000, 5, C.byref(n)) == lib.OK and n.value > 0
    a = list(ok)
    a[4], a[13] = 100000, n.value - 1
    _refused(L.moss_hip_token_logprobs(*a), "workspace needs")
    _refused(L.moss_hip_token_logprobs_workspace(4, 100000, 40, C.byref(n)), "top_k")
    assert L.moss_hip_token_logprobs_workspace(4, 1024, 5, C.byref(n)) == lib.OK and n.value == 0


def test_strides_whose_multiples_leave_64_bits():
    """11 head strides of 2^62 are negative in 64 bits, which once passed for rows that lie apart."""
    L, c = lib.load(), _cache(streams=1)
    far, r = 1 << 62, C.addressof(c)
    for i in (1, 2, 4, 5):
        a = [P, 1024, 64, P + 0x10000, 1024, 64, lib.F32, 4, 12, 64, P]
        a[i] = far
        _refused(L.moss_hip_rope_rows(*a, C.addressof(_rope()), None), "2^40")
    for k, v in ((far, 256), (256, far)):
        _refused(L.moss_hip_kv_write(r, P, k, P, v, lib.F32, 4, P, P, None, None, None), "2^40")
        _refused(L.moss_hip_kv_read(r, P, P, 4, P, k, P, v, lib.F32, None), "2^40")
    for q, o in ((far, 1024), (1024, far)):
        _refused(L.moss_hip_attn_tree(P, q, lib.F32, 16, r, P, P, None, 4, 4, 256, 0.125, P, o, lib.F32, None, P, 1 << 30, None), "2^40")
    _refused(L.moss_hip_token_logprobs(P, far, lib.F32, 4, 1024, P, 1.0, P, P, 5, P, P, P, 1 << 30, None), "2^40")


def test_nothing_to_do_is_ok():
    """No rows, no streams: OK before any device call."""
    L, c = lib.load(), _cache(streams=0)
    r, rope = C.addressof(c), _rope()
    assert L.moss_hip_rope_rows(P, 64, 64, P, 64, 64, lib.F32, 0, 1, 64, P, C.addressof(rope), None) == lib.OK
    assert L.moss_hip_kv_write(r, P, 256, P, 256, lib.F32, 3, P, P, None, None, None) == lib.OK
    assert L.moss_hip_kv_read(r, P, P, 0, P, 256, P, 256, lib.F32, None) == lib.OK
    assert L.moss_hip_attn_tree(P, 256, lib.F32, 4, r, P, P, None, 2, 1, 64, 0.125, P, 256, lib.F32, None, None, 0, None) == lib.OK
    assert L.moss_hip_token_logprobs(P, 1024, lib.F32, 0, 1024, P, 1.0, P, None, 0, None, None, None, 0, None) == lib.OK


def test_rope_freqs():
    """Against the formulas in numpy; the library's pow and numpy's may differ by a few units of 2^-53 in each."""
    i = np.arange(32)
    w = 10000.0 ** (-2.0 * i / 64)
    tol = 16 * 2.0 ** -53
    for kw, want, m in [(dict(), w, 1.0), (dict(scaling="linear", factor=8.0), w / 8, 1.0),
                        (dict(scaling="ntk", factor=4.0), (10000.0 * 4.0 ** (64 / 62)) ** (-2.0 * i / 64), 1.0),
                        (dict(base=500000.0), 500000.0 ** (-2.0 * i / 64), 1.0)]:
        f, got = lib.rope_freqs(64, **kw)
        assert got == m
        np.testing.assert_allclose(f, want, rtol=tol, atol=0)
    f, got = lib.rope_freqs(64, scaling="yarn", factor=16.0, orig_ctx=4096)
    g = np.clip((4096 * w / (2 * np.pi) - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, g * w + (1 - g) * w / 16, rtol=64 * 2.0 ** -53, atol=0)
    assert f[0] == w[0] and abs(f[-1] / (w[-1] / 16) - 1) < tol  # fast pairs keep their frequency, slow ones are stretched
    assert abs(got - (0.1 * math.log(16.0) + 1.0)) <= 2.0 ** -24 * 2
    assert lib.rope_freqs(2)[0][0] == 1.0


@pytest.mark.parametrize("args,kw,word", [
    ((0,), {}, "rot_dim"), ((63,), {}, "rot_dim"), ((514,), {}, "rot_dim"), ((64,), dict(base=1.0), "base"), ((64,), dict(base=math.nan), "base"),
    ((64,), dict(scaling="linear", factor=0.5), "factor"), ((2,), dict(scaling="ntk", factor=2.0), "rot_dim >= 4"),
    ((64,), dict(scaling="yarn", factor=2.0), "orig_ctx"), ((64,), dict(scaling="yarn", factor=2.0, orig_ctx=64, beta_fast=1.0, beta_slow=2.0), "beta")])
def test_rope_freqs_refusals(args, kw, word):
    with pytest.raises(lib.MossHipError) as e:
        lib.rope_freqs(*args, **kw)
    assert e.value.code == lib.EINVAL and word in str(e.value)


def test_binding_refuses_cpu_tensors():
    import torch
    rope = lib.Rope(64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        lib.rope_rows(torch.zeros(1, 1, 64), torch.zeros(1, dtype=torch.int32), rope)
    pool = torch.zeros(4, 2, 16, 64)
    with pytest.raises(ValueError, match="k_scale"):
        lib.KVCache(pool.to(torch.int8), pool.to(torch.int8), torch.zeros(1, 4, dtype=torch.int32), pool, pool)
    with pytest.raises(ValueError, match="pools"):
        lib.KVCache(pool.to(torch.bfloat16), pool.to(torch.bfloat16), torch.zeros(1, 4, dtype=torch.int32))
    cache = lib.KVCache(pool, pool, torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        lib.kv_write(cache, pool, pool, None, None)
