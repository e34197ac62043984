"""More of the decoding-loop operators' checks of their arguments, without a GPU."""
import ctypes as C
import math

import pytest

from mosship import lib
from test_paged_ops_args import P, _cache, _refused


def test_rope_takes_mscale_as_given():
    """With frequencies of the library's own it is used too, and what frequencies given already say is refused besides them."""
    import torch
    assert lib.Rope(64, device="cpu").struct.mscale == 1.0
    assert lib.Rope(64, mscale=0.5, device="cpu").struct.mscale == 0.5
    yarn = dict(scaling="yarn", factor=16.0, orig_ctx=4096, device="cpu")
    assert abs(lib.Rope(64, **yarn).struct.mscale - (0.1 * math.log(16.0) + 1.0)) < 2.0 ** -22
    assert lib.Rope(64, mscale=2.0, **yarn).struct.mscale == 2.0
    f = torch.ones(24, dtype=torch.float64)
    own = lib.Rope(freqs=f, halves=True)
    assert (own.struct.rot_dim, own.struct.mscale, own.struct.halves) == (48, 1.0, 1)
    assert lib.Rope(48, freqs=f, mscale=0.5).struct.mscale == 0.5
    assert lib.Rope(freqs=f, device="cpu").device == -1
    for kw in (dict(rot_dim=64), dict(scaling="linear", factor=2.0), dict(device="meta")):
        with pytest.raises(ValueError, match="freqs"):
            lib.Rope(freqs=f, **kw)


def test_attention_in_place_of_another_layout_is_refused():
    """Over the query itself, with rows that would lie elsewhere than the query's: one row's output in another's query."""
    L, c = lib.load(), _cache(streams=1)
    for q_stride, qdt, o_stride, odt in ((1024, lib.F32, 2048, lib.F32), (1024, lib.F32, 1024, lib.F16), (1024, lib.F16, 1024, lib.F32)):
        _refused(L.moss_hip_attn_tree(P, q_stride, qdt, 16, C.addressof(c), P, P, None, 4, 4, 256, 0.125, P, o_stride, odt, None, P,
                                      1 << 30, None), "same type and stride")


def test_a_cache_without_streams_has_no_table():
    """An empty tensor's address is NULL: writing and attending are nothing to do, whatever the rows."""
    import torch
    pool = torch.zeros(4, 2, 16, 64)
    c = lib.KVCache(pool, pool, torch.zeros(0, 4, dtype=torch.int32))
    assert c.struct.page_table is None and c.streams == 0
    L = lib.load()
    assert L.moss_hip_kv_write(c.ref, P, 128, P, 128, lib.F32, 3, P, P, None, None, None) == lib.OK
    assert L.moss_hip_kv_read(c.ref, P, P, 0, P, 128, P, 128, lib.F32, None) == lib.OK
    assert L.moss_hip_attn_tree(P, 256, lib.F32, 4, c.ref, P, P, None, 2, 1, 64, 0.125, P, 256, lib.F32, None, None, 0, None) == lib.OK
    assert lib.attn_tree_workspace(c, 4, 2, 1, 64) == 0
    bad = _cache(page_table=None, streams=1)
    _refused(L.moss_hip_kv_write(C.addressof(bad), P, 256, P, 256, lib.F32, 3, P, P, None, None, None), "null")


@pytest.mark.parametrize("streams,heads,kvh,rows", [(65536, 64, 64, 1), (1024, 64, 8, 64), (4096, 16, 16, 64), (64, 32, 8, 64), (97, 8, 8, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_workspaces_of_far_bounds_stay_small(streams, heads, kvh, rows, dim):
    """However many rows and far the bound: partial results of 2^20 rows at most, but for a batch so small that its keys are
    cut to fill the chip (64 pieces of each stream)."""
    c = _cache(kv_dtype=lib.I8, k_scale=P, v_scale=P, kv_heads=kvh, head_dim=dim, streams=streams)
    n = C.c_size_t()
    for keys in (1000, 16384, 65537, 131072, 1 << 20, 1 << 28):
        assert lib.load().moss_hip_attn_tree_workspace(C.addressof(c), heads, streams * rows, rows, keys, C.byref(n)) == lib.OK
        assert n.value <= (1 << 20) * (2 + dim) * 4 + 16 * streams + 8, (keys, n.value)
