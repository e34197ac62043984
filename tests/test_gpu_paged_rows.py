"""Rotary rows and cache rows at the sizes where the launches change (GPU): several units a thread, several rows a
workgroup with a remainder, rows of more units than a wave takes at once.  Against the same 64-bit forms as the small ones."""
import numpy as np
import pytest

from mosship import lib
from test_gpu_paged_ops import TOP, U16, U32, _make_cache, _rope_tol, _rot, _stored, _types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,heads,dim,rot,halves,dtype", [
    (1025, 16, 128, 128, False, "f32"), (4099, 8, 64, 64, False, "f16"), (4099, 8, 64, 64, True, "f32"), (1031, 40, 128, 96, True, "f16"),
    (16391, 1, 64, 32, True, "f32"), (16400, 2, 64, 48, False, "f16"), (2051, 6, 50, 22, True, "f16"), (1027, 12, 70, 34, False, "f32")])
@pytest.mark.parametrize("pad,first", [(0, 0), (3, 1)])
def test_rope_many_rows(torch_gpu, rows, heads, dim, rot, halves, dtype, pad, first):
    """More than 1024 workgroups: four units of a thread in flight, the last rows fewer than a workgroup takes; whole and at
    odd addresses; into another tensor and in place."""
    torch = torch_gpu
    print(f"rope many {rows}x{heads}x{dim} rot {rot} halves {halves} {dtype} pad {pad}", flush=True)
    rng = np.random.default_rng(rows + rot)
    width = heads * dim + pad
    flat = torch.full((first + rows * width,), 7.0, dtype=_types(torch)[dtype], device="cuda")
    x = flat.as_strided((rows, heads, dim), (width, dim, 1), first)
    x.copy_(torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)))
    before = flat.clone()
    pos = rng.integers(0, 1 << 17, rows).astype(np.int32)
    rope = lib.Rope(rot, halves=halves, scaling="yarn", factor=4.0, orig_ctx=4096)
    f, m = lib.rope_freqs(rot, scaling="yarn", factor=4.0, orig_ctx=4096)
    p = torch.from_numpy(pos).cuda()
    apart = torch.full((rows, heads, dim), float("nan"), dtype=flat.dtype, device="cuda")
    lib.rope_rows(x, p, rope, apart)
    assert torch.equal(flat, before)
    got = apart.double().cpu().numpy()
    want, mag = _rot(x.double().cpu().numpy(), pos, f, halves, m)
    tol = _rope_tol(mag, f, pos) + (np.abs(want) * U16 + 2.0 ** -25 if dtype == "f16" else 0)
    tol[..., rot:] = 0
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)
    lib.rope_rows(x, p, rope)
    assert torch.equal(x, apart)
    x.copy_(before.as_strided((rows, heads, dim), (width, dim, 1), first))
    assert torch.equal(flat, before)  # nothing beside the rows was written


@pytest.mark.parametrize("cache,dtype", [("f32", "f32"), ("f16", "f32"), ("i8", "f16"), ("e4m3", "f16"), ("i8", "f32"), ("e4m3", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rows,heads,dim,rot,halves", [
    (2049, 2, 64, 64, False), (2050, 3, 64, 64, True), (2051, 2, 128, 50, True),  # the three orders of angles
    (2051, 9, 128, 128, True), (70, 9, 128, 96, False), (70, 16, 128, 50, True), (2049, 17, 64, 48, False), (33, 33, 64, 64, True)])
def test_kv_many_rows(torch_gpu, cache, dtype, rows, heads, dim, rot, halves):
    """Workgroups of four rows with a remainder, and rows of more than 1024 elements, whose units a wave takes in turns;
    padded rows and rows without a place among them."""
    torch = torch_gpu
    print(f"kv many {cache} {dtype} {rows}x{heads}x{dim} rot {rot} halves {halves}", flush=True)
    rng = np.random.default_rng(rows + heads)
    streams, ctx = 3, (rows + 2) // 3 + 5
    c = _make_cache(torch, cache, streams, ctx, heads, 48, dim)
    slot = rng.permutation(streams * ctx)[:rows]
    stream, pos = (slot // ctx).astype(np.int32), (slot % ctx).astype(np.int32)
    pos[rows - 1], pos[rows // 2], stream[5] = -1, 10 ** 6, streams
    ok = np.ones(rows, bool)
    ok[[rows - 1, rows // 2, 5]] = False
    depth = rng.integers(0, 100000, rows).astype(np.int32)
    k, v = (torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).to(_types(torch)[dtype]).cuda() for _ in range(2))
    dev = [torch.from_numpy(a).cuda() for a in (stream, pos, depth)]
    lib.kv_write(c, k, v, dev[0], dev[1], rope=lib.Rope(rot, halves=halves), rope_pos=dev[2])
    ko, vo = (torch.full((rows, heads, dim), 5.0, device="cuda") for _ in range(2))
    lib.kv_read(c, dev[0], dev[1], ko, vo)
    ko, vo = ko.double().cpu().numpy(), vo.double().cpu().numpy()
    assert (ko[rows - 1] == 5).all() and (vo[rows - 1] == 5).all()
    assert np.isnan(ko[[5, rows // 2]]).all() and np.isnan(vo[[5, rows // 2]]).all()
    assert np.array_equal(vo[ok], _stored(torch, v.float().cpu().numpy(), cache)[ok])
    f, _ = lib.rope_freqs(rot)
    want, mag = _rot(k.double().cpu().numpy(), depth, f, halves)
    tol = _rope_tol(mag, f, depth)
    if cache == "f16":
        tol = tol + np.abs(want) * U16 + 2.0 ** -25
    elif cache in TOP:
        # half a step of the stored element (with the rotation's error on the element and on the scale), and the roundings of x / d
        top = np.abs(want).max(-1, keepdims=True)
        step = top / 127 if cache == "i8" else np.maximum(np.abs(want) * 2.0 ** -3, top / 448 * 2.0 ** -9)
        tol = 2 * tol + step / 2 * (1 + 2.0 ** -10) + 4 * U32 * np.abs(want)
    assert (np.abs(ko - want) <= tol)[ok].all(), np.max((np.abs(ko - want) - tol)[ok])
