"""The operators of a caller's own decoding loop against plain 64-bit forms (GPU): rotary positions, the
paged cache in fp32 / fp16 / int8 / e4m3, attention of drafted rows over it, token log probabilities, and
a run of all of them together.

Tolerances come from the arithmetic: a rounding to fp32 is 2^-24 of a value, to fp16 2^-11, to e4m3 2^-4."""
import math

import numpy as np
import pytest

from mosship import lib

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -11
TOP = {"i8": 127.0, "e4m3": 448.0}


def _types(torch):
    return {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------- rotary positions

def _rot(x, pos, freqs, halves, m=1.0):
    """x [rows][heads][dim] in 64 bits, and per element the sum of magnitudes that goes into it."""
    x = np.asarray(x, np.float64)
    r = 2 * len(freqs)
    a = np.asarray(pos, np.float64)[:, None] * np.asarray(freqs, np.float64)[None]
    co, si = (m * np.cos(a))[:, None], (m * np.sin(a))[:, None]
    one, two = (slice(0, r // 2), slice(r // 2, r)) if halves else (slice(0, r, 2), slice(1, r, 2))
    y, mag = x.copy(), np.abs(x)
    u, w = x[..., one], x[..., two]
    y[..., one], y[..., two] = u * co - w * si, w * co + u * si
    mag[..., one] = mag[..., two] = m * (np.abs(u) + np.abs(w))
    return y, mag


# sine and cosine: the fraction of a turn is rounded once (pi * 2^-24 of an angle), sincospif is good to 2
# units of 2^-24 of 1, mscale and the two products and their sum round once each: under 8 * 2^-24 of |a| + |b|
ROPE_U = 8 * U32


def _rope_tol(mag, freqs, pos):
    """The angle itself is a 64-bit product, here and in the reference: 2^-51 of it, in turns and in radians."""
    far = np.max(np.abs(np.asarray(pos, np.float64))) * np.max(np.abs(freqs)) * 2.0 ** -50
    return mag * (ROPE_U + far)


@pytest.mark.parametrize("rows,heads,dim,rot,halves,dtype", [
    (1, 24, 64, 64, False, "f32"), (1, 1, 64, 64, True, "f16"), (3, 5, 64, 48, False, "f16"), (7, 12, 128, 128, True, "f32"),
    (65, 3, 128, 96, True, "f16"), (33, 4, 64, 6, True, "f32"), (33, 4, 64, 34, False, "f16"), (5, 2, 50, 22, True, "f16"),
    (600, 40, 128, 96, True, "f16"), (2, 64, 512, 512, False, "f32"), (300, 1, 2, 2, True, "f32")])
def test_rope_rows(torch_gpu, rows, heads, dim, rot, halves, dtype):
    torch = torch_gpu
    print(f"rope {rows}x{heads}x{dim} rot {rot} halves {halves} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 31 + rot)
    x = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).to(_types(torch)[dtype])
    pos = rng.integers(-1 << 20, 1 << 20, rows).astype(np.int32)
    f, m = lib.rope_freqs(rot, scaling="yarn", factor=8.0, orig_ctx=2048)
    out = torch.full((rows, heads, dim), float("nan"), dtype=x.dtype, device="cuda")
    lib.rope_rows(x.cuda(), torch.from_numpy(pos).cuda(), lib.Rope(rot, halves=halves, scaling="yarn", factor=8.0, orig_ctx=2048), out)
    got = out.double().cpu().numpy()
    want, mag = _rot(x.double().numpy(), pos, f, halves, m)
    tol = _rope_tol(mag, f, pos) + (np.abs(want) * U16 + 2.0 ** -25 if dtype == "f16" else 0)
    tol[..., rot:] = 0  # copied
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)


def test_rope_extreme_positions(torch_gpu):
    """The ends of int32: the angle's 64-bit product is the only thing that is coarse."""
    torch = torch_gpu
    pos = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31], np.int32)
    x = np.random.default_rng(3).standard_normal((5, 2, 64)).astype(np.float32)
    out = lib.rope_rows(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), lib.Rope(64))
    f, _ = lib.rope_freqs(64)
    want, mag = _rot(x, pos, f, False)
    assert (np.abs(out.double().cpu().numpy() - want) <= _rope_tol(mag, f, pos)).all()
    assert np.array_equal(out[0].cpu().numpy(), x[0])  # position 0 turns nothing


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("dtype,pad,first", [("f32", 0, 0), ("f16", 0, 0), ("f32", 4, 0), ("f32", 3, 1), ("f16", 5, 3)])
def test_rope_strides_and_in_place(torch_gpu, halves, dtype, pad, first):
    """The query and key heads inside fused q | k | v rows, at aligned and odd addresses, into themselves and
    into another tensor: the same values, and nothing beside them touched."""
    torch = torch_gpu
    rng = np.random.default_rng(pad + 10 * first)
    rows, heads, dim = 9, 8, 64
    width = 3 * heads // 2 * dim + pad
    flat = torch.from_numpy(rng.standard_normal(rows * width + 8).astype(np.float32)).to(_types(torch)[dtype]).cuda()
    before = flat.clone()
    view = flat[first:first + rows * width].view(rows, width)[:, :heads * dim].view(rows, heads, dim) if pad == 0 else \
        flat.as_strided((rows, heads, dim), (width, dim, 1), first)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 37
    rope = lib.Rope(64, halves=halves)
    want = torch.empty(rows, heads, dim, dtype=flat.dtype, device="cuda")
    lib.rope_rows(view.contiguous(), pos, rope, want)
    apart = torch.full((rows, heads + 1, dim + 2), 7.0, dtype=flat.dtype, device="cuda")
    lib.rope_rows(view, pos, rope, apart[:, 1:, :dim])
    assert torch.equal(apart[:, 1:, :dim], want) and (apart[:, 0] == 7).all() and (apart[:, :, dim:] == 7).all()
    assert torch.equal(flat, before)
    assert lib.rope_rows(view, pos, rope) is view
    assert torch.equal(view, want)
    rest = torch.ones_like(flat, dtype=torch.bool)
    rest.as_strided((rows, heads, dim), view.stride(), view.storage_offset())[...] = False
    assert torch.equal(flat[rest], before[rest])


def test_rope_heads_outside_rows(torch_gpu):
    """[heads][rows][dim] in memory: rows within the steps of the heads."""
    torch = torch_gpu
    x = torch.randn(7, 5, 64, generator=torch.Generator().manual_seed(1)).cuda()
    pos = torch.arange(7, dtype=torch.int32, device="cuda") * 11
    rope = lib.Rope(64)
    want = lib.rope_rows(x, pos, rope, torch.empty_like(x))
    turned = torch.full((5, 7, 64), 3.0, device="cuda").transpose(0, 1)
    assert torch.equal(lib.rope_rows(x, pos, rope, turned), want)


def test_rope_undone_by_negated_angles(torch_gpu):
    """Negated angles are the inverse, and the gradient: <rope(x), y> = <x, rope^-1(y)>, as differences of
    the 64-bit form say too."""
    torch = torch_gpu
    rng = np.random.default_rng(8)
    x, y = (rng.standard_normal((4, 3, 64)) for _ in range(2))
    pos = np.array([0, 5, 900, 70000], np.int32)
    f, _ = lib.rope_freqs(48)
    back = lib.Rope(halves=True, freqs=torch.from_numpy(-f).cuda())
    g = lib.rope_rows(torch.from_numpy(y.astype(np.float32)).cuda(), torch.from_numpy(pos).cuda(), back).double().cpu().numpy()
    y32 = y.astype(np.float32)
    h = 1e-3
    for e in [(0, 0, 3), (1, 2, 25), (2, 1, 40), (3, 0, 63)]:
        up, dn = x.copy(), x.copy()
        up[e] += h
        dn[e] -= h
        d = ((_rot(up, pos, f, True)[0] - _rot(dn, pos, f, True)[0]) * y32).sum() / (2 * h)  # linear: no error of order h
        assert abs(d - g[e]) <= ROPE_U * 4 * np.abs(y32[e[0], e[1]]).max() + 1e-9


# ---------------------------------------------------------------- the paged cache

def _pool(torch, cache, n_pages, heads, page, dim, fill=0.0):
    p = torch.full((n_pages, heads, page, dim), fill, device="cuda").to(_types(torch)[cache])
    return p, (torch.zeros(n_pages, heads, page, device="cuda") if cache in TOP else None)


def _make_cache(torch, cache, streams, ctx, heads, page, dim, seed=0):
    rng = np.random.default_rng(seed)
    per = (ctx + page - 1) // page
    n = streams * per + 2
    table = torch.from_numpy(rng.permutation(n)[:streams * per].reshape(streams, per).astype(np.int32)).cuda()
    (k, ks), (v, vs) = (_pool(torch, cache, n, heads, page, dim) for _ in range(2))
    return lib.KVCache(k, v, table, ks, vs)


def _stored(torch, x, cache):
    """What the cache gives back for fp32 rows x [..., dim]: the documented steps in numpy's fp32."""
    x = np.asarray(x, np.float32)
    if cache == "f32":
        return x
    if cache == "f16":
        return x.astype(np.float16).astype(np.float32)
    d = np.abs(x).max(-1, keepdims=True) / np.float32(TOP[cache])
    d = np.where(d < 2.0 ** -126, np.float32(0), d).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), 0).astype(np.float32)
    y = np.clip(x * inv, -TOP[cache], TOP[cache])
    if cache == "i8":
        return (np.rint(y) * d).astype(np.float32)
    return torch.from_numpy(y).to(torch.float8_e4m3fn).float().numpy() * d


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache", ["f32", "f16", "i8", "e4m3"])
def test_kv_write_and_read(torch_gpu, cache, dim, dtype):
    """Every value as the documented steps give it, bit for bit, at the edges of pages of 48; positions that nobody
    wrote stay 0, a padded row is skipped, and rows without a place in the cache are not written and read as NaN."""
    torch = torch_gpu
    print(f"kv {cache} {dim} {dtype}", flush=True)
    rng = np.random.default_rng(dim)
    heads, streams = 3, 4
    c = _make_cache(torch, cache, streams, 96, heads, 48, dim)
    stream = np.array([0, 0, 1, 1, 2, 3, 3, 3, 0, 9, -1, 2, 2], np.int32)
    pos = np.array([0, 47, 48, 95, 63, 15, 16, 17, -1, 4, 4, 96, 2 ** 31 - 1], np.int32)
    ok = np.arange(13) < 8
    x = [rng.standard_normal((13, heads, dim)).astype(np.float32) * rng.choice([1e-3, 1.0, 300.0], (13, heads, 1)).astype(np.float32)
         for _ in range(2)]
    x[0][1, 0] = 0.0  # a head of zeros
    x[1][2, 1] = 1e-44  # its scale would be under 2^-126
    x[0][4, 2, :] = np.where(np.arange(dim) == 5, 127.0, 0.5 + np.arange(dim) % 7)  # ties of the rounding
    k, v = (torch.from_numpy(a).to(_types(torch)[dtype]) for a in x)
    s, p = torch.from_numpy(stream).cuda(), torch.from_numpy(pos).cuda()
    lib.kv_write(c, k.cuda(), v.cuda(), s, p)
    ko, vo = (torch.full((13, heads, dim), 5.0, dtype=torch.float32, device="cuda") for _ in range(2))
    lib.kv_read(c, s, p, ko, vo)
    for got, src in ((ko, k), (vo, v)):
        got = got.cpu().numpy()
        assert np.array_equal(got[ok], _stored(torch, src.float().numpy(), cache)[ok])
        assert (got[8] == 5.0).all() and np.isnan(got[9:]).all()
    # everything else in the pools is as it was
    for pool, src in ((c.tensors[0], k), (c.tensors[1], v)):
        live = torch.zeros(pool.shape[:3], dtype=torch.bool)
        table = c.tensors[2].cpu().numpy()
        for r in np.flatnonzero(ok):
            live[table[stream[r], pos[r] // 48], :, pos[r] % 48] = True
        assert (pool.float().cpu()[~live] == 0).all()
    h = [torch.empty(13, heads * dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    lib.kv_read(c, s, p, *h)  # the same values rounded once more
    assert torch.equal(h[0][:8], ko[:8].reshape(8, -1).half()) and torch.equal(h[1][:8], vo[:8].reshape(8, -1).half())


def test_kv_read_of_bad_pages(torch_gpu):
    torch = torch_gpu
    c = _make_cache(torch, "i8", 2, 64, 2, 32, 64)
    table = c.tensors[2]
    table[0, 1], table[1, 0] = -1, 10 ** 6
    s = torch.tensor([0, 0, 1, 1], dtype=torch.int32, device="cuda")
    p = torch.tensor([31, 32, 0, 40], dtype=torch.int32, device="cuda")
    x = torch.ones(4, 2, 64, device="cuda")
    lib.kv_write(c, x, x, s, p)
    k, v = torch.zeros_like(x), torch.zeros_like(x)
    lib.kv_read(c, s, p, k, v)
    for t in (k, v):
        assert (t[[0, 3]] - 1).abs().max() <= 2 * U32 and torch.isnan(t[[1, 2]]).all()


@pytest.mark.parametrize("cache", ["i8", "e4m3", "f16", "f32"])
def test_kv_inf_and_nan(torch_gpu, cache):
    """An 8-bit head that holds one reads back as NaN; its neighbours are as ever."""
    torch = torch_gpu
    c = _make_cache(torch, cache, 1, 16, 2, 16, 64)
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(1))
    x[0, 0, 7], x[1, 1, 0], x[2, 0, 63] = float("inf"), float("nan"), -float("inf")
    s, p = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    lib.kv_write(c, x.cuda(), x.flip(0).cuda(), s, p)
    k, v = (torch.empty(3, 2, 64, device="cuda") for _ in range(2))
    lib.kv_read(c, s, p, k, v)
    want = np.array([_stored(torch, r, cache) if cache not in TOP or np.isfinite(r).all() else np.full(64, np.nan, np.float32)
                     for r in x.reshape(6, 64).numpy()]).reshape(3, 2, 64)
    np.testing.assert_array_equal(k.cpu().numpy(), want)
    np.testing.assert_array_equal(v.cpu().numpy(), want[::-1])


@pytest.mark.parametrize("dim,rot,halves,dtype,pad", [(64, 64, False, "f32", 0), (64, 64, True, "f16", 0), (128, 96, True, "f32", 0),
                                                      (128, 50, True, "f16", 3), (64, 18, False, "f32", 1), (128, 128, False, "f16", 8)])
@pytest.mark.parametrize("cache", ["f32", "i8", "e4m3"])
def test_kv_write_rotates_keys(torch_gpu, cache, dim, rot, halves, dtype, pad):
    """Keys turned at positions of their own on the way in; rows of any stride.  Against 64 bits: the rotation's
    tolerance, and half a step of the cache (which may be the neighbouring one where that tips it)."""
    torch = torch_gpu
    print(f"kv rope {cache} {dim} {rot} {halves} {dtype} {pad}", flush=True)
    rng = np.random.default_rng(dim + rot)
    n, heads = 21, 2
    c = _make_cache(torch, cache, 1, 32, heads, 16, dim)
    rows = [torch.from_numpy(rng.standard_normal((n, heads * dim + pad)).astype(np.float32)).to(_types(torch)[dtype]).cuda() for _ in range(2)]
    k, v = (r[:, pad:] if pad else r for r in rows)
    pos = torch.from_numpy(rng.permutation(32)[:n].astype(np.int32)).cuda()
    depth = rng.integers(0, 100000, n).astype(np.int32)
    s = torch.zeros(n, dtype=torch.int32, device="cuda")
    lib.kv_write(c, k, v, s, pos, rope=lib.Rope(rot, halves=halves), rope_pos=torch.from_numpy(depth).cuda())
    ko, vo = (torch.empty(n, heads, dim, device="cuda") for _ in range(2))
    lib.kv_read(c, s, pos, ko, vo)
    assert np.array_equal(vo.cpu().numpy(), _stored(torch, v.float().cpu().numpy().reshape(n, heads, dim), cache))
    f, _ = lib.rope_freqs(rot)
    want, mag = _rot(k.double().cpu().numpy().reshape(n, heads, dim), depth, f, halves)
    tol = _rope_tol(mag, f, depth)
    if cache in TOP:
        top = np.abs(want).max(-1, keepdims=True)
        step = top / 127 if cache == "i8" else np.maximum(np.abs(want) * 2.0 ** -3, top / 448 * 2.0 ** -9)
        tol = 2 * tol + step / 2 * (1 + 2.0 ** -10) + 4 * U32 * np.abs(want)
    assert (np.abs(ko.double().cpu().numpy() - want) <= tol).all()


# ---------------------------------------------------------------- attention

def _rows_of(c, which, s, n):
    """The first n positions of stream s in 64 bits: [heads][n][dim]."""
    import torch
    pool, scale = c.tensors[which], c.tensors[3 + which]
    page = pool.shape[2]
    pages = c.tensors[2][s, :(n + page - 1) // page].long()
    x = pool.view(torch.int8)[pages].view(pool.dtype).double()
    if scale is not None:
        x = x * scale[pages].double()[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :n].cpu().numpy()


def _attn_ref(q, c, start, ctx, mask, scale, rows, heads):
    """out, lse, their tolerances for 32-bit outputs, and sum p |v|, from 64 bits.

    A score's error: the query's hi + lo (2^-21 of each value) and fp32 products and sums (the chain of D / 32
    matrix instructions and the scales, 16 roundings), of scale * sum |q k|: es = 24 * 2^-24 of it.  A weight
    e^s is then off by es, exp2's 2^-22 and hi + lo's 2^-21; sums add a chain of keys / 16 + 64 roundings.  Both
    the weighted sum and the normaliser carry it: twice."""
    out = np.zeros((rows, heads, c.head_dim))
    lse = np.full((rows, heads), -np.inf)
    tol, ltol, avg = np.zeros_like(out), np.zeros_like(lse), np.zeros_like(out)
    for s in range(len(ctx)):
        a, b = int(start[s]), int(start[s + 1])
        n = int(ctx[s]) + b - a
        if b == a:
            continue
        k, v = _rows_of(c, 0, s, n), _rows_of(c, 1, s, n)
        for r in range(a, b):
            m = (2 << (r - a)) - 1 if mask is None else int(mask[r])
            see = np.array([j < ctx[s] or (m >> (j - int(ctx[s]))) & 1 for j in range(n)], bool)
            if not see.any():
                continue
            for h in range(heads):
                kk, vv = k[h * c.kv_heads // heads][see], v[h * c.kv_heads // heads][see]
                qq = q[r, h].astype(np.float64)
                x = scale * (kk @ qq)
                x_mag = abs(scale) * (np.abs(kk) @ np.abs(qq))
                e = np.exp(x - x.max())
                p = e / e.sum()
                out[r, h] = p @ vv
                lse[r, h] = x.max() + np.log(e.sum())
                err = 24 * U32 * x_mag.max() + 8 * U32 + (n / 16 + 64) * U32
                avg[r, h] = p @ np.abs(vv)
                tol[r, h] = 2 * err * avg[r, h]
                ltol[r, h] = err + 4 * U32 * (abs(lse[r, h]) + abs(x.max()))
    return out, lse, tol, ltol, avg


def _tree_masks(rng, n, chain):
    m = []
    for i in range(n):
        parent = i - 1 if chain else int(rng.integers(-1, i))
        m.append((m[parent] if parent >= 0 else 0) | (1 << i))
    return m


def _fill(torch, c, seed, keep=None):
    """Every slot of the pools random, through the cache's own format."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for which in (0, 1):
        pool, scale = c.tensors[which], c.tensors[3 + which]
        x = torch.randn(pool.shape, generator=g, device="cuda")
        if scale is None:
            pool.copy_(x)
        else:
            top = 127.0 if pool.dtype == torch.int8 else 448.0
            scale.copy_(x.abs().amax(-1) / top * (0.5 + torch.rand(scale.shape, generator=g, device="cuda")))
            y = (x / scale[..., None]).clamp(-top, top)
            pool.copy_(y.round() if pool.dtype == torch.int8 else y)


def _attn_case(torch, cache, dim, heads, kvh, page, ctx, n, chain, seed, qdt="f32"):
    rng = np.random.default_rng(seed)
    streams = len(ctx)
    c = _make_cache(torch, cache, streams, max(a + b for a, b in zip(ctx, n)) or 1, kvh, page, dim, seed)
    _fill(torch, c, seed)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    rows = int(start[-1])
    masks = sum((_tree_masks(rng, k, chain) for k in n), [])
    q = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32) * 1.5).to(_types(torch)[qdt])
    return c, start, rows, masks, q


def _dev_masks(torch, masks):
    return torch.from_numpy(np.array(masks, np.uint64).view(np.int64)).cuda()


def _run_attn(torch, c, q, start, ctx, masks, max_rows, max_keys, odt="f32", scale=None, **kw):
    out = torch.full(q.shape, 9.0, dtype=_types(torch)[odt], device="cuda")
    lse = torch.full(q.shape[:2], 9.0, device="cuda")
    lib.attn_tree(q.cuda(), c, torch.from_numpy(start).cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), out, max_rows,
                  max_keys, row_mask=None if masks is None else _dev_masks(torch, masks), lse=lse, scale=scale, **kw)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def _check_attn(torch, c, q, start, ctx, masks, odt="f32", max_rows=None, max_keys=None, scale=None, **kw):
    n = np.diff(start)
    got, lse = _run_attn(torch, c, q, start, ctx, masks, max_rows or int(n.max()), max_keys or int((np.array(ctx) + n).max()), odt, scale, **kw)
    want, wl, tol, ltol, avg = _attn_ref(q.float().numpy(), c, start, ctx, masks, c.head_dim ** -0.5 if scale is None else scale,
                                         q.shape[0], q.shape[1])
    if odt == "f16":
        # the output's rounding, 2^-11 of it; with more than 64 packed rows the weights are fp16 too, each off by up to
        # 2^-11 of itself (times a value scale, as the sum is), so sum p v by up to 2^-11 sum p |v|
        tol = tol + np.abs(want) * U16 + 2.0 ** -25 + (avg * U16 if (max_rows or n.max()) * q.shape[1] // c.kv_heads > 64 and c.tensors[0].dtype != torch.float32 else 0)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], np.max(np.abs(got - want)), tol[bad][:5])
    fin = np.isfinite(wl)
    assert np.array_equal(fin, np.isfinite(lse)) and (np.abs(lse - wl)[fin] <= ltol[fin]).all()
    assert (lse[~fin] == -np.inf).all() and (got[~fin] == 0).all()
    return got, lse


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("dim,heads,kvh,page", [(64, 12, 12, 64), (128, 8, 2, 16), (64, 15, 5, 48), (128, 3, 3, 128)])
def test_attn_one_row(torch_gpu, cache, dim, heads, kvh, page):
    """A decode step: one row per stream, contexts from none to several splits, at the edges of spans and pages."""
    torch = torch_gpu
    print(f"attn one row {cache} {dim} {heads}/{kvh} page {page}", flush=True)
    ctx = [0, 1, 14, 15, 16, 31, 32, 62, 63, 64, 127, 128, 255, 256, 511, 700]
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, page, ctx, [1] * len(ctx), True, dim + heads)
    _check_attn(torch, c, q, start, ctx, None)
    _check_attn(torch, c, q, start, ctx, masks, odt="f16")


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("dim,heads,kvh,page,n", [(64, 4, 4, 64, [17, 1, 0, 33, 64]), (128, 8, 2, 16, [5, 16, 3]), (64, 8, 1, 32, [64, 7]),
                                                  (128, 2, 2, 48, [2, 31])])
def test_attn_trees(torch_gpu, cache, dim, heads, kvh, page, n):
    """Trees of several sizes under their ancestor masks: one to four row tiles, several groups of them."""
    torch = torch_gpu
    print(f"attn trees {cache} {dim} {heads}/{kvh} page {page} {n}", flush=True)
    ctx = [90, 0, 40, 129, 300][:len(n)]
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, page, ctx, n, False, sum(n), qdt="f16")
    _check_attn(torch, c, q, start, ctx, masks)
    _check_attn(torch, c, q.float() * 1.37, start, ctx, None, odt="f16")


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,kvh,n", [(64, 12, 12, [1] * 16), (64, 12, 12, [27, 1, 0, 14] * 4), (128, 8, 2, [4, 2] * 24), (128, 4, 4, [32, 7]),
                                             (64, 8, 8, [33, 64, 5])])
def test_attn_under_other_bounds(torch_gpu, cache, dim, heads, kvh, n):
    """The bound on the keys chooses how they are shared out (by waves of one workgroup, or cut and joined): the same rows
    under their own bound, one key more than short lengths, and a far one."""
    torch = torch_gpu
    print(f"attn bounds {cache} {dim} {heads}/{kvh} {n[:4]}", flush=True)
    ctx = [int(k) for k in np.random.default_rng(len(n)).integers(0, 480, len(n))]
    ctx[0], ctx[-1] = 470, 0
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, 32, ctx, n, False, sum(n))
    for bound in (None, 513, 1025, 1537, 9000):
        _check_attn(torch, c, q, start, ctx, masks, max_keys=bound)


@pytest.mark.parametrize("cache,dim,n", [("f16", 64, 1), ("i8", 128, 1), ("e4m3", 64, 3), ("f32", 64, 2), ("i8", 64, 40)])
def test_attn_long_context(torch_gpu, cache, dim, n):
    """Keys cut over workgroups and joined; a short stream beside a long one leaves whole splits without keys."""
    torch = torch_gpu
    print(f"attn long {cache} {dim} {n}", flush=True)
    ctx = [20011, 100]
    c, start, rows, masks, q = _attn_case(torch, cache, dim, 4, 2, 64, ctx, [n, n], False, n)
    assert lib.attn_tree_workspace(c, 4, rows, n, 20011 + n) > 0
    a = _check_attn(torch, c, q, start, ctx, masks)
    b = _run_attn(torch, c, q, start, ctx, masks, n, 20011 + n)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])  # the same call, the same bits
    # room for more than there is changes the split, not what comes out beyond rounding
    _check_attn(torch, c, q, start, ctx, masks, max_rows=64, max_keys=20011 + 64)


@pytest.mark.parametrize("streams,heads,kvh,dim", [(70, 2, 1, 64), (66, 16, 1, 128), (5, 2, 2, 64), (9, 8, 1, 128), (64, 2, 1, 64), (33, 3, 1, 128),
                                                     (17, 2, 2, 64)])
def test_attn_cuts_of_ragged_streams(torch_gpu, streams, heads, kvh, dim):
    """Keys cut into pieces over up to 64 streams by their lengths, and over more as many each: streams without rows, without
    a context and with a bad one among long and short ones."""
    torch = torch_gpu
    rng = np.random.default_rng(streams)
    ctx = [int(x) for x in rng.integers(0, 2600, streams)]
    n = [int(x) for x in rng.integers(0, 4, streams)]
    ctx[0], n[0], ctx[1], n[1], ctx[2] = 2600, 3, 0, 2, 1
    n[-1] = 1
    print(f"attn cuts {streams} {heads}/{kvh} {dim}", flush=True)
    c, start, rows, masks, q = _attn_case(torch, "i8", dim, heads, kvh, 64, ctx, n, False, streams)
    assert lib.attn_tree_workspace(c, heads, rows, 3, 2603) > 0
    a = _check_attn(torch, c, q, start, ctx, masks, max_rows=3, max_keys=2603)
    bad = list(ctx)
    bad[-1] = -5
    b = _run_attn(torch, c, q, start, bad, masks, 3, 2603)
    assert np.isnan(b[0][-1]).all() and (streams > 64 or np.abs(b[0][:-1] - a[0][:-1]).max() < 1e-5)
    # a workspace of the size that was asked for, with guards around it, full of NaN
    size = lib.attn_tree_workspace(c, heads, rows, 3, 2603)
    ws = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")
    d = _run_attn(torch, c, q, start, ctx, masks, 3, 2603, workspace=ws[256:256 + size])
    assert np.array_equal(d[0], a[0]) and (ws[:256] == 255).all() and (ws[256 + size:] == 255).all()


def test_attn_more_rows_than_max_rows(torch_gpu):
    """A stream's rows past max_rows stay as they were, and are no keys."""
    torch = torch_gpu
    c, start, rows, masks, q = _attn_case(torch, "f16", 64, 2, 2, 16, [20, 3], [5, 2], True, 8)
    got, lse = _run_attn(torch, c, q, start, [20, 3], None, 3, 25)
    want, _, tol, _, _ = _attn_ref(q.numpy(), c, start, [20, 3], None, 0.125, rows, 2)
    keep = [0, 1, 2, 5, 6]
    assert (np.abs(got - want) <= tol)[keep].all() and (got[3:5] == 9).all() and (lse[3:5] == 9).all()


def test_attn_empty_rows_and_masks(torch_gpu):
    """Rows that see nothing, bits beyond the stream's rows, rows of no stream, a stream without rows."""
    torch = torch_gpu
    ctx, n = [0, 5, 0, 3], [4, 3, 0, 2]
    c, start, rows, masks, q = _attn_case(torch, "i8", 64, 2, 2, 16, ctx, n, False, 2)
    masks[0], masks[2], masks[4] = 0, 1 << 60, 0
    masks[3] |= 1 << 63
    want_masks = [m & 0xF if r < 4 else m for r, m in enumerate(masks)]
    got, _ = _run_attn(torch, c, q, start, ctx, masks, 4, 9)
    want, wl, tol, _, _ = _attn_ref(q.numpy(), c, start, ctx, want_masks, 0.125, rows, 2)
    assert (np.abs(got - want) <= tol).all() and (got[[0, 2]] == 0).all()
    # rows behind the last stream's stay as they were
    q2 = torch.cat([q, torch.ones(3, 2, 64)])
    got2, lse2 = _run_attn(torch, c, q2, start, ctx, masks + [1, 1, 1], 4, 9)
    assert np.array_equal(got2[:rows], got) and (got2[rows:] == 9).all() and (lse2[rows:] == 9).all()


def test_attn_what_only_the_device_sees(torch_gpu):
    """Keys past max_keys or the table, a negative context and a bad page give NaN rows; a row range outside [0, rows]
    gives none; the streams beside them are as ever."""
    torch = torch_gpu
    n = [2] * 6
    ctx = [40, 40, 40, 40, 40, 40]
    c, start, rows, masks, q = _attn_case(torch, "f16", 64, 2, 1, 16, ctx, n, True, 4)
    good, _ = _run_attn(torch, c, q, start, ctx, None, 2, 42)
    bad_ctx = [40, 41, -1, 40, 2 ** 31 - 1, 40]  # 41 + 2 keys: more than max_keys
    c.tensors[2][3, 1] = c.tensors[0].shape[0]  # outside the pool
    got, lse = _run_attn(torch, c, q, start, bad_ctx, None, 2, 42)
    for s in (1, 2, 3, 4):
        assert np.isnan(got[2 * s:2 * s + 2]).all() and np.isnan(lse[2 * s:2 * s + 2]).all(), s
    for s in (0, 5):
        assert np.array_equal(got[2 * s:2 * s + 2], good[2 * s:2 * s + 2])
    got, _ = _run_attn(torch, c, q, start, [40, 48, 40, 40, 40, 40], None, 2, 64)  # 3 pages of 16 hold 48
    assert np.isnan(got[2:4]).all()
    odd = start.copy()
    odd[0], odd[6] = -1, rows + 1
    got, _ = _run_attn(torch, c, q, odd, ctx, None, 2, 42)
    assert (got[:2] == 9).all() and (got[10:] == 9).all() and np.array_equal(got[2:6], good[2:6])


@pytest.mark.parametrize("cache", ["f16", "f32", "i8", "e4m3"])
@pytest.mark.parametrize("n", [6, 40])
def test_attn_inf_and_nan_behind_the_mask(torch_gpu, cache, n):
    """What a row does not attend may hold anything: slots behind the last, and drafted slots that other rows see.
    Rows that do see such a slot become NaN (or Inf) where the formula does."""
    torch = torch_gpu
    ctx = [37, 70]
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 4, 2, 16, ctx, [n, n], False, 77)
    masks = [m & ~(1 << 2) for m in masks]  # nobody sees drafted slot 2 ...
    clean, _ = _check_attn(torch, c, q, start, ctx, masks)
    table = c.tensors[2].cpu().numpy()

    def poison(s, p, value):
        for which in (0, 1):
            pool, scale = c.tensors[which], c.tensors[3 + which]
            at = (int(table[s, p // 16]), slice(None), p % 16)
            if scale is not None:
                scale[at] = value
            if pool.dtype == torch.float8_e4m3fn:
                pool.view(torch.int8)[at] = 0x7f
            elif pool.dtype != torch.int8:
                pool[at] = value
    poison(0, 37 + 2, float("nan"))
    poison(1, 70 + 2, float("inf"))
    for p in range(37 + n, table.shape[1] * 16):  # ... nor what lies behind the rows
        poison(0, p, float("nan"))
    got, _ = _run_attn(torch, c, q, start, ctx, masks, n, 70 + n)
    assert np.isfinite(got).all() and np.array_equal(got, clean)
    one = [m | (1 << 2) if r in (1, n + 3) else m for r, m in enumerate(masks)]
    got, _ = _run_attn(torch, c, q, start, ctx, one, n, 70 + n)
    hit = np.isin(np.arange(rows), (1, n + 3))
    assert not np.isfinite(got[hit]).any(), got[hit]
    assert np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_attn_scales_far_apart(torch_gpu, cache):
    """Value scales over twelve orders of magnitude, rising and falling along the context, and zeros among them."""
    torch = torch_gpu
    ctx = [900]
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 2, 2, 64, ctx, [3], True, 5)
    g = torch.Generator(device="cuda").manual_seed(4)
    scale = c.tensors[4]
    scale.copy_(10.0 ** (12 * torch.rand(scale.shape, generator=g, device="cuda") - 6))
    scale[torch.rand(scale.shape, generator=g, device="cuda") < 0.1] = 0.0
    _check_attn(torch, c, q * 0.2, start, ctx, None)
    scale.zero_()
    got, _ = _run_attn(torch, c, q, start, ctx, None, 3, 903)
    assert (got == 0).all()


def test_attn_large_queries_and_scores(torch_gpu):
    """Queries far past fp16's range, scores of thousands: one key takes all the weight; scale 0 and a negative scale."""
    torch = torch_gpu
    ctx = [300, 20]
    c, start, rows, masks, q = _attn_case(torch, "f16", 64, 2, 2, 32, ctx, [2, 2], True, 6)
    for f in (1e6, 1e-12):
        got, lse = _run_attn(torch, c, q * f, start, ctx, None, 2, 302)
        want, wl, tol, ltol, _ = _attn_ref((q * f).numpy(), c, start, ctx, None, 0.125, rows, 2)
        gap = f < 1 or 24 * U32 * 0.125 * float((q.abs() * f).sum(-1).max()) * 5 < 1  # scores exact enough to rank
        assert np.isfinite(got).all() and np.isfinite(lse).all()
        if gap:
            assert (np.abs(got - want) <= tol).all()
    _check_attn(torch, c, q, start, ctx, None, scale=0.0)
    _check_attn(torch, c, q, start, ctx, None, scale=-0.3)


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_attn_inf_and_nan_queries(torch_gpu, cache, n):
    """A head of a row with a NaN or an Inf in its query is NaN; not a bit of any other changes, those packed with it
    among them.  In place, the output over the query, gives the same."""
    torch = torch_gpu
    print(f"attn queries {cache} {n}", flush=True)
    ctx = [700, 45]
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 8, 2, 32, ctx, [n, n], False, 40 + n)
    a, la = _run_attn(torch, c, q, start, ctx, masks, n, 700 + n)
    odd = q.clone()
    odd[0, 1, 5], odd[rows - 1, 4, 63], odd[rows - 1, 7, 0] = math.nan, math.inf, -math.inf
    b, lb = _run_attn(torch, c, odd, start, ctx, masks, n, 700 + n)
    bad = np.zeros((rows, 8), bool)
    bad[0, 1] = bad[rows - 1, 4] = bad[rows - 1, 7] = True
    assert np.isnan(b[bad]).all() and np.isnan(lb[bad]).all()
    assert np.array_equal(a[~bad], b[~bad]) and np.array_equal(la[~bad], lb[~bad])
    x = q.cuda()
    lib.attn_tree(x, c, torch.from_numpy(start).cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), x, n, 700 + n,
                  row_mask=_dev_masks(torch, masks))
    assert np.array_equal(x.double().cpu().numpy(), a)


def test_attn_strided_rows(torch_gpu):
    """Queries inside wider rows and at odd addresses, outputs inside wider rows; nothing beside them is written."""
    torch = torch_gpu
    ctx = [70, 9]
    c, start, rows, masks, q = _attn_case(torch, "i8", 64, 4, 2, 16, ctx, [3, 5], False, 9)
    want, wl = _run_attn(torch, c, q, start, ctx, masks, 5, 75)
    wide = torch.full((rows, 4 * 64 + 7), 3.0, device="cuda")
    wide[:, 3:3 + 256] = q.reshape(rows, -1).cuda()
    out = torch.full((rows, 300), 9.0, device="cuda")
    lib.attn_tree(wide[:, 3:3 + 256], c, torch.from_numpy(start).cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), out[:, 1:257],
                  5, 75, row_mask=_dev_masks(torch, masks))
    got = out.double().cpu().numpy()
    assert np.array_equal(got[:, 1:257], want.reshape(rows, -1)) and (got[:, 0] == 9).all() and (got[:, 257:] == 9).all()


def test_attn_equals_attn_paged(torch_gpu):
    """A decode step over the same fp16 pages as moss_hip_attn_paged: both within their own rounding of each other."""
    torch = torch_gpu
    ctx = [5, 63, 64, 300]
    c, start, rows, masks, q = _attn_case(torch, "f16", 64, 12, 12, 64, ctx, [1] * 4, True, 12)
    got, _ = _check_attn(torch, c, q, start, ctx, None)
    _, _, tol, _, _ = _attn_ref(q.numpy(), c, start, ctx, None, 0.125, rows, 12)
    out = torch.empty(4, 768, device="cuda")
    lib.attn_paged(q.reshape(4, 768).cuda(), c.tensors[0], c.tensors[1], 12, c.tensors[2], c.tensors[2].shape[1], 64,
                   torch.tensor(ctx, dtype=torch.int32, device="cuda"), 301, out)
    assert (np.abs(out.double().cpu().numpy().reshape(got.shape) - got) <= 2 * tol).all()


def test_attn_offsets_past_32_bits(torch_gpu):
    """A pool of more than 2^32 bytes, its last pages in use."""
    torch = torch_gpu
    page, heads, dim = 16384, 8, 128
    n = 2 ** 32 // (page * heads * dim) + 2
    k = torch.zeros(n, heads, page, dim, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.ones(n, heads, page, device="cuda") for _ in range(2))
    table = torch.tensor([[n - 1, n - 2]], dtype=torch.int32, device="cuda")
    c = lib.KVCache(k, v, table, ks, vs)
    x = torch.randn(40, heads, dim, generator=torch.Generator().manual_seed(2)).cuda()
    pos = torch.arange(page - 30, page + 10, dtype=torch.int32, device="cuda")
    s = torch.zeros(40, dtype=torch.int32, device="cuda")
    lib.kv_write(c, x, 2 * x, s, pos)
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    lib.kv_read(c, s, pos, ko, vo)
    assert np.array_equal(ko.cpu().numpy(), _stored(torch, x.cpu().numpy(), "i8"))
    q = torch.randn(1, heads, dim, generator=torch.Generator().manual_seed(3))
    _check_attn(torch, c, q, np.array([0, 1], np.int32), [page + 9], None)
    del k, v, c
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- log probabilities

def _lp_ref(x, tokens, inv_t, k):
    """logprob, entropy, ids and their log probabilities in 64 bits, and a tolerance.

    z = x / T rounds once (2^-24 |z|); a term e^(z - m) is off by that, by exp2's argument (2^-24 |z - m|) and by 2 units;
    sums chain at most 32 + 16 + 128 roundings; the logarithm adds 4 units of its value."""
    z = np.asarray(x, np.float64) * float(np.float32(inv_t))
    rows, vocab = z.shape
    lp, ent = np.full(rows, -np.inf), np.zeros(rows)
    ids, top = np.full((rows, k), -1), np.full((rows, k), -np.inf)
    tol = np.zeros(rows)
    for r in range(rows):
        order = [i for i in np.lexsort((np.arange(vocab), -z[r])) if z[r, i] > -np.inf][:k]
        ok = z[r] > -np.inf
        if ok.any():
            m = z[r][ok].max()
            lse = m + np.log(np.exp(z[r][ok] - m).sum())
            p = np.exp(z[r][ok] - lse)
            t = tokens[r]
            lp[r] = z[r, t] - lse if 0 <= t < vocab else np.nan
            ent[r] = -(p * (z[r][ok] - lse)).sum()
            ids[r, :len(order)] = order
            top[r, :len(order)] = z[r, order] - lse
            spread = (p * np.abs(z[r][ok] - m)).sum()
            tol[r] = U32 * (4 * np.abs(z[r][ok]).max() + 4 * spread + 200 + 4 * abs(lse - m)) * (1 + spread)
        elif not 0 <= tokens[r] < vocab:
            lp[r] = np.nan
    return lp, ent, ids, top, tol


def _run_lp(torch, x, tokens, k, inv_t=1.0, **kw):
    rows = x.shape[0]
    lp, ent = (torch.full((rows,), 9.0, device="cuda") for _ in range(2))
    ids = torch.full((rows, k), 99, dtype=torch.int32, device="cuda")
    top = torch.full((rows, k), 9.0, device="cuda")
    lib.token_logprobs(x, torch.tensor(tokens, dtype=torch.int32, device="cuda"), lp, ent, ids, top, inv_temperature=inv_t, **kw)
    torch.cuda.synchronize()
    return lp.double().cpu().numpy(), ent.double().cpu().numpy(), ids.cpu().numpy(), top.double().cpu().numpy()


def _check_lp(torch, x, tokens, k, inv_t=1.0):
    lp, ent, ids, top = _run_lp(torch, x, tokens, k, inv_t)
    wlp, went, wids, wtop, tol = _lp_ref(x.float().cpu().numpy(), tokens, inv_t, k)
    assert np.array_equal(ids, wids), (ids[(ids != wids).any(1)][:2], wids[(ids != wids).any(1)][:2])
    assert np.array_equal(np.isnan(lp), np.isnan(wlp))
    fin = np.isfinite(wlp)
    assert (np.abs(lp[fin] - wlp[fin]) <= tol[fin]).all(), np.max(np.abs(lp[fin] - wlp[fin]) - tol[fin])
    assert (lp[wlp == -np.inf] == -np.inf).all()
    assert (np.abs(ent - went) <= tol).all()
    fin = np.isfinite(wtop)
    assert np.array_equal(fin, np.isfinite(top)) and (np.abs(top[fin] - wtop[fin]) <= np.broadcast_to(tol[:, None], top.shape)[fin]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 5), (1, 1023, 0), (16, 1024, 5), (5, 1025, 32), (3, 2049, 20), (2, 16384, 32), (1100, 2500, 3),
                                          (300, 16384, 7), (1, 262145, 32), (2, 50001, 8)])
def test_token_logprobs(torch_gpu, dtype, rows, vocab, k):
    """One chunk and several, one value and many, fewer tokens than alternatives; ties in fp16."""
    torch = torch_gpu
    print(f"logprobs {rows}x{vocab} top {k} {dtype}", flush=True)
    rng = np.random.default_rng(vocab + k)
    x = torch.from_numpy((3 * rng.standard_normal((rows, vocab))).astype(np.float32)).to(_types(torch)[dtype]).cuda()
    _check_lp(torch, x, rng.integers(0, vocab, rows), k, 1.0 if rows % 2 else 0.7)


@pytest.mark.parametrize("vocab", [700, 1024, 5000, 16384, 70001])
def test_token_logprobs_ties_and_ruled_out(torch_gpu, vocab):
    """All equal; few values many times over; +0 and -0; most or all tokens ruled out; the type's lowest value; tokens
    outside the vocabulary."""
    torch = torch_gpu
    rng = np.random.default_rng(vocab)
    x = np.zeros((9, vocab), np.float32)
    x[1] = rng.integers(-2, 3, vocab)
    x[2] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[3] = -np.inf
    x[4] = -np.inf
    x[4, [vocab - 1, 3, vocab // 2]] = [1.0, 1.0, 5.0]
    x[5] = np.finfo(np.float32).min
    x[5, 17] = 2.0
    x[6] = np.arange(vocab) / 64  # rising: the best come last
    x[7] = -np.arange(vocab) / 64
    x[8] = np.where(np.arange(vocab) % 256 == 3, 5 + rng.standard_normal(vocab), rng.standard_normal(vocab))  # one thread's share
    tokens = [0, vocab - 1, 1, 0, 3, 17, -1, vocab, 3]
    _check_lp(torch, torch.from_numpy(x).cuda(), tokens, 32)


@pytest.mark.parametrize("vocab", [700, 5000, 70001])
@pytest.mark.parametrize("inv_t", [1.5, 1e-38, 3e38])
def test_token_logprobs_scaled_past_the_range(torch_gpu, vocab, inv_t):
    """The type's lowest value everywhere, in all places but one and in all but two, under temperatures that scale it past
    the type's range, or everything to nothing.  The exact results are log vocab, log 2 and 0: the sum of vocab equal
    terms is off by vocab / 256 + 16 units at most, the logarithm by 4."""
    torch = torch_gpu
    low = float(np.finfo(np.float32).min)
    x = np.full((4, vocab), low, np.float32)
    x[1, 17] = x[2, [17, vocab - 1]] = 2.0
    x[3] = 0.0
    lp, ent, ids, top = _run_lp(torch, torch.from_numpy(x).cuda(), [vocab - 1, 17, 17, 5], 3, inv_t)
    assert np.array_equal(ids, [[0, 1, 2], [17, 0, 1], [17, vocab - 1, 0], [0, 1, 2]])
    even = math.log(vocab)
    tol = U32 * (vocab / 256 + 16 + 4 * even)
    for r in (0, 3):
        assert abs(lp[r] + even) <= tol and abs(ent[r] - even) <= tol and (np.abs(top[r] + even) <= tol).all()
    if inv_t < 1:  # differences of 3.4 * (1 +- 2^-24), each rounded twice, in 64 bits
        z = np.where(np.arange(vocab) == 17, 0.0, low * np.float64(np.float32(inv_t)))
        p = np.exp(z - np.log(np.exp(z).sum()))
        assert abs(lp[1] - math.log(p[17])) <= tol + 16 * U32 and abs(ent[1] + (p * np.log(p)).sum()) <= 16 * (tol + 16 * U32)
    else:
        assert lp[1] == 0 and ent[1] == 0 and top[1, 0] == 0 and (top[1, 1:] == -np.inf).all()
        assert abs(lp[2] + math.log(2)) <= 8 * U32 and abs(ent[2] - math.log(2)) <= 8 * U32 and top[2, 2] == -np.inf


@pytest.mark.parametrize("vocab", [1000, 40000])
def test_token_logprobs_nan_and_inf(torch_gpu, vocab):
    """A NaN or +inf makes the row's probabilities NaN; NaN is no alternative; rows beside it are as ever."""
    torch = torch_gpu
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, vocab)).astype(np.float32)
    x[1, 7], x[2, vocab - 1], x[3] = np.nan, np.inf, np.nan
    lp, ent, ids, top = _run_lp(torch, torch.from_numpy(x).cuda(), [7, 7, 7, 7, 7], 3)
    assert np.isnan(lp[1:4]).all() and np.isnan(ent[1:4]).all()
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")
    for r in (0, 1, 2, 4):
        assert np.array_equal(ids[r], order[r, :3])
    assert (ids[3] == -1).all() and (top[3] == -np.inf).all() and np.isnan(top[1:3]).all()
    wlp, went, _, wtop, tol = _lp_ref(x[[0, 4]], [7, 7], 1.0, 3)
    assert (np.abs(lp[[0, 4]] - wlp) <= tol).all() and (np.abs(top[[0, 4]] - wtop) <= tol[:, None]).all()


def test_token_logprobs_stays_in_its_workspace(torch_gpu):
    """Guards around a workspace of the size that was asked for, odd numbers of chunks and alternatives."""
    torch = torch_gpu
    x = torch.randn(3, 21003, generator=torch.Generator().manual_seed(3)).cuda()
    for k in (0, 1, 5, 32):
        size = lib.token_logprobs_workspace(3, 21003, k)
        assert size > 0
        ws = torch.full((size + 512,), 255, dtype=torch.uint8, device="cuda")
        a = _run_lp(torch, x, [1, 2, 3], k, workspace=ws[256:256 + size])
        b = _run_lp(torch, x, [1, 2, 3], k)
        assert all(np.array_equal(p, q) for p, q in zip(a, b)) and (ws[:256] == 255).all() and (ws[256 + size:] == 255).all()


def test_token_logprobs_strides_and_no_extras(torch_gpu):
    """Rows inside wider rows at odd addresses; without entropy and alternatives."""
    torch = torch_gpu
    rng = np.random.default_rng(2)
    for dtype in ("f32", "f16"):
        wide = torch.from_numpy(rng.standard_normal((6, 3007)).astype(np.float32)).to(_types(torch)[dtype]).cuda()
        for first in (0, 1, 4):
            x = wide[:, first:first + 2999]
            a = _run_lp(torch, x, [5] * 6, 4)
            b = _run_lp(torch, x.contiguous(), [5] * 6, 4)
            assert all(np.array_equal(p, q) for p, q in zip(a, b))
            lp = torch.empty(6, device="cuda")
            lib.token_logprobs(x, torch.full((6,), 5, dtype=torch.int32, device="cuda"), lp)
            assert np.array_equal(lp.double().cpu().numpy(), a[0])


# ---------------------------------------------------------------- together, streams and graphs

class _Step:
    """One step of a loop that verifies drafted trees: rotate, write, attend, project, score."""

    def __init__(self, torch, cache, seed, ctx=(150, 33, 0), n=(7, 1, 12), heads=4, kvh=2, dim=64, vocab=3001):
        self.torch, self.ctx, self.n, self.heads, self.kvh, self.dim, self.vocab = torch, list(ctx), list(n), heads, kvh, dim, vocab
        self.c = _make_cache(torch, cache, len(ctx), max(ctx) + 64, kvh, 16, dim, seed)
        self.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.rows = int(self.start[-1])
        rng = np.random.default_rng(seed)
        self.masks = sum((_tree_masks(rng, k, False) for k in n), [])
        slot = np.concatenate([np.arange(c, c + k) for c, k in zip(ctx, n)])
        depth = np.concatenate([[c + bin(m).count("1") - 1 for m in self.masks[a:a + k]]
                                for c, k, a in zip(ctx, n, self.start)])
        dev = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()
        self.slot, self.depth, self.stream = dev(slot), dev(depth), dev(np.repeat(np.arange(len(n)), n))
        self.dstart, self.dctx, self.dmask = dev(self.start), dev(ctx), _dev_masks(torch, self.masks)
        self.rope = lib.Rope(48, halves=True, scaling="ntk", factor=2.0)
        self.w = torch.from_numpy((rng.standard_normal((heads * dim, vocab)) / 8).astype(np.float32)).cuda()
        self.qkv = torch.zeros(self.rows, heads + 2 * kvh, dim, device="cuda")
        self.tokens = dev(rng.integers(0, vocab, self.rows))
        self.q, self.out = torch.zeros(self.rows, heads, dim, device="cuda"), torch.zeros(self.rows, heads, dim, device="cuda")
        self.logits = torch.zeros(self.rows, vocab, device="cuda")
        self.lp, self.ent = torch.zeros(self.rows, device="cuda"), torch.zeros(self.rows, device="cuda")
        self.ids = torch.zeros(self.rows, 5, dtype=torch.int32, device="cuda")
        self.top = torch.zeros(self.rows, 5, device="cuda")
        self.ws = torch.zeros(max(16, lib.attn_tree_workspace(self.c, heads, self.rows, max(n), max(ctx) + 64)), dtype=torch.uint8, device="cuda")
        self.ws2 = torch.zeros(max(16, lib.token_logprobs_workspace(self.rows, vocab, 5)), dtype=torch.uint8, device="cuda")
        # the committed context
        for s, k in enumerate(ctx):
            if k:
                x = [torch.from_numpy(rng.standard_normal((k, kvh, dim)).astype(np.float32)).cuda() for _ in range(2)]
                lib.kv_write(self.c, *x, torch.full((k,), s, dtype=torch.int32, device="cuda"), torch.arange(k, dtype=torch.int32, device="cuda"),
                             rope=self.rope)

    def inputs(self, seed):
        g = self.torch.Generator(device="cuda").manual_seed(seed)
        self.qkv.copy_(self.torch.randn(self.qkv.shape, generator=g, device="cuda"))

    def run(self):
        h, k = self.heads, self.kvh
        lib.rope_rows(self.qkv[:, :h], self.depth, self.rope, self.q)
        lib.kv_write(self.c, self.qkv[:, h:h + k], self.qkv[:, h + k:], self.stream, self.slot, rope=self.rope, rope_pos=self.depth)
        lib.attn_tree(self.q, self.c, self.dstart, self.dctx, self.out, max(self.n), max(self.ctx) + 64, row_mask=self.dmask, workspace=self.ws)
        self.torch.mm(self.out.view(self.rows, -1), self.w, out=self.logits)
        lib.token_logprobs(self.logits, self.tokens, self.lp, self.ent, self.ids, self.top, workspace=self.ws2)

    def results(self):
        self.torch.cuda.synchronize()
        return [t.clone() for t in (self.out, self.lp, self.ent, self.ids, self.top)]


@pytest.mark.parametrize("cache", ["i8", "e4m3", "f16", "f32"])
def test_a_whole_step(torch_gpu, cache):
    """All four together against 64 bits, each on what the one before left; then the accepted row is written again at
    its final place and the next step attends it there."""
    torch = torch_gpu
    st = _Step(torch, cache, 21)
    st.inputs(1)
    st.run()
    out, lp, ent, ids, top = st.results()
    f, _ = lib.rope_freqs(48, scaling="ntk", factor=2.0)
    depth = st.depth.cpu().numpy()
    want, mag = _rot(st.qkv[:, :4].double().cpu().numpy(), depth, f, True)
    assert (np.abs(st.q.double().cpu().numpy() - want) <= _rope_tol(mag, f, depth)).all()
    want, _, tol, _, _ = _attn_ref(st.q.cpu().numpy(), st.c, st.start, st.ctx, st.masks, 0.125, st.rows, 4)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    wlp, went, wids, wtop, ltol = _lp_ref(st.logits.cpu().numpy(), st.tokens.cpu().numpy(), 1.0, 5)
    assert np.array_equal(ids.cpu().numpy(), wids) and (np.abs(lp.double().cpu().numpy() - wlp) <= ltol).all()
    assert (np.abs(ent.double().cpu().numpy() - went) <= ltol).all()
    # stream 0 accepts node 3 as its next position
    x = st.qkv[3:4]
    zero, at = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([150], dtype=torch.int32, device="cuda")
    lib.kv_write(st.c, x[:, 4:6], x[:, 6:], zero, at, rope=st.rope)
    st.ctx[0] += 1
    q = st.q[:3].cpu()
    _check_attn(torch, st.c, q, np.array([0, 1, 2, 3], np.int32), st.ctx, None)


def test_steps_on_streams_of_their_own(torch_gpu):
    """Two steps at once on two streams, and one on a stream given by its handle: the results of steps alone."""
    torch = torch_gpu
    a, b = _Step(torch, "i8", 31), _Step(torch, "f16", 32, ctx=(900, 5), n=(3, 30))
    want = []
    for st in (a, b):
        st.inputs(5)
        st.run()
        want.append(st.results())
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(sa):
            a.run()
        with torch.cuda.stream(sb):
            b.run()
    for st, w in zip((a, b), want):
        assert all(torch.equal(x, y) for x, y in zip(st.results(), w))
    a.out.zero_()
    torch.cuda.synchronize()
    lib.attn_tree(a.q, a.c, a.dstart, a.dctx, a.out, max(a.n), max(a.ctx) + 64, row_mask=a.dmask, workspace=a.ws, stream=sa.cuda_stream)
    sa.synchronize()
    assert torch.equal(a.out, want[0][0])
    need = lib.attn_tree_workspace(b.c, 4, b.rows, 30, 964)
    if need:
        with pytest.raises(ValueError, match="workspace"):
            lib.attn_tree(b.q, b.c, b.dstart, b.dctx, b.out, 30, 964, row_mask=b.dmask, stream=sa.cuda_stream)


def test_captured_steps(torch_gpu):
    """Two captured steps with workspaces of their own, replayed with new inputs, eager steps of a third between the
    replays: every replay equals the eager step on its inputs."""
    torch = torch_gpu
    steps = [_Step(torch, "i8", 41, ctx=(2000, 100), n=(5, 9)), _Step(torch, "e4m3", 42)]
    eager = _Step(torch, "f16", 43)
    graphs = []
    s = torch.cuda.Stream()
    for st in steps:
        st.inputs(1)
        with torch.cuda.stream(s):
            st.run()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            st.run()
        graphs.append(g)
    for rep in range(4):
        print(f"replay {rep}", flush=True)
        want = []
        for st in steps:
            st.inputs(50 + rep)
            st.run()
            want.append(st.results())
            st.out.zero_()
            st.lp.zero_()
        for st, g, w in zip(steps, graphs, want):
            eager.inputs(rep)
            eager.run()
            g.replay()
            assert all(torch.equal(x, y) for x, y in zip(st.results(), w))


def test_wrong_tensors_are_refused(torch_gpu):
    """Shapes, types and strides that the binding cannot describe to the call."""
    torch = torch_gpu
    st = _Step(torch, "i8", 51)
    h = st.heads
    with pytest.raises(ValueError, match="row_pos"):
        lib.kv_write(st.c, st.qkv[:, h:h + 2], st.qkv[:, h + 2:], st.stream, st.slot.long())
    with pytest.raises(ValueError, match="contiguous"):
        lib.kv_write(st.c, st.qkv[:, h:h + 4:2], st.qkv[:, h + 2:], st.stream, st.slot)
    with pytest.raises(ValueError, match="row_mask"):
        lib.attn_tree(st.q, st.c, st.dstart, st.dctx, st.out, 12, 300, row_mask=st.dmask[:-1])
    with pytest.raises(ValueError, match="ctx_len"):
        lib.attn_tree(st.q, st.c, st.dstart, st.dctx[:2], st.out, 12, 300)
    with pytest.raises(TypeError):
        lib.rope_rows(st.q.bfloat16(), st.depth, st.rope)
    with pytest.raises(ValueError, match="contiguous"):
        lib.token_logprobs(st.logits.t(), st.tokens, st.lp)
    with pytest.raises(ValueError, match="top"):
        lib.token_logprobs(st.logits, st.tokens, st.lp, top_ids=st.ids)
    with pytest.raises(lib.MossHipError):  # a workspace too small
        lib.attn_tree(st.q[:1], st.c, st.dstart, st.dctx, st.out[:1], 1, 8192, workspace=st.ws[:16])
