"""Attention of drafted rows where its arithmetic can go wrong (GPU), against plain 64-bit forms: small weights beside
large ones, value scales far apart, long sums, scores past 32-bit whole numbers, Inf in queries, fp16 outputs of many rows.

Tolerances come from the arithmetic: a rounding to fp32 is 2^-24 of a value, to fp16 2^-11."""
import math

import numpy as np
import pytest

from mosship import lib
from test_gpu_paged_ops import (U16, U32, _attn_case, _attn_ref, _make_cache, _run_attn, _types)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- fp16 outputs, and the kernel for many rows

@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,kvh,n,ctx", [
    (128, 8, 2, [20, 17], [200, 77]), (128, 8, 2, [20, 17], [1500, 333]),  # 80 and 68 rows a key head
    (128, 4, 1, [40, 1, 33], [131, 0, 90]), (128, 4, 1, [40, 1, 33], [1111, 0, 700]),  # 160 and 132
    (128, 8, 1, [64, 33], [45, 130]), (128, 8, 1, [64, 33], [900, 1301]),  # 512 and 264: two groups of row tiles
    (64, 4, 2, [64, 50, 3], [70, 260, 1000]), (64, 8, 1, [30, 19], [517, 203])])
@pytest.mark.parametrize("qdt,odt", [("f32", "f32"), ("f32", "f16"), ("f16", "f32"), ("f16", "f16")])
def test_attn_many_rows(torch_gpu, cache, dim, heads, kvh, n, ctx, qdt, odt):
    """More than 64 rows a key head, uncut and cut, each type of query and output.  A 16-bit output is the 32-bit result
    rounded once: 2^-11 of it (2^-25 where that is under fp16's normal range), and nothing more."""
    torch = torch_gpu
    print(f"attn many rows {cache} {dim} {heads}/{kvh} {n} {ctx} {qdt} {odt}", flush=True)
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, 48, ctx, n, False, sum(n) + sum(ctx), qdt=qdt)
    got, lse = _run_attn(torch, c, q, start, ctx, masks, max(n), max(a + b for a, b in zip(ctx, n)), odt)
    want, wl, tol, ltol, _ = _attn_ref(q.float().numpy(), c, start, ctx, masks, dim ** -0.5, rows, heads)
    if odt == "f16":
        tol = tol + np.abs(want) * U16 + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    assert (np.abs(lse - wl) <= ltol).all()


# ---------------------------------------------------------------- weights and value scales

def _put(c, s, pos, k=None, v=None, ks=None, vs=None):
    """Elements (as the pools hold them) and scales of positions `pos` of stream s, every head."""
    import torch
    page = c.tensors[0].shape[2]
    for p in pos:
        at = (int(c.tensors[2][s, p // page]), slice(None), p % page)
        for pool, scale, x, d in ((c.tensors[0], c.tensors[3], k, ks), (c.tensors[1], c.tensors[4], v, vs)):
            if x is not None:
                x = torch.as_tensor(x).expand(pool[at].shape)
                pool[at] = x.to(pool.dtype).to(pool.device)
            if d is not None and scale is not None:
                scale[at] = d


def _raw(c, which, s, n):
    """The first n positions of stream s in 64 bits: elements [heads][n][dim] and their scales [heads][n]."""
    import torch
    pool, scale = c.tensors[which], c.tensors[3 + which]
    page = pool.shape[2]
    pages = c.tensors[2][s, :(n + page - 1) // page].long()
    x = pool.view(torch.int8)[pages].view(pool.dtype).double().transpose(0, 1).flatten(1, 2)[:, :n].cpu().numpy()
    if scale is None:
        return x, np.ones(x.shape[:2])
    return x, scale[pages].double().transpose(0, 1).flatten(1, 2)[:, :n].cpu().numpy()


def _fine_ref(q, c, start, ctx, mask, scale, heads, exact_products=False):
    """out and lse in 64 bits, and tolerances key by key.

    A score is off by 24 roundings of scale * sum |q k| (none where the products are exact), a weight by 4 roundings of the
    scores it is the difference of, exp2's and the weight's own 2^-22 (with the value scale's product 2^-21); sums chain
    keys / 16 + 64 roundings.  Below its 22 bits a weight (times its value scale) has a step: it is off by up to 2^-35 of the
    row's largest."""
    rows = len(q)
    out, tol = np.zeros((rows, heads, c.head_dim)), np.zeros((rows, heads, c.head_dim))
    lse, ltol = np.full((rows, heads), -np.inf), np.zeros((rows, heads))
    for s in range(len(ctx)):
        a, b, n = int(start[s]), int(start[s + 1]), int(ctx[s] + start[s + 1] - start[s])
        if b == a:
            continue
        (k, ks), (v, vs) = _raw(c, 0, s, n), _raw(c, 1, s, n)
        for r in range(a, b):
            m = (2 << (r - a)) - 1 if mask is None else int(mask[r])
            see = np.array([j < ctx[s] or (m >> (j - int(ctx[s]))) & 1 for j in range(n)], bool)
            if not see.any():
                continue
            for h in range(heads):
                g = h * c.kv_heads // heads
                kk, u, d, qq = k[g][see] * ks[g][see][:, None], v[g][see], vs[g][see], q[r, h].astype(np.float64)
                x = scale * (kk @ qq)
                e = np.exp(x - x.max())
                p = e / e.sum()
                w = p * np.abs(d)
                err = 4 * U32 * (np.abs(x) + np.abs(x.max())) + 2.0 ** -21
                if not exact_products:
                    err = err + 24 * U32 * abs(scale) * (np.abs(kk) @ np.abs(qq))
                chain = (n / 16 + 64) * U32
                norm = (p * err).sum() + chain
                out[r, h] = (p * d) @ u
                tol[r, h] = ((err + norm + chain) * w) @ np.abs(u) + 2.0 ** -35 * w.max() * np.abs(u).sum(0) + 2 * U32 * np.abs(out[r, h])
                lse[r, h] = x.max() + np.log(e.sum())
                ltol[r, h] = norm + 4 * U32 * (np.abs(lse[r, h]) + np.abs(x.max()))
    return out, lse, tol, ltol


def _check_fine(torch, c, q, start, ctx, masks, heads, exact_products=False, scale=None, **kw):
    n = np.diff(start)
    got, lse = _run_attn(torch, c, q, start, ctx, masks, int(n.max()), int((np.array(ctx) + n).max()), scale=scale, **kw)
    want, wl, tol, ltol = _fine_ref(q.float().numpy(), c, start, ctx, masks, c.head_dim ** -0.5 if scale is None else scale, heads,
                                    exact_products)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])
    fin = np.isfinite(wl)
    assert np.array_equal(fin, np.isfinite(lse)) and (np.abs(lse[fin] - wl[fin]) <= ltol[fin]).all()
    return got, lse


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,kvh,n", [(64, 4, 2, 6), (128, 8, 2, 6), (64, 4, 1, 40), (128, 8, 2, 20)])
def test_attn_finite_scales_behind_the_mask(torch_gpu, cache, dim, heads, kvh, n):
    """A drafted key's value scale, however large, changes not a bit of the rows that do not see it: roots beside it without
    a context, and rows with one.  A row that does see it is as good as ever."""
    torch = torch_gpu
    print(f"attn scales behind the mask {cache} {dim} {heads}/{kvh} {n}", flush=True)
    ctx = [37, 0]
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, 16, ctx, [n, n], False, 78)
    masks = [m & ~(1 << 2) for m in masks]
    masks = [m | (1 << 2) if r in (1, n + 3) else m for r, m in enumerate(masks)]
    hit = np.isin(np.arange(rows), (1, n + 3))
    clean, lse = _check_fine(torch, c, q, start, ctx, masks, heads)
    for big in (1e4, 1e6, 1e8, 1e30):
        for s in (0, 1):
            _put(c, s, [ctx[s] + 2], vs=big)
        got, l = _check_fine(torch, c, q, start, ctx, masks, heads)
        assert np.array_equal(got[~hit], clean[~hit]) and np.array_equal(l, lse), big


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,kvh,n", [(64, 2, 1, 1), (64, 4, 1, 40), (128, 8, 2, 20)])
@pytest.mark.parametrize("big", [2.0 ** 6, 1e4, 1e12, 1e30])
def test_attn_scale_of_a_key_without_weight(torch_gpu, cache, dim, heads, kvh, n, big):
    """One value scale of the context far above the others, on a key with next to no weight."""
    torch = torch_gpu
    print(f"attn scale without weight {cache} {dim} {heads}/{kvh} {n} {big}", flush=True)
    ctx = [541]
    c, start, rows, masks, q = _attn_case(torch, cache, dim, heads, kvh, 64, ctx, [n], False, 79)
    q[..., 0] = 8.0
    k = torch.zeros(dim)
    k[0] = -64.0
    _put(c, 0, [100], k=k, ks=2.0 if dim == 128 else 1.5, vs=big)  # a score of -90 or -96
    _check_fine(torch, c, q, start, ctx, masks, heads)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("scale", [1e-33, 1e-25, 1e25, 1e34])
@pytest.mark.parametrize("n", [1, 40])
def test_attn_scales_at_the_ends(torch_gpu, cache, n, scale):
    """All value scales tiny or huge: the bits are kept."""
    torch = torch_gpu
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 4, 1, 64, [300], [n], False, 80)
    c.tensors[4].mul_(scale / float(c.tensors[4].mean()))
    _check_fine(torch, c, q, start, [300], masks, 4)


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("ctx,heads,n", [(541, 2, 1), (541, 2, 20), (541, 2, 40), (4096, 2, 1), (4096, 3, 64)])
@pytest.mark.parametrize("gap", [8.0, 11.0, 14.0, 17.0])
def test_attn_sink(torch_gpu, cache, ctx, heads, n, gap):
    """A first key that takes nearly all the weight and has values of zero: the output is made of the small weights, e^-gap
    of the largest each, with values of one sign.  Queries with one element, so that the scores' products are exact."""
    torch = torch_gpu
    print(f"attn sink {cache} ctx {ctx} rows {n * heads} gap {gap}", flush=True)
    rng = np.random.default_rng(ctx + n)
    total = ctx + n
    c = _make_cache(torch, cache, 1, total, 1, 64, 64)
    k = rng.integers(-100, 100, (total, 64)).astype(np.float32)
    k[:, 0] = rng.integers(0, 5, total)
    k[0, 0] = 112
    v = rng.integers(64, 128, (total, 64)).astype(np.float32)
    if cache == "e4m3":
        k, v = torch.from_numpy(k).to(torch.float8_e4m3fn).float().numpy(), torch.from_numpy(v).to(torch.float8_e4m3fn).float().numpy()
    v[0] = 0
    table = c.tensors[2].cpu().numpy()[0]
    at = (torch.from_numpy(table[np.arange(total) // 64].astype(np.int64)), 0, torch.arange(total) % 64)
    for pool, x in ((c.tensors[0], k), (c.tensors[1], v)):
        host = pool.float().cpu()
        host[at] = torch.from_numpy(x)
        pool.copy_(host.to(pool.dtype))
    if cache in ("i8", "e4m3"):
        c.tensors[3].fill_(2.0 ** -4)
        c.tensors[4].fill_(2.0 ** -6)
    q = torch.zeros(n, heads, 64)
    q[..., 0] = 2.0 ** -8
    scale = gap / (112 * 2.0 ** -8 * (2.0 ** -4 if cache in ("i8", "e4m3") else 1))
    start = np.array([0, n], np.int32)
    _check_fine(torch, c, q, start, [ctx], None, heads, exact_products=True, scale=float(np.float32(scale)))


@pytest.mark.parametrize("n", [1, 30])
def test_attn_fp32_values_near_the_largest(torch_gpu, n):
    """Values of an fp32 cache within a hundredth of the type's largest: no weight is more than 1, so sums are in range."""
    torch = torch_gpu
    c, start, rows, masks, q = _attn_case(torch, "f32", 64, 2, 2, 16, [100], [n], False, 101)
    c.tensors[1].clamp_(-3, 3).mul_(1e36)
    _check_fine(torch, c, q, start, [100], masks, 2)


# ---------------------------------------------------------------- long sums

@pytest.mark.parametrize("cache,streams,heads,kvh,most", [("i8", 17, 16, 8, 40), ("f16", 17, 16, 8, 40), ("e4m3", 97, 8, 8, 1), ("f16", 97, 8, 8, 1), ("f32", 97, 8, 8, 1)])
def test_attn_long_sums(torch_gpu, cache, streams, heads, kvh, most):
    """131072 equal weights under so many streams and heads that nothing is cut to fill the chip: neither sum drifts.  lse is
    the score plus log 131073 within 72 roundings of the sum, and those of the result's own size.  The values' sum is a chain
    of up to 1024 products' results, each cut by up to 2^-23 of the sum so far (2^-24 of the whole on average), and 64 roundings."""
    torch = torch_gpu
    print(f"attn long sums {cache} {streams} {heads}/{kvh}", flush=True)
    ctx, page = 131072, 1024
    k = torch.zeros(2, kvh, page, 64, device="cuda")
    k[..., 0] = 1.0
    v = torch.ones(2, kvh, page, 64, device="cuda")
    ones = torch.ones(2, kvh, page, device="cuda") if cache in ("i8", "e4m3") else None
    dt = _types(torch)[cache]
    table = torch.zeros(streams, ctx // page + 1, dtype=torch.int32, device="cuda")  # every page is the same
    c = lib.KVCache(k.to(dt), v.to(dt), table, ones, ones)
    n = [most] + [1] * (streams - 1)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    rows = int(start[-1])
    q = torch.zeros(rows, heads, 64)
    q[..., 0] = 8 * torch.rand(rows, heads, generator=torch.Generator().manual_seed(1)) - 4
    masks = [1 << (r if r < most else 0) for r in range(rows)]  # itself
    got, lse = _run_attn(torch, c, q, start, [ctx] * streams, masks, most, ctx + most)
    want = 0.125 * q[..., 0].double().numpy() + math.log(ctx + 1)
    assert (np.abs(lse - want) <= 72 * U32 + 4 * U32 * (np.abs(want) + 0.5)).all(), np.max(np.abs(lse - want)) / U32
    assert (np.abs(got - 1) <= (1024 + 64 + 72) * U32).all(), np.max(np.abs(got - 1)) / U32


# ---------------------------------------------------------------- what is not finite, and what is far out

@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("qdt", ["f32", "f16"])
@pytest.mark.parametrize("n", [1, 2, 40])
def test_attn_inf_queries_over_few_keys(torch_gpu, cache, qdt, n):
    """An Inf or NaN in a query makes its head NaN also where one key is all it sees (its products may then all be -Inf), and
    one that sees nothing is 0 all the same."""
    torch = torch_gpu
    print(f"attn inf queries {cache} {qdt} {n}", flush=True)
    ctx = [0, 1, 2, 0]
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 8, 2, 16, ctx, [n] * 4, False, 90 + n, qdt=qdt)
    masks = [1 << (r % n) for r in range(rows)]
    for r in range(3 * n, rows):
        masks[r] = 0
    clean, cl = _run_attn(torch, c, q, start, ctx, masks, n, n + 2)
    odd, bad = q.clone(), np.zeros((rows, 8), bool)
    for i in range(8 * rows):
        r, h = divmod(i, 8)
        if i % 3:
            odd[r, h, (7 * i) % 64] = (math.inf, -math.inf, math.nan)[i // 3 % 3]
            bad[r, h] = r < 3 * n
    got, lse = _run_attn(torch, c, odd, start, ctx, masks, n, n + 2)
    assert np.isnan(got[bad]).all() and np.isnan(lse[bad]).all()
    assert np.array_equal(got[~bad], clean[~bad]) and np.array_equal(lse[~bad], cl[~bad])
    assert (got[3 * n:] == 0).all() and (lse[3 * n:] == -np.inf).all()


@pytest.mark.parametrize("cache", ["f16", "i8", "e4m3", "f32"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n", [1, 40])
def test_attn_scores_past_whole_numbers(torch_gpu, cache, sign, n):
    """Scores of 1e10, whose last bits are worth hundreds: the keys of the largest take all the weight, two equal ones
    half each, and rows with ordinary scores beside them do not change by a bit."""
    torch = torch_gpu
    print(f"attn far scores {cache} {sign} {n}", flush=True)
    ctx = [70]
    c, start, rows, masks, q = _attn_case(torch, cache, 64, 4, 1, 16, ctx, [n], False, 100)
    step, scale = {"f16": (2000.0, 1.0), "f32": (2000.0, 1.0), "i8": (2.0, 60000.0), "e4m3": (16.0, 300.0)}[cache]
    for p in range(ctx[0] + n):  # of 17 sizes, each several times
        _put(c, 0, [p], k=(1.0 + p % 17) * step, ks=scale)
    q *= 1e-5
    clean, cl = _run_attn(torch, c, q, start, ctx, masks, n, ctx[0] + n)
    far = q.clone()
    far[:, 1] = sign * 60000.0
    far[:, 2] = sign * 30000.0
    got, lse = _run_attn(torch, c, far, start, ctx, masks, n, ctx[0] + n)
    assert np.array_equal(got[:, [0, 3]], clean[:, [0, 3]]) and np.array_equal(lse[:, [0, 3]], cl[:, [0, 3]])
    (kr, ks), (v, vs) = _raw(c, 0, 0, ctx[0] + n), _raw(c, 1, 0, ctx[0] + n)
    key, val = kr[0, :, 0] * ks[0], v[0] * vs[0][:, None]
    for r in range(n):
        see = np.array([j < ctx[0] or (masks[r] >> (j - ctx[0])) & 1 for j in range(ctx[0] + n)], bool)
        for h in (1, 2):
            score = 0.125 * 64 * float(far[r, h, 0]) * key
            assert abs(score).max() > 2.0 ** 33 or h == 2
            top = see & (score == score[see].max())
            want = val[top].mean(0)
            assert (np.abs(got[r, h] - want) <= 64 * U32 * np.abs(val[top]).mean(0) + 1e-30).all(), (r, h, got[r, h][:3], want[:3])
            assert abs(lse[r, h] - score[top][0]) <= 16 * U32 * abs(score[top][0])
