"""The operators of a serving loop against plain sequential forms in 64 bits (GPU): verification of drafted tokens, pages that
streams share, accepted rows moved to their positions, adapters beside a projection, and a run of all of them together.

Decisions and moved bytes have to be equal.  Where a random number is compared with a probability, the call's is off by up to
2^-18 (acceptance) or some 2^-40 (draws); each test makes sure that no number of its own lies that near to a border."""
import numpy as np
import pytest

import serving_oracle as so
from mosship import lib

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -11


def _cu(torch, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


# ---------------------------------------------------------------- verification

def _draft(rng, n_list, vocab, chain, near=0.7, banned=0.0, peak=9.0, gap=0, spare=0):
    """Rows of several streams: logits, tokens near their peaks, masks, starts.  gap: rows of no stream before each."""
    x, tok, mask, start = [], [], [], [0]
    for n in n_list:
        z = 2.0 * rng.standard_normal((n, vocab))
        top = rng.integers(0, vocab, n)
        z[np.arange(n), top] += peak * rng.random(n)
        if banned:
            z[rng.random((n, vocab)) < banned] = -np.inf
            z[np.arange(n), top] = 7.0
        parent = [max(i - 1, 0) if chain else max(0, i - 1 - int(rng.integers(0, 4))) for i in range(n)]
        m = []
        for i in range(n):
            m.append((m[parent[i]] if i else 0) | 1 << i)
        tok += [int(top[parent[i]]) if rng.random() < near else int(rng.integers(0, vocab)) for i in range(n)]
        x.append(z)
        mask += m
        start.append(start[-1] + n)
    x = np.concatenate([*x, np.full((spare, vocab), np.nan)]) if x else np.zeros((spare, vocab))
    return (x.astype(np.float32), np.array(tok + [0] * spare, np.int32), np.array(mask + [1] * spare, np.uint64), np.array(start, np.int32))


def _verify(torch, x, tok, start, max_rows, u=None, y=None, mask=None, dtype=None, pad=0, **kw):
    """The call's answer, with sentinels in path before it."""
    rows, vocab = x.shape
    dtype = dtype or torch.float32

    def dev(z):
        t = torch.full((rows, vocab + pad), float("nan"), dtype=dtype, device="cuda")
        t[:, :vocab] = _cu(torch, z, dtype)
        return t[:, :vocab]
    streams = len(start) - 1
    acc, nxt = (torch.full((streams,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    path = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    lib.verify_tokens(dev(x), _cu(torch, tok), _cu(torch, start), acc, path, nxt, max_rows, uniforms=None if u is None else _cu(torch, u),
                      draft_logits=None if y is None else dev(y), row_mask=None if mask is None else _cu(torch, mask.view(np.int64)), **kw)
    return acc.cpu().numpy(), path.cpu().numpy(), nxt.cpu().numpy()


def _held(torch, z, dtype):
    return torch.from_numpy(z).to(dtype).double().numpy()


def _check_verify(torch, x, tok, start, max_rows, u=None, y=None, mask=None, dtype=None, pad=0, inv_temperature=1.0,
                  draft_inv_temperature=None, greedy=False):
    dtype = dtype or torch.float32
    got = _verify(torch, x, tok, start, max_rows, u, y, mask, dtype, pad, inv_temperature=inv_temperature,
                  draft_inv_temperature=draft_inv_temperature, greedy=greedy)
    *want, near = so.verify(_held(torch, x, dtype), tok, start, u, max_rows, None if y is None else _held(torch, y, dtype), mask, inv_temperature,
                            inv_temperature if draft_inv_temperature is None else draft_inv_temperature, greedy, path=np.full(len(tok), -7))
    assert near > 1, near
    for name, g, w in zip(("accepted", "path", "next"), got, want):
        assert np.array_equal(g, w), (name, g, w)
    return got


@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("draft", [True, False])
def test_verify_long_paths(torch_gpu, chain, draft):
    """Likely tokens: many are accepted."""
    torch = torch_gpu
    if draft and not chain:
        pytest.skip("draft_logits are for chains")
    rng = np.random.default_rng(77)
    x, tok, mask, start = _draft(rng, [64, 30, 3, 17, 64], 4000, chain, near=0.95, peak=60.0)
    y = (x + 0.3 * rng.standard_normal(x.shape)).astype(np.float32) if draft else None
    acc, _, _ = _check_verify(torch, x, tok, start, 64, rng.random(len(tok)), y=y, mask=None if draft else mask)
    assert acc.max() >= 2


VOCABS = [1, 2, 31, 1000, 1024, 1025, 16384, 16389]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_verify_picked_outright(torch_gpu, vocab, chain, dtype):
    torch = torch_gpu
    print(f"verify outright {vocab} {chain} {dtype}", flush=True)
    rng = np.random.default_rng(vocab * 2 + chain)
    n = [1, 5, 27, 0, 64, 2, 12]
    x, tok, mask, start = _draft(rng, n, vocab, chain, banned=0.3 if vocab > 100 else 0.0, spare=2)
    u = rng.random(len(tok))
    got = _check_verify(torch, x, tok, start, 64, u, mask=mask, dtype=getattr(torch, dtype), pad=3, inv_temperature=1.0 / 0.8)
    if chain:
        again = _verify(torch, x, tok, start, 64, u, dtype=getattr(torch, dtype), inv_temperature=1.0 / 0.8)
        assert all(np.array_equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_verify_drafted_with_probabilities(torch_gpu, vocab, dtype):
    torch = torch_gpu
    print(f"verify drafted {vocab} {dtype}", flush=True)
    rng = np.random.default_rng(vocab * 3 + 1)
    x, tok, _, start = _draft(rng, [6, 1, 9, 0, 4, 64, 7], vocab, True, near=0.8, banned=0.2 if vocab > 100 else 0.0, spare=1)
    y = (x + 0.8 * rng.standard_normal(x.shape)).astype(np.float32)
    y[start[1:][start[1:] > start[:-1]] - 1] = np.nan  # the rows behind which nothing was drafted
    u = rng.random(len(tok)) * 0.98
    _check_verify(torch, x, tok, start, 64, u, y=y, dtype=getattr(torch, dtype), pad=1, inv_temperature=1.25, draft_inv_temperature=0.9)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_wide(torch_gpu, draft):
    """Rows of many chunks; one and several streams."""
    torch = torch_gpu
    for streams, vocab in ((1, 130001), (9, 130001), (2, 400003)):
        print(f"verify wide {streams} {vocab}", flush=True)
        rng = np.random.default_rng(streams + vocab)
        x, tok, mask, start = _draft(rng, [5 - s % 3 for s in range(streams)], vocab, draft, near=0.9, peak=16.0)
        y = (x + 0.5 * rng.standard_normal(x.shape)).astype(np.float32) if draft else None
        _check_verify(torch, x, tok, start, 5, rng.random(len(tok)), y=y, mask=None if draft else mask, dtype=torch.float16)


@pytest.mark.parametrize("vocab", [1, 3, 1024, 5000, 130001])
def test_verify_greedy(torch_gpu, vocab):
    """Ties go to the lowest index; NaN is nobody's likeliest token, +inf is."""
    torch = torch_gpu
    rng = np.random.default_rng(vocab)
    x, _, mask, start = _draft(rng, [1, 6, 30, 64], vocab, False)
    x = np.round(x * 2) / 2  # many equal values
    x[3, rng.integers(0, vocab, 3)] = np.nan
    x[9, vocab // 2:] = np.inf
    x[12] = -np.inf
    x[13] = np.nan
    best = np.argmax(np.where(np.isnan(x), -np.inf, x), 1).astype(np.int32)
    tok = np.zeros(len(x), np.int32)
    for s in range(4):
        for i in range(start[s], start[s + 1]):
            up = so._parent(i - start[s], mask[start[s]:])
            tok[i] = best[start[s] + max(up, 0)] if rng.random() < 0.8 else rng.integers(0, vocab)
    _check_verify(torch, x, tok, start, 64, mask=mask, greedy=True)
    _check_verify(torch, x, tok, start, 64, greedy=True, dtype=torch.float16)


def test_verify_rows_that_are_no_distribution(torch_gpu):
    torch = torch_gpu
    vocab = 1500
    rng = np.random.default_rng(5)
    x, tok, _, start = _draft(rng, [4] * 8, vocab, True, near=1.0, peak=40.0)
    y = (x + 0.1 * rng.standard_normal(x.shape)).astype(np.float32)
    u = np.full(len(tok), 0.3)
    x[0] = -np.inf
    x[4 + 1, 1400] = np.nan
    x[8 + 2, 3] = np.inf
    x[12 + 3] = np.nan
    y[16 + 1] = -np.inf  # the draft's: its child is rejected, p is drawn from
    y[20 + 2, 7] = np.nan
    y[24, 1499] = np.inf
    tok[29], tok[30] = -1, vocab
    print("no distribution, drafted", flush=True)
    acc, _, nxt = _check_verify(torch, x, tok, start, 4, u, y=y)
    assert nxt[0] == -1 and acc[1] == 1 and nxt[1] == -1 and acc[4] == 1 and nxt[4] >= 0
    print("no distribution, outright", flush=True)
    _check_verify(torch, x, tok, start, 4, u)


def test_verify_siblings(torch_gpu):
    """Equal tokens among siblings, children with no probability, certain ones, tokens outside the vocabulary."""
    torch = torch_gpu
    vocab, n = 1030, 9
    rng = np.random.default_rng(11)
    x = rng.standard_normal((n, vocab)).astype(np.float32)
    x[:, 1029] = -np.inf
    mask = np.array([1] + [1 | 1 << i for i in range(1, n)], np.uint64)  # all children of the root
    start = np.array([0, n], np.int32)
    for case, toks in enumerate(([5, 5, 5, 5, 5, 5, 5, 5], [1029] * 8, [-1, vocab, 1 << 30, 7, 7, 8, 9, 1029], list(range(8)))):
        tok = np.array([0] + toks, np.int32)
        for u in (0.0, 0.5, 0.999, 1.0):
            print("siblings", case, u, flush=True)
            _check_verify(torch, x, tok, start, n, np.full(n, u), mask=mask)
    # nearly all of the probability at one child that a number of 1 rejects: what is left is drawn from, to the last bit
    x[:] = -700.0
    x[:, 17], x[:, 1029] = 50.0, -np.inf
    _check_verify(torch, x, np.array([0, 17] + [3] * 7, np.int32), start, n, np.array([0.5] + [1.0] * 8), mask=mask)
    # nothing but that child: p itself
    x[:] = -np.inf
    x[:, 17] = 1.0
    _check_verify(torch, x, np.array([0] + [17] * 8, np.int32), start, n, np.full(n, 1.0), mask=mask)


def test_verify_odd_masks(torch_gpu):
    """Nodes whose masks lack their own bit, name later nodes, or have no ancestor are not reached."""
    torch = torch_gpu
    rng = np.random.default_rng(2)
    x, tok, mask, start = _draft(rng, [40, 64], 300, False, near=1.0, peak=30.0)
    mask[3] = 0
    mask[5] = 1 << 5
    mask[7] = np.uint64(mask[7]) & ~np.uint64(1 << 7)
    mask[20:60] = rng.integers(0, 1 << 63, 40, dtype=np.uint64)
    mask[60] = np.uint64(2 ** 64 - 1)
    _check_verify(torch, x, tok, start, 64, rng.random(104), mask=mask)


def test_verify_numbers_outside_their_range(torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(4)
    x, tok, _, start = _draft(rng, [5] * 6, 700, True, near=1.0)
    for bad in (-3.0, 1.0, 9.0, np.inf, -np.inf, np.nan, 0.0):
        u = rng.random(30)
        u[[0, 7, 10, 11, 19, 20]] = bad
        _check_verify(torch, x, tok, start, 5, u)
        _check_verify(torch, x, tok, start, 5, u, y=(x + rng.standard_normal(x.shape)).astype(np.float32))


def test_verify_row_ranges(torch_gpu):
    """Gaps between streams, ranges that are none, more rows than max_rows: nothing else is written."""
    torch = torch_gpu
    rng = np.random.default_rng(6)
    x, tok, _, _ = _draft(rng, [40], 900, True, near=0.9, peak=14.0)
    u = rng.random(40)
    y = (x + 0.3 * rng.standard_normal(x.shape)).astype(np.float32)
    for start in ([0, 4, 11, 40], [3, 3, 9, 41], [-1, 5, 2, 8], [40, 40, 40, 40], [0, 40, 40, 40]):
        for draft in (None, y):
            _check_verify(torch, x, tok, np.array(start, np.int32), 7, u, y=draft)


def test_verify_no_rows(torch_gpu):
    torch = torch_gpu
    acc, path, nxt = _verify(torch, np.zeros((0, 50), np.float32), np.zeros(0, np.int32), np.zeros(4, np.int32), 5, np.zeros(0))
    assert (acc == 0).all() and (nxt == -1).all() and len(path) == 0


def test_verify_equal_distributions(torch_gpu):
    """A draft that is the target is always accepted."""
    torch = torch_gpu
    rng = np.random.default_rng(9)
    x, tok, _, start = _draft(rng, [8, 8], 20000, True, near=0.5)
    acc, _, _ = _check_verify(torch, x, tok, start, 8, rng.random(16) * 0.999, y=x)
    assert (acc == 7).all()


def test_verify_keeps_the_distribution(torch_gpu):
    """Over many numbers the token that follows the root, accepted or drawn, comes as often as p says, for chains and trees: a
    count of n draws is within 5 standard deviations, sqrt(n p (1 - p)), of n p."""
    torch = torch_gpu
    rng = np.random.default_rng(21)
    vocab, draws = 6, 20000
    z, zq = rng.standard_normal(vocab).astype(np.float32), rng.standard_normal(vocab).astype(np.float32)
    p, q = so.softmax(z, 1.0), so.softmax(zq, 1.0)
    for kids in (1, 2, 3):
        n = kids + 1
        x = np.repeat(z[None], draws * n, 0)
        start = (np.arange(draws + 1) * n).astype(np.int32)
        u = rng.random(draws * n)
        if kids == 1:
            tok = rng.choice(vocab, draws * n, p=q).astype(np.int32)
            acc, _, nxt = _verify(torch, x, tok, start, n, u, y=np.repeat(zq[None], draws * n, 0))
        else:
            tok = np.tile(np.array([0, 4, 1, 5][:n], np.int32), draws)
            mask = np.tile(np.array([1] + [1 | 1 << i for i in range(1, n)], np.uint64), draws)
            acc, path, nxt = _verify(torch, x, tok, start, n, u, mask=mask)
        first = nxt.copy()
        took = acc > 0
        if kids == 1:
            first[took] = tok[start[:-1][took] + 1]
        else:
            first[took] = tok[start[:-1][took] + path[start[:-1][took] + 1]]
        count = np.bincount(first, minlength=vocab)
        assert (np.abs(count - draws * p) <= 5 * np.sqrt(draws * p * (1 - p))).all(), (kids, count, draws * p)


def test_verify_captured_and_streams(torch_gpu):
    """Replays of a captured call see the inputs of their time; a call on another stream has its own workspace."""
    torch = torch_gpu
    rng = np.random.default_rng(14)
    x, tok, _, start = _draft(rng, [6, 3, 5], 9000, True)
    y = (x + 0.5 * rng.standard_normal(x.shape)).astype(np.float32)
    dx, dy, dt, ds = (_cu(torch, a) for a in (x, y, tok, start))
    du = torch.empty(14, dtype=torch.float64, device="cuda")
    out = [torch.empty(k, dtype=torch.int32, device="cuda") for k in (3, 14, 3)]
    ws = torch.full((lib.verify_tokens_workspace(3, 6, 9000, True),), 255, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    du.fill_(0.5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        lib.verify_tokens(dx, dt, ds, out[0], out[1], out[2], 6, uniforms=du, draft_logits=dy, workspace=ws)
    for _ in range(4):
        u = rng.random(14)
        du.copy_(torch.from_numpy(u))
        out[1].fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        *want, near = so.verify(x, tok, start, u, 6, y, path=np.full(14, -7))
        assert near > 1
        assert all(np.array_equal(o.cpu().numpy(), w) for o, w in zip(out, want))
        eager = _verify(torch, x, tok, start, 6, u, y=y)
        assert all(np.array_equal(e, w) for e, w in zip(eager, want))
    other = [torch.empty_like(o) for o in out]
    ws2 = torch.empty_like(ws)
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s2):
        lib.verify_tokens(dx, dt, ds, *other, 6, uniforms=du, draft_logits=dy, workspace=ws2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(other[0], out[0]) and torch.equal(other[2], out[2])
    with pytest.raises(ValueError):
        lib.verify_tokens(dx, dt, ds, *other, 6, uniforms=du, draft_logits=dy, stream=s2.cuda_stream)


# ---------------------------------------------------------------- pages

CACHES = ["f32", "f16", "i8", "e4m3"]


def _pools(torch, rng, cache, layers, n_pages, heads, page, dim):
    kinds = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
    out = {}
    for name in "kv":
        # any bits at all: they are moved as they are
        raw = torch.from_numpy(rng.integers(0, 256, (layers, n_pages, heads, page, dim * {"f32": 4, "f16": 2}.get(cache, 1)), dtype=np.uint8))
        out[name] = raw.cuda().view(kinds[cache])
        if cache in ("i8", "e4m3"):
            out[name + "s"] = torch.from_numpy(rng.integers(0, 256, (layers, n_pages, heads, page * 4), dtype=np.uint8)).cuda().view(torch.float32)
    return out


def _layers(torch, pools, table):
    return lib.KVLayers([lib.KVCache(pools["k"][i], pools["v"][i], table, *(pools[n][i] if n in pools else None for n in ("ks", "vs")))
                         for i in range(pools["k"].shape[0])])


def _bytes(pools):
    return {n: t.cpu().view(__import__("torch").uint8).numpy() for n, t in pools.items()}


def _moved(before, moves):
    """Pools as bytes after `moves` of ((page, slot) to (page, slot)), all from what was there before."""
    out = {n: a.copy() for n, a in before.items()}
    for (p, i), (q, j) in moves:
        for n, a in before.items():
            w = 4 if n in ("ks", "vs") else None
            if w:
                out[n][:, q, :, 4 * j:4 * j + 4] = a[:, p, :, 4 * i:4 * i + 4]
            else:
                out[n][:, q, :, j] = a[:, p, :, i]
    return out


def _same(a, b):
    return all(np.array_equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("streams,stride,n_pages", [(1, 1, 1), (4, 5, 30), (64, 10, 300), (1024, 1, 999), (300, 40, 5000), (700, 50, 2000),
                                                    (1024, 65, 100)])
def test_fork(torch_gpu, streams, stride, n_pages):
    """Reorderings, cuts, ends and streams that share, in tables that also hold what names no page."""
    torch = torch_gpu
    print(f"fork {streams} {stride} {n_pages}", flush=True)
    rng = np.random.default_rng(streams + stride)
    table = rng.integers(-3, n_pages + 3, (streams, stride)).astype(np.int32)
    refs = np.bincount(table[(table >= 0) & (table < n_pages)], minlength=n_pages).astype(np.int32) + (rng.random(n_pages) < 0.1)
    refs = refs.astype(np.int32)
    dt, dr = _cu(torch, table), _cu(torch, refs)
    pages = lib.KVPages(dt, dr, 16)
    for step in range(3):
        parent = rng.integers(-2, streams + 2, streams).astype(np.int32)
        length = rng.integers(-20, stride * 16 + 40, streams).astype(np.int32) if step else None
        lib.kv_fork(pages, _cu(torch, parent), None if length is None else _cu(torch, length))
        table, refs = so.fork(table, refs, parent, length, 16)
        assert np.array_equal(dt.cpu().numpy(), table), step
        assert np.array_equal(dr.cpu().numpy(), refs), step


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("streams,stride,n_pages,page,heads,dim,layers,max_rows", [
    (1, 3, 4, 16, 1, 64, 1, 1), (6, 6, 24, 16, 3, 64, 2, 5), (16, 9, 60, 48, 2, 128, 3, 64), (9, 12, 200, 16, 1, 128, 1, 100)])
def test_fork_and_reserve(torch_gpu, cache, streams, stride, n_pages, page, heads, dim, layers, max_rows):
    """A random life: streams grow, share, split, run short of pages and end."""
    torch = torch_gpu
    print(f"reserve {cache} {streams} {stride} {n_pages} {page}", flush=True)
    rng = np.random.default_rng(n_pages + max_rows)
    pools = _pools(torch, rng, cache, layers, n_pages, heads, page, dim)
    table, refs = np.full((streams, stride), -1, np.int32), np.zeros(n_pages, np.int32)
    refs[rng.integers(0, n_pages)] = 1  # held by the caller
    dt, dr, ok = _cu(torch, table), _cu(torch, refs), torch.full((streams,), -7, dtype=torch.int32, device="cuda")
    pages, ls = lib.KVPages(dt, dr, page), _layers(torch, pools, dt)
    ctx, short, copied = np.zeros(streams, np.int64), 0, 0
    for step in range(25):
        n = rng.integers(0, max_rows + 1, streams) * (rng.random(streams) < 0.8)
        if step % 7 == 6:
            n[rng.integers(0, streams)] = max_rows + 1  # more than it may
        if step % 5 == 4:
            ctx[rng.integers(0, streams)] = -1
        start = np.concatenate([[0], np.cumsum(n)])
        before = _bytes(pools)
        lib.kv_reserve(pages, ls, _cu(torch, start.astype(np.int32)), _cu(torch, ctx.astype(np.int32)), ok, max_rows)
        table, refs, want, copies = so.reserve(table, refs, start, ctx, max_rows, page)
        assert np.array_equal(ok.cpu().numpy(), want), step
        assert np.array_equal(dt.cpu().numpy(), table), step
        assert np.array_equal(dr.cpu().numpy(), refs), step
        after = _moved(before, [((p, i), (q, i)) for p, q, slots in copies for i in range(slots)])
        assert _same(_bytes(pools), after), step
        short += int((want == 0).sum())
        copied += len(copies)
        ctx = np.where(want == 1, np.maximum(ctx, 0) + np.minimum(n, max_rows), np.maximum(ctx, 0))
        parent = np.where(rng.random(streams) < 0.6, np.arange(streams), rng.integers(-1, streams, streams)).astype(np.int32)
        length = np.where(parent >= 0, ctx[np.maximum(parent, 0)], 0)
        cut = rng.random(streams) < 0.3
        length[cut] = (length[cut] * rng.random(cut.sum())).astype(np.int64)
        lib.kv_fork(pages, _cu(torch, parent), _cu(torch, length.astype(np.int32)))
        table, refs = so.fork(table, refs, parent, length, page)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs), step
        ctx = length.copy()
        # what is held adds up
        held = np.bincount(table[table >= 0], minlength=n_pages)
        assert ((refs - held >= 0) & (refs - held <= 1)).all() and (refs - held).sum() == 1
    assert streams == 1 or (short > 0 and copied > 0)


@pytest.mark.parametrize("held_from", [3000, 1200])
def test_reserve_many_streams(torch_gpu, held_from):
    """More streams than the threads that keep the books, most of them on shared pages; and too few pages at the end."""
    torch = torch_gpu
    streams, stride, page = 2500, 3, 16
    rng = np.random.default_rng(3)
    table = np.full((streams, stride), -1, np.int32)
    groups = rng.integers(0, 400, streams)
    ctx = (rng.integers(1, 32, 400)[groups]).astype(np.int32)
    n_pages = 5000
    order = rng.permutation(n_pages).astype(np.int32)
    for s in range(streams):
        for j in range(-(-int(ctx[s]) // page)):
            table[s, j] = order[2 * groups[s] + j]
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    refs[order[held_from:]] += 1
    n = rng.integers(0, 3, streams)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    pools = _pools(torch, rng, "f16", 1, n_pages, 1, page, 64)
    dt, dr, ok = _cu(torch, table), _cu(torch, refs), torch.empty(streams, dtype=torch.int32, device="cuda")
    before = _bytes(pools)
    lib.kv_reserve(lib.KVPages(dt, dr, page), _layers(torch, pools, dt), _cu(torch, start), _cu(torch, ctx), ok, 2)
    table, refs, want, copies = so.reserve(table, refs, start, ctx, 2, page)
    assert np.array_equal(ok.cpu().numpy(), want) and np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    assert copies and (want.all() or held_from == 1200)
    assert _same(_bytes(pools), _moved(before, [((p, i), (q, i)) for p, q, k in copies for i in range(k)]))


def test_reserve_last_pages_of_a_large_pool(torch_gpu):
    """The free pages stand behind many held ones."""
    torch = torch_gpu
    n_pages, page = 30000, 16
    refs = np.ones(n_pages, np.int32)
    refs[[4095, 4096, 17000, 29999]] = 0
    table = np.full((2, 4), -1, np.int32)
    pools = _pools(torch, np.random.default_rng(0), "i8", 1, n_pages, 1, page, 64)
    dt, dr, ok = _cu(torch, table), _cu(torch, refs), torch.empty(2, dtype=torch.int32, device="cuda")
    lib.kv_reserve(lib.KVPages(dt, dr, page), _layers(torch, pools, dt), _cu(torch, np.array([0, 30, 64], np.int32)),
                   _cu(torch, np.array([0, 16], np.int32)), ok, 34)
    assert ok.tolist() == [1, 0] and dt.tolist() == [[4095, 4096, -1, -1], [-1] * 4]
    lib.kv_reserve(lib.KVPages(dt, dr, page), _layers(torch, pools, dt), _cu(torch, np.array([0, 0, 20], np.int32)),
                   _cu(torch, np.array([30, 28], np.int32)), ok, 34)
    assert ok.tolist() == [1, 1] and dt.tolist() == [[4095, 4096, -1, -1], [-1, 17000, 29999, -1]]
    assert (dr == 1).all()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("streams,heads,dim,page,layers,max_rows", [(1, 1, 64, 16, 1, 64), (5, 12, 64, 64, 12, 27), (3, 8, 128, 48, 2, 64),
                                                                     (70, 2, 128, 16, 1, 5)])
def test_compact(torch_gpu, cache, streams, heads, dim, page, layers, max_rows):
    """Any row to any place, many to one, none, places that do not exist: bits move, nothing else does."""
    torch = torch_gpu
    print(f"compact {cache} {streams} {heads}x{dim} page {page}", flush=True)
    rng = np.random.default_rng(streams * 5 + dim)
    stride = 200 // page + 2
    n_pages = streams * stride + 2
    pools = _pools(torch, rng, cache, layers, n_pages, heads, page, dim)
    table = rng.permutation(n_pages)[:streams * stride].reshape(streams, stride).astype(np.int32)
    table[rng.random(table.shape) < 0.05] = -1
    table[0, -1] = n_pages
    dt = _cu(torch, table)
    ls = _layers(torch, pools, dt)
    for how in range(4):
        n = rng.integers(0, max_rows + 1, streams)
        n[0] = max_rows + (2 if how == 3 else 0)
        start = np.concatenate([[0], np.cumsum(n)])
        ctx = rng.integers(0, stride * page, streams) if how == 1 else rng.integers(0, 130, streams)
        kept = np.full(int(start[-1]) + 3, -1, np.int32)
        for s in range(streams):
            m = int(n[s])
            if how == 0:  # a path: increasing
                got = np.sort(rng.permutation(m)[:rng.integers(0, m + 1)])
            elif how == 1:  # any order, out of range too
                got = rng.integers(-2, m + 3, m)
            else:
                got = rng.permutation(m)
            kept[start[s]:start[s] + len(got)] = got
        if how == 2 and streams > 2:
            ctx[1] = -5

        def place(s, pos):
            j = pos // page
            return (int(table[s, j]), pos % page) if j < stride and 0 <= table[s, j] < n_pages else None
        before = _bytes(pools)
        lib.kv_compact(ls, _cu(torch, start.astype(np.int32)), _cu(torch, ctx.astype(np.int32)), _cu(torch, kept), max_rows)
        assert _same(_bytes(pools), _moved(before, so.compact(place, ctx, start, kept, max_rows))), how


def test_page_calls_captured(torch_gpu):
    """A step of four beams as a graph: each replay goes on from where the last one ended."""
    torch = torch_gpu
    rng = np.random.default_rng(8)
    streams, stride, n_pages, page = 4, 8, 40, 16
    pools = _pools(torch, rng, "f16", 2, n_pages, 2, page, 64)
    table, refs = np.full((streams, stride), -1, np.int32), np.zeros(n_pages, np.int32)
    dt, dr = _cu(torch, table), _cu(torch, refs)
    ok, ctx, parent = (torch.zeros(streams, dtype=torch.int32, device="cuda") for _ in range(3))
    start = torch.arange(streams + 1, dtype=torch.int32, device="cuda") * 3
    pages, ls = lib.KVPages(dt, dr, page), _layers(torch, pools, dt)
    ws = torch.full((max(lib.kv_fork_workspace(pages), lib.kv_reserve_workspace(pages, 3), 16),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        lib.kv_fork(pages, parent, ctx, workspace=ws)
        lib.kv_reserve(pages, ls, start, ctx, ok, 3, workspace=ws)
    h = 0
    for step in range(12):
        want_parent = rng.integers(0, streams, streams).astype(np.int32)
        parent.copy_(torch.from_numpy(want_parent))
        ctx.fill_(h)
        before = _bytes(pools)
        g.replay()
        torch.cuda.synchronize()
        table, refs = so.fork(table, refs, want_parent, np.full(streams, h), page)
        table, refs, want, copies = so.reserve(table, refs, np.arange(5) * 3, np.full(streams, h), 3, page)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs) and np.array_equal(ok.cpu().numpy(), want)
        assert _same(_bytes(pools), _moved(before, [((p, i), (q, i)) for p, q, k in copies for i in range(k)]))
        h += 3


# ---------------------------------------------------------------- adapters

def _adapter_case(rng, rows, cols, out, rank, n, mixed=True):
    a = (rng.standard_normal((n, rank, cols)) / np.sqrt(cols)).astype(np.float16)
    b = (0.3 * rng.standard_normal((n, out, rank))).astype(np.float16)
    ranks = rng.integers(0, rank + 1, n).astype(np.int32) if mixed else np.full(n, rank, np.int32)
    ranks[0] = rank
    for i in range(n):  # what stands behind an adapter's rank is nobody's business
        a[i, ranks[i]:] = np.nan
        b[i, :, ranks[i]:] = np.inf
    scale = rng.uniform(-2, 2, n).astype(np.float32)
    return a, b, ranks, scale


def _adapter_want(x, base, which, a, b, ranks, scale, x_f32):
    """y in 64 bits, and how far 32-bit sums may be from it."""
    y, tol = base.copy(), np.zeros_like(base)
    cols = x.shape[1]
    for r, i in enumerate(which):
        if not 0 <= i < len(a):
            continue
        k = int(ranks[i])
        A, B = a[i, :k].astype(np.float64), b[i, :, :k].astype(np.float64)
        t, mag = A @ x[r], np.abs(A) @ np.abs(x[r])
        # A sum of 128 products: 32 at a time and no more than 8 such steps, each cut by up to 2^-23 of the magnitudes, then one rounding
        # for each 128 columns of a wave and each wave: within (16 + cols / 128) 2^-23.  32-bit rows: 22 bits of an element, or
        # 2^-36 of the largest near it.
        dt = mag * (16 + cols / 128) * 2 * U32
        if x_f32:
            dt = dt + mag * 2.0 ** -22 + np.abs(A).sum(1) * np.abs(x[r]).max() * 2.0 ** -36
        # t itself in 22 bits, the sum over ranks in the same way, scale and base: two roundings of 32 bits
        s = abs(float(scale[i]))
        y[r] = base[r] + float(scale[i]) * (B @ t)
        B = np.abs(B)
        tol[r] = s * (B @ (dt + np.abs(t) * 2.0 ** -22) + B @ np.abs(t) * 16 * 2 * U32 + B.sum(1) * (np.abs(t).max() if k else 0.0) * 2.0 ** -36)
        tol[r] += 4 * U32 * (np.abs(y[r]) + np.abs(base[r]))
    return y, tol


@pytest.mark.parametrize("rows,cols,out,rank,n", [(1, 32, 16, 16, 1), (1, 768, 2304, 16, 4), (3, 64, 48, 32, 2), (15, 768, 768, 16, 20),
                                                  (16, 160, 80, 64, 3), (17, 1024, 272, 128, 17), (64, 768, 2304, 16, 64), (33, 4096, 4112, 64, 5),
                                                  (70, 96, 16, 48, 200), (181, 768, 2304, 16, 2), (700, 288, 144, 112, 9), (2100, 64, 64, 16, 3),
                                                  (1500, 512, 528, 32, 600)])
@pytest.mark.parametrize("x_dtype,y_dtype", [("float32", "float32"), ("float16", "float16"), ("float32", "float16"), ("float16", "float32")])
def test_adapter_rows(torch_gpu, rows, cols, out, rank, n, x_dtype, y_dtype):
    torch = torch_gpu
    print(f"adapters {rows} {cols}->{out} rank {rank} of {n} {x_dtype} {y_dtype}", flush=True)
    rng = np.random.default_rng(rows + cols + n)
    a, b, ranks, scale = _adapter_case(rng, rows, cols, out, rank, n)
    x = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).to(getattr(torch, x_dtype))
    base = torch.from_numpy(rng.standard_normal((rows, out)).astype(np.float32)).to(getattr(torch, y_dtype))
    which = rng.integers(-1, n + 1, rows).astype(np.int32) if rows % 3 else np.repeat(rng.integers(-1, n, rows // 3), 3).astype(np.int32)
    which[0] = 0
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    y = torch.full((rows, out), float("nan"), dtype=base.dtype, device="cuda")
    lib.adapter_rows(x.cuda(), ad, _cu(torch, which), y, base=base.cuda())
    want, tol = _adapter_want(x.double().numpy(), base.double().numpy(), which, a, b, ranks, scale, x_dtype == "float32")
    got = y.double().cpu().numpy()
    if y_dtype == "float16":
        tol += U16 * (np.abs(want) + tol) + 2.0 ** -25
    tol[(which < 0) | (which >= n)] = 0  # those rows are copied
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) - tol)
    # in place, rows at odd strides and addresses: the same bits, nothing beside them touched
    wide = torch.full((rows, out + 3), 5.0, dtype=base.dtype, device="cuda")
    place = wide[:, 1:1 + out]
    place.copy_(base.cuda())
    xs = torch.full((rows, cols + 5), float("nan"), dtype=x.dtype, device="cuda")
    xs[:, 3:3 + cols] = x.cuda()
    lib.adapter_rows(xs[:, 3:3 + cols], ad, _cu(torch, which), place)
    assert torch.equal(place, y)
    assert (wide[:, 0] == 5).all() and (wide[:, 1 + out:] == 5).all()


def test_adapters_without_ranks_and_scales(torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(2)
    a, b, ranks, scale = _adapter_case(rng, 40, 128, 64, 32, 3, mixed=False)
    x, base = (rng.standard_normal((40, w)).astype(np.float32) for w in (128, 64))
    which = rng.integers(0, 3, 40).astype(np.int32)
    y, y2 = (torch.empty(40, 64, device="cuda") for _ in range(2))
    lib.adapter_rows(_cu(torch, x), lib.Adapters(_cu(torch, a), _cu(torch, b)), _cu(torch, which), y, base=_cu(torch, base))
    ones = np.ones(3, np.float32)
    lib.adapter_rows(_cu(torch, x), lib.Adapters(*(_cu(torch, v) for v in (a, b, np.full(3, 99, np.int32), ones))), _cu(torch, which), y2,
                     base=_cu(torch, base))
    want, tol = _adapter_want(x.astype(np.float64), base.astype(np.float64), which, a, b, ranks, ones, True)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all() and torch.equal(y, y2)
    lib.adapter_rows(_cu(torch, x), lib.Adapters(_cu(torch, a), _cu(torch, b), _cu(torch, np.array([0, -5, 0], np.int32))), _cu(torch, which), y,
                     base=_cu(torch, base))
    assert np.array_equal(y.cpu().numpy(), base)


@pytest.mark.parametrize("scale_of_x", [1e-30, 1e-6, 1e6, 1e30])
def test_adapters_far_from_one(torch_gpu, scale_of_x):
    """32-bit rows of any size, and rows of different sizes next to each other: nothing leaves a 16-bit range."""
    torch = torch_gpu
    rng = np.random.default_rng(12)
    a, b, ranks, scale = _adapter_case(rng, 20, 384, 64, 16, 2, mixed=False)
    x = rng.standard_normal((20, 384)).astype(np.float32)
    x[::2] *= np.float32(scale_of_x)
    x[5] = 0
    x[7, :128] *= np.float32(1e-20)
    base = np.zeros((20, 64), np.float32)
    which = (np.arange(20) % 2).astype(np.int32)
    y = torch.empty(20, 64, device="cuda")
    lib.adapter_rows(_cu(torch, x), lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale))), _cu(torch, which), y, base=_cu(torch, base))
    want, tol = _adapter_want(x.astype(np.float64), base.astype(np.float64), which, a, b, ranks, scale, True)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol + 2.0 ** -140).all()


def test_adapter_rows_keep_to_themselves(torch_gpu):
    """A row with an Inf or NaN spoils no other row; the same row gives the same bits wherever it stands."""
    torch = torch_gpu
    rng = np.random.default_rng(3)
    a, b, ranks, scale = _adapter_case(rng, 50, 256, 96, 16, 2, mixed=False)
    x, base = (rng.standard_normal((50, w)).astype(np.float32) for w in (256, 96))
    which = rng.integers(0, 2, 50).astype(np.int32)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    y, z = (torch.empty(50, 96, device="cuda") for _ in range(2))
    lib.adapter_rows(_cu(torch, x), ad, _cu(torch, which), y, base=_cu(torch, base))
    bad = x.copy()
    bad[[4, 20]], bad[33, 5], bad[34, 7] = np.inf, np.nan, -np.inf
    lib.adapter_rows(_cu(torch, bad), ad, _cu(torch, which), z, base=_cu(torch, base))
    spoilt = [4, 20, 33, 34]
    good = np.setdiff1d(np.arange(50), spoilt)
    assert torch.equal(y[good], z[good]) and not torch.isfinite(z[spoilt]).any()
    order = rng.permutation(50)
    lib.adapter_rows(_cu(torch, x[order]), ad, _cu(torch, which[order]), z, base=_cu(torch, base[order]))
    assert torch.equal(z, y[torch.from_numpy(order).cuda()])
    one = torch.empty(1, 96, device="cuda")
    lib.adapter_rows(_cu(torch, x[7:8]), ad, _cu(torch, which[7:8]), one, base=_cu(torch, base[7:8]))
    assert torch.equal(one[0], y[7])


def test_adapters_captured(torch_gpu):
    torch = torch_gpu
    rng = np.random.default_rng(13)
    a, b, ranks, scale = _adapter_case(rng, 30, 768, 2304, 16, 4, mixed=False)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    x, y = torch.zeros(30, 768, device="cuda"), torch.zeros(30, 2304, device="cuda")
    base, which = torch.randn(30, 2304, device="cuda"), torch.zeros(30, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        lib.adapter_rows(x, ad, which, y, base=base)
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((30, 768)).astype(np.float32)))
        which.copy_(torch.from_numpy(rng.integers(-1, 4, 30).astype(np.int32)))
        g.replay()
        eager = torch.empty_like(y)
        lib.adapter_rows(x, ad, which, eager, base=base)
        torch.cuda.synchronize()
        assert torch.equal(eager, y)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_a_serving_loop(torch_gpu, cache):
    """Steps of three streams with voices of their own: room in the cache, the shared projection and the adapters, rotation, cache,
    attention of a drafted tree, verification, accepted nodes to their places; then the streams are reordered.  What the
    cache holds at the end is what each stream's accepted tokens put there."""
    torch = torch_gpu
    rng = np.random.default_rng(31)
    streams, heads, dim, page, n_pages, vocab, tree = 3, 2, 64, 16, 40, 97, 6
    width = heads * dim
    w = torch.from_numpy(rng.standard_normal((vocab, width)).astype(np.float32)).cuda()
    emb = torch.from_numpy(rng.standard_normal((vocab, width)).astype(np.float32)).cuda()
    proj = torch.from_numpy((rng.standard_normal((3 * width, width)) / 12).astype(np.float32)).cuda()
    a, b, ranks, scale = _adapter_case(rng, 0, width, 3 * width, 16, 2, mixed=False)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    pools = _pools(torch, rng, cache, 1, n_pages, heads, page, dim)
    table = torch.full((streams, 6), -1, dtype=torch.int32, device="cuda")
    refs, ok = torch.zeros(n_pages, dtype=torch.int32, device="cuda"), torch.zeros(streams, dtype=torch.int32, device="cuda")
    pages, ls = lib.KVPages(table, refs, page), _layers(torch, pools, table)
    kv, rope = ls.caches[0], lib.Rope(dim)
    ctx, last = np.zeros(streams, np.int64), np.array([3, 5, 7])
    said = [[] for _ in range(streams)]  # tokens whose keys are committed, with the voice that wrote them
    voice = np.array([0, 1, -1], np.int32)
    i32 = lambda v: _cu(torch, np.asarray(v, np.int32))  # noqa: E731

    def project(tok, who):
        x = emb[torch.as_tensor(np.asarray(tok), device="cuda")]
        y = x @ proj.T
        lib.adapter_rows(x, ad, i32(who), y)
        return (t.reshape(-1, heads, dim).contiguous() for t in y.split(width, 1))
    for step in range(9):
        n = rng.integers(2, tree + 1, streams)
        start = np.concatenate([[0], np.cumsum(n)])
        stream = np.repeat(np.arange(streams), n)
        node = np.concatenate([np.arange(k) for k in n])
        tok, mask, depth = rng.integers(0, vocab, start[-1]), np.zeros(start[-1], np.uint64), np.zeros(start[-1], np.int64)
        for r in range(start[-1]):
            s0 = start[stream[r]]
            if node[r] == 0:
                tok[r], mask[r] = last[stream[r]], 1
            else:
                up = int(rng.integers(0, node[r]))
                mask[r], depth[r] = int(mask[s0 + up]) | 1 << int(node[r]), depth[s0 + up] + 1
        lib.kv_reserve(pages, ls, i32(start), i32(ctx), ok, tree)
        assert ok.tolist() == [1, 1, 1]
        q, k, v = project(tok, voice[stream])
        pos = ctx[stream] + depth
        lib.rope_rows(q, i32(pos), rope)
        lib.kv_write(kv, k, v, i32(stream), i32(ctx[stream] + node), rope=rope, rope_pos=i32(pos))
        out = torch.empty_like(q)
        lib.attn_tree(q, kv, i32(start), i32(ctx), out, tree, 96, row_mask=_cu(torch, mask.view(np.int64)))
        logits = out.reshape(-1, width) @ w.T
        u = rng.random(start[-1]) * 0.5  # (a number below a half accepts more often)
        acc, nxt = (torch.empty(streams, dtype=torch.int32, device="cuda") for _ in range(2))
        path = torch.empty(int(start[-1]), dtype=torch.int32, device="cuda")
        # the likeliest token after each parent is what is drafted, so that paths grow
        best = logits.argmax(1).cpu().numpy()
        for r in range(start[-1]):
            if node[r]:
                up = so._parent(int(node[r]), mask[start[stream[r]]:])
                tok[r] = best[start[stream[r]] + up]
        q, k, v = project(tok, voice[stream])  # (the keys of the tokens that were drafted after all)
        lib.kv_write(kv, k, v, i32(stream), i32(ctx[stream] + node), rope=rope, rope_pos=i32(pos))
        lib.verify_tokens(logits, i32(tok), i32(start), acc, path, nxt, tree, uniforms=_cu(torch, u), row_mask=_cu(torch, mask.view(np.int64)))
        *want, near = so.verify(logits.double().cpu().numpy(), tok, start, u, tree, mask=mask, path=np.zeros(start[-1]))
        assert near > 1 and np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(path.cpu().numpy(), want[1])
        lib.kv_compact(ls, i32(start), i32(ctx), path, tree)
        for s in range(streams):
            said[s] += [(int(tok[start[s] + j]), int(voice[s])) for j in want[1][start[s]:start[s + 1]] if j >= 0]
        ctx, last = ctx + want[0] + 1, want[2].copy()
        if step % 3 == 1:
            parent = rng.integers(0, streams, streams)
            lib.kv_fork(pages, i32(parent), i32(ctx[parent]))
            ctx, last, said = ctx[parent], last[parent], [list(said[p]) for p in parent]
            voice = voice[parent]
    assert max(len(x) for x in said) > 12
    # written once more, one after the other, into a cache of its own
    plain = _pools(torch, rng, cache, 1, streams * 6, heads, page, dim)
    own = torch.arange(streams * 6, dtype=torch.int32, device="cuda").view(streams, 6)
    kv2 = _layers(torch, plain, own).caches[0]
    for s in range(streams):
        m = len(said[s])
        assert m == ctx[s]
        _, k, v = project([t for t, _ in said[s]], [g for _, g in said[s]])
        at, who = i32(np.arange(m)), i32(np.full(m, s))
        lib.kv_write(kv2, k, v, who, at, rope=rope)
        got, want = ([torch.empty(m, heads, dim, device="cuda") for _ in range(2)] for _ in range(2))
        lib.kv_read(kv, who, at, *got)
        lib.kv_read(kv2, who, at, *want)
        for g, x in zip(got, want):
            # rows of a product of 128 columns of another shape: their sums may be taken in another order (128 * 2^-24 of the
            # magnitudes, which are within 12 times the largest of a head here), then a step of the cache
            top = x.abs().amax(-1, keepdim=True)
            step = 2.0 ** -11 if cache == "f16" else 1.01 / 127.0
            assert ((g - x).abs() <= top * (step + 12 * 128 * U32)).all()
