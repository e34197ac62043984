"""The serving-loop operators at the edges of what they may touch (GPU): workspaces with guards around them, broadcast inputs, adapters
that are replaced, calls on a stream of their own and two at once."""
import numpy as np
import pytest

import serving_oracle as so
from mosship import lib
from test_gpu_serving_ops import _adapter_case, _adapter_want, _cu, _draft, _layers, _pools

pytestmark = pytest.mark.gpu
GUARD = 4096


def _guarded(torch, size):
    """A workspace of exactly this size inside sentinels."""
    whole = torch.full((size + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
    return whole, whole[GUARD:GUARD + size]


def _untouched(whole, size):
    return bool((whole[:GUARD] == 0xA5).all()) and bool((whole[GUARD + size:] == 0xA5).all())


@pytest.mark.parametrize("vocab,streams,rows,draft", [(1024, 3, 9, True), (40000, 5, 6, True), (40000, 5, 30, False), (131073, 2, 64, False),
                                                      (70001, 3, 12, True), (5000, 40, 3, False)])
def test_verify_workspace(torch_gpu, vocab, streams, rows, draft):
    torch = torch_gpu
    print(f"verify workspace {vocab} {streams} {rows} {draft}", flush=True)
    rng = np.random.default_rng(vocab + rows)
    x, tok, mask, start = _draft(rng, [rows] * streams, vocab, draft, near=0.9, peak=18.0)
    y = (x + 0.5 * rng.standard_normal(x.shape)).astype(np.float32) if draft else None
    u = rng.random(len(tok))
    size = lib.verify_tokens_workspace(streams, rows, vocab, draft)
    whole, ws = _guarded(torch, size)
    acc, nxt = (torch.empty(streams, dtype=torch.int32, device="cuda") for _ in range(2))
    path = torch.empty(len(tok), dtype=torch.int32, device="cuda")
    lib.verify_tokens(_cu(torch, x), _cu(torch, tok), _cu(torch, start), acc, path, nxt, rows, uniforms=_cu(torch, u),
                      draft_logits=None if y is None else _cu(torch, y), row_mask=None if draft else _cu(torch, mask.view(np.int64)), workspace=ws)
    *want, near = so.verify(x, tok, start, u, rows, y, None if draft else mask, path=np.zeros(len(tok)))
    assert near > 1
    for got, w in zip((acc, path, nxt), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert _untouched(whole, size)


@pytest.mark.parametrize("streams,stride,max_rows", [(5, 4, 20), (1030, 40, 33), (200, 8, 100)])
def test_page_workspaces(torch_gpu, streams, stride, max_rows):
    torch = torch_gpu
    print(f"page workspaces {streams} {stride}", flush=True)
    rng = np.random.default_rng(streams)
    page, n_pages = 16, 3 * streams + 50
    pools = _pools(torch, rng, "i8", 1, n_pages, 1, page, 64)
    table, refs = np.full((streams, stride), -1, np.int32), np.zeros(n_pages, np.int32)
    dt, dr, ok = _cu(torch, table), _cu(torch, refs), torch.empty(streams, dtype=torch.int32, device="cuda")
    pages, ls = lib.KVPages(dt, dr, page), _layers(torch, pools, dt)
    ctx = np.zeros(streams, np.int64)
    side = torch.cuda.Stream()
    for step in range(3):
        n = rng.integers(0, min(max_rows, 30) + 1, streams)
        start = np.concatenate([[0], np.cumsum(n)])
        parent = rng.integers(-1, streams, streams).astype(np.int32)
        args = [_cu(torch, a.astype(np.int32)) for a in (start, ctx, parent)]
        sizes = lib.kv_reserve_workspace(pages, max_rows), lib.kv_fork_workspace(pages)
        guards = [_guarded(torch, s) for s in sizes]
        side.wait_stream(torch.cuda.current_stream())
        lib.kv_reserve(pages, ls, args[0], args[1], ok, max_rows, workspace=guards[0][1], stream=side.cuda_stream)
        table, refs, want, _ = so.reserve(table, refs, start, ctx, max_rows, page)
        ctx = np.where(want == 1, ctx + n, ctx)
        length = np.where(parent >= 0, ctx[parent], 0)
        new_len = _cu(torch, length.astype(np.int32))
        side.wait_stream(torch.cuda.current_stream())
        lib.kv_fork(pages, args[2], new_len, workspace=guards[1][1], stream=side.cuda_stream)
        side.synchronize()
        table, refs = so.fork(table, refs, parent, length, page)
        ctx = length
        assert np.array_equal(ok.cpu().numpy(), want) and np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
        assert all(_untouched(w, s) for (w, _), s in zip(guards, sizes))


def test_adapters_of_broadcast_rows(torch_gpu):
    """One row of x, and one of base, for all rows (stride 0)."""
    torch = torch_gpu
    rng = np.random.default_rng(1)
    a, b, ranks, scale = _adapter_case(rng, 0, 96, 80, 32, 5)
    x, base = (rng.standard_normal((1, w)).astype(np.float32) for w in (96, 80))
    which = rng.integers(-1, 5, 40).astype(np.int32)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    y = torch.full((40, 80), float("nan"), device="cuda")
    lib.adapter_rows(_cu(torch, x).expand(40, 96), ad, _cu(torch, which), y, base=_cu(torch, base).expand(40, 80))
    want, tol = _adapter_want(np.repeat(x, 40, 0).astype(np.float64), np.repeat(base, 40, 0).astype(np.float64), which, a, b, ranks, scale, True)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


def test_adapters_replaced(torch_gpu):
    """New weights for some adapters; the others' stay."""
    torch = torch_gpu
    rng = np.random.default_rng(2)
    a, b, ranks, scale = _adapter_case(rng, 0, 160, 144, 48, 6)
    a2, b2, ranks2, _ = _adapter_case(rng, 0, 160, 144, 48, 2)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    ad.set(3, _cu(torch, a2), _cu(torch, b2), _cu(torch, ranks2))
    a[3:5], b[3:5], ranks[3:5] = a2, b2, ranks2
    x, base = (rng.standard_normal((30, w)).astype(np.float32) for w in (160, 144))
    which = (np.arange(30) % 6).astype(np.int32)
    y = torch.empty(30, 144, device="cuda")
    lib.adapter_rows(_cu(torch, x), ad, _cu(torch, which), y, base=_cu(torch, base))
    want, tol = _adapter_want(x.astype(np.float64), base.astype(np.float64), which, a, b, ranks, scale, True)
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    with pytest.raises(lib.MossHipError):
        ad.set(5, _cu(torch, a2), _cu(torch, b2), _cu(torch, ranks2))


def test_two_calls_at_once(torch_gpu):
    """Adapters and verification on two streams, each with buffers of its own: what they give alone."""
    torch = torch_gpu
    rng = np.random.default_rng(3)
    a, b, ranks, scale = _adapter_case(rng, 0, 768, 2304, 16, 8)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    x = torch.randn(500, 768, device="cuda")
    base, which = torch.randn(500, 2304, device="cuda"), torch.randint(-1, 8, (500,), dtype=torch.int32, device="cuda")
    z, tok, _, start = _draft(rng, [6] * 20, 30000, True, near=0.9, peak=16.0)
    y = (z + 0.4 * rng.standard_normal(z.shape)).astype(np.float32)
    dz, dy, dt, ds, du = (_cu(torch, v) for v in (z, y, tok, start, rng.random(120)))

    def both(out, acc, path, nxt, ws, stream):
        lib.adapter_rows(x, ad, which, out, base=base, stream=stream)
        lib.verify_tokens(dz, dt, ds, acc, path, nxt, 6, uniforms=du, draft_logits=dy, workspace=ws, stream=stream)
    i32 = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    sets = [(torch.empty(500, 2304, device="cuda"), i32(20), i32(120), i32(20),
             torch.empty(lib.verify_tokens_workspace(20, 6, 30000, True), dtype=torch.uint8, device="cuda")) for _ in range(3)]
    both(*sets[0], None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for bufs, s in zip(sets[1:], streams):
            both(*bufs, s.cuda_stream)
    torch.cuda.synchronize()
    for bufs in sets[1:]:
        assert all(torch.equal(p, q) for p, q in zip(bufs[:4], sets[0][:4]))
