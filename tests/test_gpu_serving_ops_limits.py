"""The serving-loop operators at the ends of the sizes that they take, and what their row ranges may hold (GPU)."""
import numpy as np
import pytest

import serving_oracle as so
from mosship import lib
from test_gpu_serving_ops import _adapter_want, _cu, _draft, _layers, _pools

pytestmark = pytest.mark.gpu


def test_reserve_the_largest_table(torch_gpu):
    """65536 streams of 1024 pages, any of which a call may touch: 2^26 entries, whose books take 2^26 waves.  Streams with
    rows take the lowest free pages in their order; a shared page of the last one is copied."""
    torch = torch_gpu
    streams, stride, page, n_pages = 65536, 1024, 16, 64
    print("largest table", flush=True)
    pools = _pools(torch, np.random.default_rng(0), "i8", 1, n_pages, 1, page, 64)
    table = torch.full((streams, stride), -1, dtype=torch.int32, device="cuda")
    refs = np.zeros(n_pages, np.int32)
    refs[[0, 2]] = 2, 1  # page 0 is that of the last two streams
    table[-2:, 0] = 0
    dr, ok = _cu(torch, refs), torch.full((streams,), -7, dtype=torch.int32, device="cuda")
    n, ctx = np.zeros(streams, np.int64), np.zeros(streams, np.int32)
    n[[0, 1, 30000, 65535]] = 20, 33, 16, 5
    ctx[[30000, 65534, 65535]] = 1023 * 16, 7, 7
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    before = pools["k"].clone(), pools["ks"].clone()
    lib.kv_reserve(lib.KVPages(table, dr, page), _layers(torch, pools, table), _cu(torch, start), _cu(torch, ctx), ok, 1023 * 16)
    torch.cuda.synchronize()
    want = {(0, 0): 1, (0, 1): 3, (1, 0): 4, (1, 1): 5, (1, 2): 6, (30000, 1023): 7, (65534, 0): 0, (65535, 0): 8}
    at = (table >= 0).nonzero().tolist()
    assert {(s, j): int(table[s, j]) for s, j in at} == want
    refs[:9] = 1
    assert np.array_equal(dr.cpu().numpy(), refs) and bool((ok == 1).all())
    before[0][0, 8, :, :7], before[1][0, 8, :, :7] = before[0][0, 0, :, :7], before[1][0, 0, :, :7]
    assert torch.equal(pools["k"], before[0]) and torch.equal(pools["ks"].view(torch.int32), before[1].view(torch.int32))


def test_compact_row_ranges_that_end_far_below_their_start(torch_gpu):
    """A range whose length does not fit 32 bits is one of no rows, as any that ends before it starts: nothing moves, and nothing
    behind the list is looked at (what follows it here would move rows)."""
    torch = torch_gpu
    print("compact row ranges", flush=True)
    streams, page, n_pages, rows = 6, 16, 12, 40
    pools = _pools(torch, np.random.default_rng(1), "e4m3", 2, n_pages, 2, page, 64)
    table = _cu(torch, np.arange(n_pages, dtype=np.int32).reshape(streams, 2))
    ls = _layers(torch, pools, table)
    whole = (torch.arange(rows + 128, device="cuda", dtype=torch.int32) * 7 + 3) % 20
    before = {k: v.view(torch.uint8).clone() for k, v in pools.items()}
    low = -(2 ** 31)
    # ranges of streams 0, 2 and 4 start within the rows and end at the lowest numbers; the others start below 0
    start = _cu(torch, np.array([1, low, rows, low + 1, 39, low + 39, 0], np.int32))
    lib.kv_compact(ls, start, torch.zeros(streams, dtype=torch.int32, device="cuda"), whole[:rows], 64)
    torch.cuda.synchronize()
    assert all(torch.equal(v.view(torch.uint8), before[k]) for k, v in pools.items())


def test_verify_batches_that_shrink(torch_gpu):
    """One workspace, of the bytes that the largest batch asks for, through batches of fewer streams and rows: all as by themselves."""
    torch = torch_gpu
    rng = np.random.default_rng(17)
    vocab, most, rows = 16384, 17, 4
    x, tok, _, start = _draft(rng, [rows] * most, vocab, True, near=0.9, peak=18.0)
    y = (x + 0.5 * rng.standard_normal(x.shape)).astype(np.float32)
    u = rng.random(len(tok))
    size = lib.verify_tokens_workspace(most, rows, vocab, draft=True)
    whole = torch.full((size + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    for streams, max_rows, drafted in ((17, 4, True), (16, 4, True), (16, 4, False), (11, 4, True), (5, 3, True), (1, 4, True), (2, 2, True)):
        print(f"shrink {streams} {max_rows} {drafted}", flush=True)
        n = streams * rows
        acc, nxt = (torch.empty(streams, dtype=torch.int32, device="cuda") for _ in range(2))
        path = torch.full((n,), -7, dtype=torch.int32, device="cuda")
        d = _cu(torch, y[:n]) if drafted else None
        lib.verify_tokens(_cu(torch, x[:n]), _cu(torch, tok[:n]), _cu(torch, start[:streams + 1]), acc, path, nxt, max_rows,
                          uniforms=_cu(torch, u[:n]), draft_logits=d, workspace=whole[4096:4096 + size])
        *want, near = so.verify(x[:n], tok[:n], start[:streams + 1], u[:n], max_rows, y[:n] if drafted else None, path=np.full(n, -7))
        assert near > 1
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip((acc, path, nxt), want))
    assert bool((whole[:4096] == 0xA5).all()) and bool((whole[4096 + size:] == 0xA5).all())


def test_more_adapters_than_a_launch_packs(torch_gpu):
    """70001 adapters, laid out at once and some of them replaced across the first 65535."""
    torch = torch_gpu
    print("many adapters", flush=True)
    n, cols, out, rank = 70001, 32, 16, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    a = (torch.randn(n, rank, cols, generator=g, device="cuda") * cols ** -0.5).half()
    b = (torch.randn(n, out, rank, generator=g, device="cuda") * 0.3).half()
    ranks = torch.randint(0, rank + 1, (n,), generator=g, device="cuda").to(torch.int32)
    scale = torch.rand(n, generator=g, device="cuda") + 0.5
    which = torch.tensor([0, 1, 65534, 65535, 65536, 69999, 70000, 70001, -1, 40000, 65533, 68000], dtype=torch.int32, device="cuda")
    x, base = (torch.randn(which.numel(), w, generator=g, device="cuda") for w in (cols, out))
    ad, y = lib.Adapters(a, b, ranks, scale), torch.empty(which.numel(), out, device="cuda")

    def check():
        lib.adapter_rows(x, ad, which, y, base=base)
        used = which.cpu().numpy().astype(np.int64)
        at = [int(i) if 0 <= i < n else 0 for i in used]
        pick = lambda t: t[at].cpu().numpy()  # noqa: E731
        rows = np.where((used >= 0) & (used < n), np.arange(len(used)), -1).astype(np.int32)
        want, tol = _adapter_want(x.double().cpu().numpy(), base.double().cpu().numpy(), rows, pick(a), pick(b), pick(ranks), pick(scale), True)
        assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    check()
    first, count = 2, 69000
    a[first:first + count] = a[first:first + count].flip(0)
    ranks[first:first + count] = ranks[first:first + count].flip(0)
    ad.set(first, a[first:first + count].contiguous(), b[first:first + count].contiguous(), ranks[first:first + count].contiguous())
    check()
