"""Forms of the serving-loop operators that their documentation allows: rows that are no distribution behind which a tree branches, bases and
outputs at strides of their own, a tree's verification and its compaction in one captured graph (GPU)."""
import numpy as np
import pytest

import serving_oracle as so
from mosship import lib
from test_gpu_serving_ops import (U16, _adapter_case, _adapter_want, _bytes, _check_verify, _cu, _draft, _layers, _moved, _pools, _same)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,rows", [(900, 12), (5000, 12), (70000, 12)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_branching_rows_that_are_no_distribution(torch_gpu, vocab, rows, dtype):
    """A NaN or +inf, or nothing but -inf, in a whole row, in one piece of it or as one value: no child is accepted, no token follows; -inf
    over whole pieces is ruled out."""
    torch = torch_gpu
    print(f"branching no distribution {vocab} {dtype}", flush=True)
    rng = np.random.default_rng(vocab)
    x, tok, _, start = _draft(rng, [rows] * 8, vocab, True, near=1.0, peak=30.0)
    mask = np.tile(np.array([1] + [1 | 1 << i for i in range(1, rows)], np.uint64), 8)  # all children of the root
    root = np.arange(8) * rows
    x[root[0]] = -np.inf
    x[root[1]] = np.nan
    x[root[2], vocab - 1] = np.nan
    x[root[3], vocab // 2] = np.inf
    x[root[4], :vocab // 3] = np.nan
    keep = x[root[5], 5:9].copy()
    x[root[5]] = -np.inf
    x[root[5], 5:9] = keep
    x[root[6], vocab // 2:] = -np.inf
    u = rng.random(len(tok))
    acc, _, nxt = _check_verify(torch, x, tok, start, rows, u, mask=mask, dtype=getattr(torch, dtype))
    assert (acc[:5] == 0).all() and (nxt[:5] == -1).all() and (nxt[5:] >= 0).all() and (5 <= nxt[5] < 9 or acc[5] > 0)


@pytest.mark.parametrize("x_dtype,y_dtype", [("float32", "float32"), ("float16", "float16"), ("float32", "float16"), ("float16", "float32")])
def test_adapters_of_strided_bases_and_outputs(torch_gpu, x_dtype, y_dtype):
    """x, base and y each with a stride and an address of its own, none of them a multiple of 16 bytes; what lies between stays."""
    torch = torch_gpu
    print(f"strided {x_dtype} {y_dtype}", flush=True)
    rng = np.random.default_rng(8)
    rows, cols, out, rank, n = 45, 352, 208, 48, 4
    a, b, ranks, scale = _adapter_case(rng, rows, cols, out, rank, n)
    which = rng.integers(-1, n + 1, rows).astype(np.int32)
    xt, yt = getattr(torch, x_dtype), getattr(torch, y_dtype)
    x = torch.full((rows, cols + 7), float("nan"), dtype=xt, device="cuda")[:, 3:3 + cols]
    base = torch.full((rows, out + 9), float("nan"), dtype=yt, device="cuda")[:, 1:1 + out]
    whole = torch.full((rows + 2, out + 5), 7.0, dtype=yt, device="cuda")
    y = whole[1:-1, 3:3 + out]
    x.copy_(torch.randn(rows, cols, device="cuda"))
    base.copy_(torch.randn(rows, out, device="cuda"))
    lib.adapter_rows(x, lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale))), _cu(torch, which), y, base=base)
    want, tol = _adapter_want(x.double().cpu().numpy(), base.double().cpu().numpy(), which, a, b, ranks, scale, x_dtype == "float32")
    if y_dtype == "float16":
        tol += U16 * (np.abs(want) + tol) + 2.0 ** -25
    tol[(which < 0) | (which >= n)] = 0
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
    y.fill_(7.0)
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("vocab", [700, 9000])
def test_verification_and_compaction_captured(torch_gpu, vocab):
    """One graph that verifies trees and moves the accepted nodes: each replay goes by the numbers and the rows of its time."""
    torch = torch_gpu
    print(f"captured trees {vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    streams, rows, page, stride = 3, 9, 16, 4
    x, tok, mask, start = _draft(rng, [rows] * streams, vocab, False, near=0.9, peak=20.0)
    pools = _pools(torch, rng, "i8", 2, streams * stride, 2, page, 64)
    table = rng.permutation(streams * stride).reshape(streams, stride).astype(np.int32)
    dt = _cu(torch, table)
    ls = _layers(torch, pools, dt)
    dx, dtok, dm, ds = (_cu(torch, v) for v in (x, tok, mask.view(np.int64), start))
    du, ctx = torch.zeros(len(tok), dtype=torch.float64, device="cuda"), torch.zeros(streams, dtype=torch.int32, device="cuda")
    acc, nxt = (torch.empty(streams, dtype=torch.int32, device="cuda") for _ in range(2))
    path = torch.full((len(tok),), -1, dtype=torch.int32, device="cuda")
    ws = torch.full((max(16, lib.verify_tokens_workspace(streams, rows, vocab)),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        lib.verify_tokens(dx, dtok, ds, acc, path, nxt, rows, uniforms=du, row_mask=dm, workspace=ws)
        lib.kv_compact(ls, ds, ctx, path, rows)

    def place(s, pos):
        return int(table[s, pos // page]), pos % page
    for step in range(6):
        u, at = rng.random(len(tok)), rng.integers(0, 40, streams)
        du.copy_(torch.from_numpy(u))
        ctx.copy_(torch.from_numpy(at.astype(np.int32)))
        before = _bytes(pools)
        g.replay()
        torch.cuda.synchronize()
        *want, near = so.verify(x, tok, start, u, rows, mask=mask, path=np.zeros(len(tok)))
        assert near > 1
        assert all(np.array_equal(t.cpu().numpy(), w) for t, w in zip((acc, path, nxt), want)), step
        assert _same(_bytes(pools), _moved(before, so.compact(place, at, start, want[1], rows))), step
