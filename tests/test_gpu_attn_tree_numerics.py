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
