"""Greedy verification of streams of few short rows, which one launch serves, and at the sizes where it ends (GPU)."""
import numpy as np
import pytest

import serving_oracle as so
from test_gpu_serving_ops import _check_verify, _draft

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,rows", [(1, 8), (3, 8), (1000, 5), (1024, 5), (1025, 16), (1025, 17), (4000, 8), (4097, 6), (4097, 7), (10001, 3),
                                        (10001, 4), (32768, 1), (32769, 1)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_greedy_of_few_rows(torch_gpu, vocab, rows, dtype):
    """Chains and trees of 1 to `rows` nodes and more: ties go to the lowest index, also between the pieces of a row; NaN is nobody's
    likeliest token, +inf is; a row of nothing but NaN or -inf has none."""
    torch = torch_gpu
    print(f"greedy {vocab} {rows} {dtype}", flush=True)
    rng = np.random.default_rng(vocab + rows)
    n = [1, rows, 0, *(int(k) for k in rng.integers(1, rows + 1, 20)), rows, rows + 2]  # (those past max_rows take no part)
    x, _, mask, start = _draft(rng, n, vocab, False, spare=1)
    x = np.round(x * 2) / 2  # many equal values
    total, kinds = int(start[-1]), rng.integers(0, 9, int(start[-1]))
    for r in range(total):
        if kinds[r] == 0:
            x[r, rng.integers(0, vocab, max(1, vocab // 3))] = np.nan
        elif kinds[r] == 1:
            x[r, rng.integers(0, vocab, 2)] = np.inf
        elif kinds[r] == 2:
            x[r] = -np.inf
        elif kinds[r] == 3:
            x[r] = np.nan
        elif kinds[r] == 4:  # the same largest value in every piece
            x[r, rng.integers(0, 64)::64] = 30.0
    best = np.argmax(np.where(np.isnan(x), -np.inf, x), 1).astype(np.int32)
    for chain in (False, True):
        tok = np.full(len(x), -1, np.int32)
        for s in range(len(n)):
            for i in range(start[s], start[s + 1]):
                up = i - start[s] - 1 if chain else so._parent(i - start[s], mask[start[s]:])
                tok[i] = best[start[s] + max(up, 0)] if rng.random() < 0.85 else rng.integers(-1, vocab + 1)
        acc, _, nxt = _check_verify(torch, x, tok, start, rows, mask=None if chain else mask, greedy=True, pad=1, dtype=getattr(torch, dtype))
        assert nxt[2] == -1 and acc[2] == 0 and (rows < 3 or acc.max() > 1)
