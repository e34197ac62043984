"""Decisions of the verification that come near their borders, and those behind likely siblings that were rejected, where what is left of the
probability is a small difference (GPU)."""
import numpy as np
import pytest

import serving_oracle as so
from test_gpu_serving_ops import _held, _verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,kids", [(50, 2), (1024, 2), (1024, 3), (16384, 2), (70001, 3)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("left", [6e-4, 2e-5, 1e-7])
def test_verify_behind_likely_siblings(torch_gpu, vocab, kids, dtype, left):
    """The last child's number is 2^-16 of itself above or below the border p(t) / (1 - p of its elder siblings).  The call's
    probabilities are off by up to 2^-44 of themselves, so what is left of 1 by 2^-44 / 1e-7 = 2^-20.7 of itself at most; its draws by
    some 2^-40.  The elder children's numbers, 1, come within 1e-7 of their borders, the draws' within a hundredth of 1e-10."""
    torch = torch_gpu
    print(f"siblings {vocab} {kids} {dtype} {left}", flush=True)
    rng = np.random.default_rng(vocab + kids)
    streams, n = 40 if vocab < 2000 else 12, kids + 1
    x = 2.0 * rng.standard_normal((streams * n, vocab)).astype(np.float32)
    tok, u = rng.integers(0, vocab, streams * n).astype(np.int32), rng.random(streams * n)
    for s in range(streams):
        r = s * n
        tok[r + 1:r + n] = rng.permutation(vocab)[:kids]
        rest = np.log(np.exp(np.delete(x[r].astype(np.float64), tok[r + 1:r + kids])).sum())
        # the elder children have all but `left` of the probability, the first of two the most of it
        for i, t in enumerate(tok[r + 1:r + kids]):
            x[r, t] = rest - np.log(left) - 3.0 * i
        p = so.softmax(_held(torch, x[r:r + 1], getattr(torch, dtype))[0], 1.0)
        u[r + 1:r + kids] = 1.0
        gone = p[tok[r + 1:r + kids]]
        u[r + kids] = p[tok[r + kids]] / np.delete(p, tok[r + 1:r + kids]).sum() * (1.0 + (2.0 ** -16 if s % 2 else -(2.0 ** -16)))
        assert (gone < 1).all() and 0 < u[r + kids] < 1
    mask = np.tile(np.array([1] + [1 | 1 << i for i in range(1, n)], np.uint64), streams)
    start, dt = (np.arange(streams + 1) * n).astype(np.int32), getattr(torch, dtype)
    *want, near = so.verify(_held(torch, x, dt), tok, start, u, n, None, mask, path=np.full(len(tok), -7))
    assert near > 0.01  # of 2^-18 and of 1e-10: 2^-24.6 and 2^-39.9
    got = _verify(torch, x, tok, start, n, u, mask=mask, dtype=dt)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    assert np.array_equal(got[0], (np.arange(streams) + 1) % 2)


@pytest.mark.parametrize("vocab,rows", [(300, 6), (1024, 5), (9000, 6), (40000, 4), (130001, 5)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("draft", [False, True])
def test_verify_numbers_at_their_borders(torch_gpu, vocab, rows, dtype, draft):
    """Numbers 2^-30 of themselves above or below the border of their child, several in one chain: probabilities are within 2^-44 there.
    (Only what is accepted is compared: the draws' numbers come near to no border on purpose.)"""
    torch = torch_gpu
    print(f"borders {vocab} {dtype} {draft}", flush=True)
    rng = np.random.default_rng(vocab + rows)
    streams, dt = 24 if vocab < 50000 else 6, getattr(torch, dtype)
    x = 2.0 * rng.standard_normal((streams * rows, vocab)).astype(np.float32)
    tok = rng.integers(0, vocab, streams * rows).astype(np.int32)
    x[np.arange(len(tok))[:-1], tok[1:]] += np.float32(12.0)
    y = None
    if draft:  # the draft is surer of its tokens than the target, so that every border is below 1
        y = (x + 0.2 * rng.standard_normal(x.shape)).astype(np.float32)
        y[np.arange(len(tok))[:-1], tok[1:]] += np.float32(3.0)
    u, want = rng.random(len(tok)), np.zeros(streams, np.int64)
    for s in range(streams):
        stop = int(rng.integers(1, rows + 1))  # the first node that is rejected, or none
        want[s] = stop - 1
        for i in range(1, rows):
            r = s * rows + i
            p = so.softmax(_held(torch, x[r - 1:r], dt)[0], 0.8)[tok[r]]
            border = p / (so.softmax(_held(torch, y[r - 1:r], dt)[0], 0.9)[tok[r]] if draft else 1.0)
            assert 0 < border < 0.9999999
            u[r] = border * (1.0 + (2.0 ** -30 if i >= stop else -(2.0 ** -30)))
    start = (np.arange(streams + 1) * rows).astype(np.int32)
    kw = dict(inv_temperature=0.8, draft_inv_temperature=0.9)
    for mask in [None] if draft else [None, np.tile(np.array([(1 << i + 1) - 1 for i in range(rows)], np.uint64), streams)]:
        acc, path, _ = _verify(torch, x, tok, start, rows, u, y=y, mask=mask, dtype=dt, **kw)
        assert np.array_equal(acc, want)
        assert np.array_equal(path.reshape(streams, rows), np.where(np.arange(rows) <= want[:, None], np.arange(rows), -1))
