"""Adapters at the ends of the 32-bit range: what scales a row goes into a product as a power of two and a factor of the caller's, which may lie
far from each other (GPU)."""
import numpy as np
import pytest

from mosship import lib
from test_gpu_serving_ops import _adapter_want, _cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [16, 64])
@pytest.mark.parametrize("x_size,b_size,scale", [(1e-33, 0.3, 1.37 * 2.0 ** -6), (1e-33, 300.0, 1.37 * 2.0 ** -12), (1e-30, 3000.0, 1.71 * 2.0 ** -30),
                                                 (1e36, 2.0 ** -18, 1.37 * 2.0 ** 18), (1e36, 2.0 ** -22, -1.9 * 2.0 ** 22), (1e30, 1e-4, 1e4)])
def test_scales_far_from_the_rows(torch_gpu, rank, x_size, b_size, scale):
    """Results within the type's range, of rows and scales whose powers of two, multiplied first, leave it: below 2^-126 that
    product loses bits, above 2^128 it makes NaN of outputs without weights, which are base."""
    torch = torch_gpu
    print(f"range {rank} {x_size} {scale}", flush=True)
    rng = np.random.default_rng(rank)
    rows, cols, out, n = 20, 256, 96, 2
    a = (rng.standard_normal((n, rank, cols)) / np.sqrt(cols)).astype(np.float16)
    b = (b_size * rng.standard_normal((n, out, rank))).astype(np.float16)
    b[:, 7] = 0
    scales = np.array([scale, scale / 3], np.float32)
    x = (x_size * rng.standard_normal((rows, cols))).astype(np.float32)
    base, which = np.zeros((rows, out), np.float32), (np.arange(rows) % n).astype(np.int32)
    y = torch.empty(rows, out, device="cuda")
    lib.adapter_rows(_cu(torch, x), lib.Adapters(_cu(torch, a), _cu(torch, b), scale=_cu(torch, scales)), _cu(torch, which), y, base=_cu(torch, base))
    want, tol = _adapter_want(x.astype(np.float64), base.astype(np.float64), which, a, b, np.full(n, rank), scales, True)
    assert np.abs(want).max() < 2.0 ** 127
    # numbers below 2^-126 have steps of 2^-149: half a one for y, and one for each rank's t, times its weights
    tol += 2.0 ** -150 + 2.0 ** -149 * (np.abs(scales[which])[:, None] * np.abs(b[which].astype(np.float64)).sum(2))
    got = y.double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) / tol)
    assert (got[:, 7] == 0).all()
