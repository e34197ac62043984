"""Adapters of every rank over rows of several chunks of columns and outputs of several groups of a wave (GPU)."""
import numpy as np
import pytest

from mosship import lib
from test_gpu_serving_ops import U16, _adapter_case, _adapter_want, _cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [16, 32, 64, 80, 128])
@pytest.mark.parametrize("cols,out", [(2208, 1104), (1056, 528), (4096, 48), (32, 2064), (3104, 64)])
@pytest.mark.parametrize("x_dtype,y_dtype", [("float32", "float32"), ("float16", "float16"), ("float32", "float16"), ("float16", "float32")])
def test_ranks_over_chunks_and_groups(torch_gpu, rank, cols, out, x_dtype, y_dtype):
    torch = torch_gpu
    print(f"rank {rank} {cols}->{out} {x_dtype} {y_dtype}", flush=True)
    rng = np.random.default_rng(rank + cols)
    n, rows = 5, 37
    a, b, ranks, scale = _adapter_case(rng, rows, cols, out, rank, n)
    x = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).to(getattr(torch, x_dtype))
    base = torch.from_numpy(rng.standard_normal((rows, out)).astype(np.float32)).to(getattr(torch, y_dtype))
    which = rng.integers(-1, n, rows).astype(np.int32)
    ad = lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale)))
    y = torch.full((rows, out), float("nan"), dtype=base.dtype, device="cuda")
    lib.adapter_rows(x.cuda(), ad, _cu(torch, which), y, base=base.cuda())
    want, tol = _adapter_want(x.double().numpy(), base.double().numpy(), which, a, b, ranks, scale, x_dtype == "float32")
    if y_dtype == "float16":
        tol += U16 * (np.abs(want) + tol) + 2.0 ** -25
    tol[which < 0] = 0  # those rows are copied
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()
