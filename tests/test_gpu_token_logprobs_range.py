"""Log probabilities of rows that span the type's range (GPU), against 64 bits."""
import numpy as np
import pytest

from test_gpu_paged_ops import _check_lp, _run_lp

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [700, 5000, 70001])
@pytest.mark.parametrize("inv_t", [1e-38, 3e-38])
def test_token_logprobs_from_end_to_end(torch_gpu, vocab, inv_t):
    """Logits from the type's lowest value to its largest under a temperature that brings them to a few units: differences
    that pass the type's range count."""
    torch = torch_gpu
    rng = np.random.default_rng(vocab)
    x = (rng.uniform(-1, 1, (4, vocab)) * 3.4e38).astype(np.float32)
    x[0, 5], x[0, 9] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[1] = np.where(np.arange(vocab) % 2, np.finfo(np.float32).max, np.finfo(np.float32).min)
    _check_lp(torch, torch.from_numpy(x).cuda(), [9, 0, vocab - 1, 3], 9, inv_t)


@pytest.mark.parametrize("vocab", [700, 70001])
def test_token_logprobs_one_tiny_and_one_huge(torch_gpu, vocab):
    """The two ends under an ordinary temperature: one token has it all."""
    torch = torch_gpu
    x = np.full((1, vocab), np.finfo(np.float32).min, np.float32)
    x[0, 3] = np.finfo(np.float32).max
    lp, ent, ids, top = _run_lp(torch, torch.from_numpy(x).cuda(), [3], 2)
    assert lp[0] == 0 and ent[0] == 0 and list(ids[0]) == [3, 0] and top[0, 0] == 0 and top[0, 1] == -np.inf
