"""The serving-loop operators where byte and element offsets pass 32 bits (GPU)."""
import numpy as np
import pytest

import serving_oracle as so
from mosship import lib
from test_gpu_serving_ops import U16, _adapter_case, _adapter_want, _cu

pytestmark = pytest.mark.gpu


def test_pages_behind_4_gib(torch_gpu):
    """A copy between, and rows moved within, pages that lie behind 4 GiB of a pool, with their scales."""
    torch = torch_gpu
    print("pages behind 4 GiB", flush=True)
    n_pages, heads, page, dim = 70000, 8, 64, 128
    shape = (n_pages, heads, page, dim)
    k, v = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(shape[:3], device="cuda") for _ in range(2))
    assert k.numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(3)
    for t in (k, v):
        t[69000] = torch.randint(-127, 128, shape[1:], generator=g, device="cuda").to(torch.int8)
    for t in (ks, vs):
        t[69000] = torch.rand(shape[1:3], generator=g, device="cuda")
    refs = torch.ones(n_pages, dtype=torch.int32, device="cuda")
    refs[69000], refs[69997] = 2, 0
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    table[:, 1] = 69000
    layers = lib.KVLayers([lib.KVCache(k, v, table, ks, vs)])
    ok = torch.zeros(2, dtype=torch.int32, device="cuda")
    ctx = _cu(torch, np.array([64 + 41, 64 + 41], np.int32))
    lib.kv_reserve(lib.KVPages(table, refs, page), layers, _cu(torch, np.array([0, 20, 40], np.int32)), ctx, ok, 20)
    assert ok.tolist() == [1, 1] and table[:, 1].tolist() == [69997, 69000] and refs[[69000, 69997]].tolist() == [1, 1]
    for t in (k, v, ks, vs):
        assert torch.equal(t[69997, :, :41], t[69000, :, :41]) and not t[69997, :, 41:].any()
        assert not t[:69000].any() and not t[69998:].any()
    # rows 3 and 9 behind 41 positions of the second stream, to places 0 and 1
    was = [t[69000].clone() for t in (k, v, ks, vs)]
    kept = _cu(torch, np.array([-1] * 20 + [3, 9] + [-1] * 18, np.int32))
    lib.kv_compact(layers, _cu(torch, np.array([0, 20, 40], np.int32)), ctx, kept, 20)
    for t, w in zip((k, v, ks, vs), was):
        w[:, [41, 42]] = w[:, [44, 50]].clone()
        assert torch.equal(t[69000], w) and not t[:69000].any() and not t[69998:].any()


@pytest.mark.parametrize("draft", [False, True])
def test_logits_behind_4_gib(torch_gpu, draft):
    """The last of many streams' rows, whose logits lie behind 2^31 elements."""
    torch = torch_gpu
    print(f"logits behind 4 GiB {draft}", flush=True)
    vocab, each, streams = 130001, 5, 3400
    rows = each * streams
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    assert x.numel() > 1 << 31
    look = np.array([0, 1700, 3398, 3399])
    at = np.concatenate([np.arange(s * each, s * each + each) for s in look])
    x[at] = (2.0 * torch.randn(len(at), vocab, generator=g, device="cuda")).half()
    rng = np.random.default_rng(6)
    peak = rng.integers(0, vocab, rows)
    x[torch.from_numpy(np.arange(rows)).cuda(), torch.from_numpy(peak).cuda()] = 17.0
    tok = np.roll(peak, 1).astype(np.int32)  # the likeliest behind the row before
    u = rng.random(rows) * 0.9
    y = None
    if draft:
        y = x.roll(0).contiguous()
        y[at] = (x[at].float() + 0.3 * torch.randn(len(at), vocab, generator=g, device="cuda")).half()
    start = (np.arange(streams + 1) * each).astype(np.int32)
    acc, nxt = (torch.empty(streams, dtype=torch.int32, device="cuda") for _ in range(2))
    path = torch.empty(rows, dtype=torch.int32, device="cuda")
    lib.verify_tokens(x, _cu(torch, tok), _cu(torch, start), acc, path, nxt, each, uniforms=_cu(torch, u), draft_logits=y)
    for s in look:
        r = slice(s * each, s * each + each)
        want, t, near = so.verify_stream(x[r].double().cpu().numpy(), tok[r], u[r], None if y is None else y[r].double().cpu().numpy())
        assert near > 1
        assert path[r].tolist() == want + [-1] * (each - len(want)) and acc[s] == len(want) - 1 and nxt[s] == t


def test_rows_behind_4_gib(torch_gpu):
    """Adapters of rows, bases and outputs behind 2^31 elements."""
    torch = torch_gpu
    print("rows behind 4 GiB", flush=True)
    rows, cols, out, rank, n = 540000, 4096, 4112, 16, 3
    rng = np.random.default_rng(7)
    a, b, ranks, scale = _adapter_case(rng, 0, cols, out, rank, n, mixed=False)
    x = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    y = torch.zeros(rows, out, dtype=torch.float16, device="cuda")
    assert x.numel() > 1 << 31
    look = np.array([0, 17, 524288, 524300, 530001, 539998, 539999])
    x[look], y[look] = (torch.randn(len(look), w, device="cuda").half() for w in (cols, out))
    base = y[look].double().cpu().numpy()
    which = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    which[look] = _cu(torch, (np.arange(len(look)) % n).astype(np.int32))
    lib.adapter_rows(x, lib.Adapters(*(_cu(torch, v) for v in (a, b, ranks, scale))), which, y)
    want, tol = _adapter_want(x[look].double().cpu().numpy(), base, np.arange(len(look)) % n, a, b, ranks, scale, False)
    tol += U16 * (np.abs(want) + tol) + 2.0 ** -25
    assert (np.abs(y[look].double().cpu().numpy() - want) <= tol).all()
    y[look] = 0
    assert not y.any()
