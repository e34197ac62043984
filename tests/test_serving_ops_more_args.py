"""Sizes and limits of the serving-loop operators that the host decides, without a GPU."""
import ctypes as C

import pytest

from mosship import lib

P = 0x1000  # a 16-byte aligned address that no refused call may touch
INT_MAX = 2 ** 31 - 1


def _reserve_bytes(streams, stride, page, max_rows):
    pages, n = lib.KVPagesStruct(page_table=P, table_stride=stride, streams=streams, refs=P, n_pages=8, page_size=page), C.c_size_t()
    assert lib.load().moss_hip_kv_reserve_workspace(C.addressof(pages), max_rows, C.byref(n)) == lib.OK
    return n.value


@pytest.mark.parametrize("streams,stride,page,max_rows", [
    (1, 1 << 26, 32768, INT_MAX), (1, 1 << 26, 32768, INT_MAX - 32766), (1, 1 << 26, 32768, INT_MAX - 32765), (1, 1 << 26, 32, INT_MAX),
    (3, 1 << 24, 128, INT_MAX), (65536, 1024, 16, 16384), (65536, 1024, 16, 1023 * 16), (5, 4, 16, 20), (1, 1, 16, 16), (7, 3, 48, 144)])
def test_reserve_workspace_of_many_rows(streams, stride, page, max_rows):
    """A copy's place per stream and, for more than 1024 entries, two ints per entry: a stream's rows touch as many pages as max_rows
    positions from the last of a page on do, and no more than its table has."""
    entries = streams * min((max_rows - 1 + page - 1) // page + 1, stride)
    assert _reserve_bytes(streams, stride, page, max_rows) == 16 * streams + (8 * entries if entries > 1024 else 0)


def _verify_bytes(streams, max_rows, vocab, draft):
    n = C.c_size_t()
    assert lib.load().moss_hip_verify_tokens_workspace(streams, max_rows, vocab, draft, C.byref(n)) == lib.OK
    return n.value


@pytest.mark.parametrize("vocab", [1, 1000, 1024, 1025, 4000, 5000, 16384, 16385, 33000, 65537, 130001])
def test_verify_workspace_of_smaller_calls(vocab):
    """What is enough for some streams and rows is enough for fewer of them, across the sizes where rows are cut finer (1024 pieces of all
    rows) or fit one launch (32 pieces of a stream), and with a draft also without."""
    sizes = {(s, r): [_verify_bytes(s, r, vocab, d) for d in (0, 1)]
             for s in [*range(1, 40), 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 341, 342, 512, 513, 1024, 1025, 4096, 65536]
             for r in [*range(1, 33), 40, 63, 64] if s * r * vocab <= 1 << 34}
    grid = sorted(sizes)
    for s, r in grid:
        for (s2, r2) in ((s, max((x for y, x in grid if y == s and x < r), default=r)), (max((y for y, x in grid if x == r and y < s), default=s), r)):
            assert all(a <= b for a, b in zip(sizes[s2, r2], sizes[s, r])), (s2, r2, s, r)
        assert sizes[s, r][0] <= sizes[s, r][1]


def test_verify_takes_the_workspace_of_a_larger_batch():
    """A call of fewer streams under the bytes for all of them passes the check of its workspace: what refuses it is named behind that."""
    L = lib.load()
    for vocab, most, rows in ((16384, 11, 6), (16384, 17, 4), (5000, 40, 12)):
        have = _verify_bytes(most, rows, vocab, 1)
        for streams in range(1, most + 1):
            for max_rows in range(1, rows + 1):
                if _verify_bytes(streams, max_rows, vocab, 1) == 0:
                    continue  # (one launch holds all of it: nothing would refuse the call)
                rc = L.moss_hip_verify_tokens(P, vocab, lib.F32, P, vocab, 8, vocab, P, P, None, streams, max_rows, P, 1.0, 1.0, 0, P, P, P, P + 8,
                                              have, None)
                assert rc == lib.EINVAL and "aligned" in L.moss_hip_last_error().decode(), (streams, max_rows)
