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
