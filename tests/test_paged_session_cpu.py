"""session.PagedBatch hands the library what its arguments say, or refuses them: on the CPU, where the library answers -1 for want of a context."""
import os

import numpy as np
import pytest

import hipsupport as H

pkg = H.load_package()
from voxtral_tts_c_amd.session import PagedBatch                                        # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(pkg.LIB_PATH), reason="library not built (run __graft_entry__.build())")


@pytest.fixture
def batch():
    b = PagedBatch(10, 16, 32, 8, 128, max_seqs=3, max_rows=64, max_table=10)
    yield b
    b.free()


@pytest.mark.parametrize("past,rows,tables", [
    ([3, 4], [1], [[1], [2]]), ([3], [1, 1], [[1]]), ([3, 4], [1, 1], [[1]]), ([3], [1], []), ([], [1], []), ([3], [1], [[1], [2]]),
    ([[3]], [1], [[1]]), (3, [1], [[1]]), ([3], [1], [[[1]]]),
    (np.array([1 << 32]), [1], [[1]]), ([3], np.array([(1 << 32) + 1]), [[1]]), ([3], [1], [np.array([(1 << 32) + 1])]), ([3], [1], [[1 << 40]]),
    ([3], [1], [np.array([2 ** 64 - 1], np.uint64)]), ([3.5], [1], [[1]]), ([float("nan")], [1], [[1]]), (["three"], [1], [[1]])])
def test_what_does_not_fit_is_refused(batch, past, rows, tables):
    n = batch.lib.tts_hip_error_count()
    with pytest.raises(ValueError):
        batch.set(past, rows, tables)
    assert batch.lib.tts_hip_error_count() == n                                         # the library was not asked


@pytest.mark.parametrize("past,rows,tables", [
    ([3, 4], [1, 1], [[1], [2, 3]]), ((3,), (1,), ((1,),)), (np.array([3], np.int64), np.array([1], np.uint8), np.array([[1]], np.int64)), ([], [], []),
    ([3, 0], [1, 0], [[1], []])])
def test_the_library_is_asked_for_the_others(batch, past, rows, tables, monkeypatch):
    asked = []

    class Lib:
        def tts_hip_paged_set(self, ptr, n, past, rows, tables, stride):
            read = lambda p, k: np.ctypeslib.as_array((np.ctypeslib.ctypes.c_int * k).from_address(p)).tolist() if k else []
            asked.append((ptr, n, read(past, n), read(rows, n), [r[:stride] for r in np.array(read(tables, n * stride)).reshape(n, stride).tolist()]))
            return 0

    monkeypatch.setattr(batch, "lib", Lib())
    ptr = batch.ptr
    assert batch.set(past, rows, tables) == 0
    (p, n, some_past, some_rows, some_tables), = asked
    assert p == ptr and n == len(past) and some_past == [int(x) for x in past] and some_rows == [int(x) for x in rows]
    for got, t in zip(some_tables, tables):
        assert got == [int(x) for x in t] + [-1] * (len(got) - len(t))
    monkeypatch.undo()
