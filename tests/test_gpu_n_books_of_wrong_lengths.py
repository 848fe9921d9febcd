"""Books whose lengths name more rows than a table row has entries for: every operator tells it, and touches nothing outside."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import lib, ok, ptr, stream  # noqa: E402
from tests.paged_util import host, u32  # noqa: E402
from tests.test_gpu_h_beam_search import Book  # noqa: E402


@pytest.mark.parametrize("length", [13, 4000000000, 0xffffffff])
@pytest.mark.parametrize("what", ["fork", "release", "compact", "reserve"])
def test_a_length_beyond_its_table_row_is_told(what, length):
    book = Book(3, 3, 4, 20)
    book.reserve([12, 5, 1])
    book.check()
    book.release([1])
    book.check()
    wrong = [length, 0, 1]
    book.lengths.copy_(u32(wrong))
    table, holders = host(book.table), host(book.holders)
    calls = {"fork": lambda: lib().tnsr_b200_pages_fork(C.byref(book.c_book), ptr(u32([0, 1, 2])), stream()),
             "release": lambda: lib().tnsr_b200_pages_release(C.byref(book.c_book), ptr(torch.tensor([1, 0, 0], dtype=torch.uint8, device="cuda")), stream()),
             "compact": lambda: lib().tnsr_b200_pages_compact(C.byref(book.c_book), C.byref(book.c_pools), None, stream()),
             "reserve": lambda: lib().tnsr_b200_pages_reserve(C.byref(book.c_book), C.byref(book.c_pools), None, 1, stream())}
    ok(calls[what]())
    torch.cuda.synchronize()
    assert int(book.status[0]) == 3
    assert host(book.lengths).tolist() == ([0, 0, 1] if what == "release" else wrong)
    if what == "release":               # its three pages are free, and nothing else is
        holders[table[0, :3]] -= 1
    if what == "compact":               # page 5 moves to 3
        assert table[0, :3].tolist() == [0, 1, 2] and table[2, 0] == 5
        table[2, 0], holders[3], holders[5] = 3, 1, 0
    assert host(book.table).tolist() == table.tolist() and host(book.holders).tolist() == holders.tolist()
