"""Steps whose reserve is refused: what is appended behind it, queued or captured, leaves the caches as they are."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import _KEEP, lib, ok, ptr, stream  # noqa: E402
from tests.paged_util import host, u32  # noqa: E402
from tests.test_gpu_h_beam_search import Book  # noqa: E402
from tnsr_b200 import _native  # noqa: E402

KV, DIM = 2, 8


def appends(book, refused):
    """A step's new rows, one per sequence, into the book's two pools as keys and values in f32."""
    t = [torch.randn(book.s, KV, DIM, device="cuda") for _ in range(2)]
    _KEEP.extend(t)
    return t, _native.PagedAppendArgs(
        k=t[0].data_ptr(), v=t[1].data_ptr(), k_pool=book.pools[0].data_ptr(), v_pool=book.pools[1].data_ptr(), table=book.table.data_ptr(),
        lengths=book.lengths.data_ptr(), d_status=book.status.data_ptr(), sequences=book.s, chunk=1, rows=book.s, k_ld=KV * DIM, v_ld=KV * DIM, kv_heads=KV, dim=DIM,
        vdim=DIM, table_ld=book.ld, page_rows=book.r, pool_pages=book.pool, dtype=0, refused=refused)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("why", ["no pages", "full row"])
def test_rows_behind_a_refused_reserve_are_not_written(why, captured):
    page_rows = 4
    book = Book(4, 2 if why == "full row" else 6, page_rows, 5 if why == "no pages" else 20, (page_rows * KV * DIM * 4,) * 2)
    word = u32([77])
    book.c_book.refused = ptr(word)
    book.reserve([6, 0, 0, 0] if why == "no pages" else [8, 3, 0, 0])
    book.check()
    assert host(word).tolist() == [0]
    book.fork([0, 0, 0, 0] if why == "no pages" else [0, 1, 1, 1])      # all four hold the last page
    book.check()
    if why == "no pages":
        book.release([])
        book.reserve([4, 0, 0, 0])                                         # a copy and one page more: of the other three beams two need a copy, and one page is free
        book.check()
    rows, args = appends(book, word.data_ptr())
    before = [p.clone() for p in book.pools]
    table, lengths, holders = (x.clone() for x in (book.table, book.lengths, book.holders))

    def step():
        ok(lib().tnsr_b200_pages_reserve(C.byref(book.c_book), C.byref(book.c_pools), None, 1, stream()))
        ok(lib().tnsr_b200_paged_append(C.byref(args), stream()))

    graph = None
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step()
    for _ in range(2):
        graph.replay() if captured else step()
        torch.cuda.synchronize()
        code = 5 if why == "no pages" else 3
        assert int(book.status[0]) == code and host(word).tolist() == [code]
        assert all(torch.equal(a, b) for a, b in zip(book.pools, before))
        assert torch.equal(book.table, table) and torch.equal(book.lengths, lengths) and torch.equal(book.holders, holders)
    # room again: the same step is granted, and its rows are there
    book.status.zero_()
    book.release([0] if why == "full row" else [0, 1])
    graph.replay() if captured else step()
    torch.cuda.synchronize()
    assert int(book.status[0]) == 0 and host(word).tolist() == [0]
    table, lengths = host(book.table), host(book.lengths)
    assert lengths.tolist() == ([1, 4, 4, 4] if why == "full row" else [1, 1, 7, 7])
    for pool, fresh in zip(book.pools, rows):
        pool = pool.view(torch.float32).view(book.pool, page_rows, KV, DIM)
        for s in range(book.s):
            at = int(lengths[s]) - 1
            assert torch.equal(pool[int(table[s, at // page_rows]), at % page_rows], fresh[s])


def test_the_word_is_optional_and_follows_the_last_reserve():
    book = Book(2, 2, 4, 3, (16,))
    word = u32([9])
    book.reserve(1)
    book.check()
    book.c_book.refused = ptr(word)
    book.reserve([8, 0], status=3)
    book.check(status=3)
    assert host(word).tolist() == [3]
    book.reserve([0, 0])
    book.check()
    assert host(word).tolist() == [0]
    book.reserve([4, 4], status=5)
    book.check(status=5)
    assert host(word).tolist() == [5]
    table = host(book.table)
    table[1, 0] = 3
    book.table.copy_(u32(table))
    ok(lib().tnsr_b200_pages_reserve(C.byref(book.c_book), C.byref(book.c_pools), None, 1, stream()))
    torch.cuda.synchronize()
    assert host(word).tolist() == [4] and int(book.status[0]) == 4
