"""Steps whose reserve is refused: what is appended behind it, queued or captured, leaves the caches as they are."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import _KEEP, lib, ok, ptr, stream  # noqa: E402
from tests.paged_util import host, scratch, status_word, u32  # noqa: E402
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


@pytest.mark.parametrize("sequences,rows,page_rows", [(12288, 349526, 1), (12288, 2 * 349526, 2)])
def test_more_pages_are_wanted_than_32_bits_count(sequences, rows, page_rows):
    """12288 x 349526 = 2^32 + 8192 pages of a pool of 10000: refused, and nothing has changed."""
    ld, pool = -(-rows // page_rows), 10000
    assert sequences * ld % (1 << 32) < pool
    table = torch.empty(sequences * ld, dtype=torch.int32, device="cuda")
    lengths, holders, status, word = u32(np.zeros(sequences)), u32(np.zeros(pool)), status_word(), u32([0])
    work = scratch(lib().tnsr_b200_pages_workspace(sequences, pool))
    book = _native.PageBook(table=table.data_ptr(), lengths=lengths.data_ptr(), holders=holders.data_ptr(), workspace=work.data_ptr(), d_status=status.data_ptr(),
                            workspace_bytes=work.numel(), sequences=sequences, table_ld=ld, page_rows=page_rows, pool_pages=pool, refused=word.data_ptr())
    pools = _native.PagePools(count=0)
    ok(lib().tnsr_b200_pages_reserve(C.byref(book), C.byref(pools), None, rows, stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == 5 and host(word).tolist() == [5]
    assert int(lengths.abs().max()) == 0 and int(holders.abs().max()) == 0
    # what there is room for is granted
    status.zero_()
    few = np.zeros(sequences)
    few[[0, 5, sequences - 1]] = [4000 * page_rows, 1, 5999 * page_rows]
    few_rows = u32(few)
    ok(lib().tnsr_b200_pages_reserve(C.byref(book), C.byref(pools), few_rows.data_ptr(), 0, stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == 0 and int(holders.sum()) == 10000 and host(lengths).tolist() == few.astype(int).tolist()
    rows_of = table.view(sequences, ld)
    assert rows_of[0, :4000].tolist() == list(range(4000)) and rows_of[5, 0] == 4000 and rows_of[sequences - 1, :5999].tolist() == list(range(4001, 10000))
    del table, rows_of
    torch.cuda.empty_cache()
