"""Attention over caches in pages and the rows appended to them, against a plain implementation in 64 bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import _KEEP, lib, ok, stream  # noqa: E402
from tests.paged_util import DTYPES, NONE, Cache, scratch, status_word, u32  # noqa: E402
from tnsr_b200 import _native  # noqa: E402

# heads, kv_heads, dim, vdim, page_rows
SHAPES = [(1, 1, 64, 64, 16), (4, 4, 64, 64, 16), (8, 2, 128, 128, 16), (6, 2, 64, 64, 24), (5, 1, 80, 80, 7), (12, 1, 32, 64, 32), (3, 3, 96, 40, 1),
          (2, 1, 256, 256, 64), (40, 2, 64, 64, 16), (4, 2, 128, 64, 128), (2, 2, 7, 9, 5), (2, 1, 36, 100, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_new_token_per_sequence(shape, dtype):
    lengths = [1, 300, 0, 16, 17, 63, 64, 65, 129, 2]
    cache = Cache(lengths, [1] * len(lengths), *shape, dtype, seed=sum(shape), uniform=True)
    cache.check(cache.run())
    assert float(cache.out[2].abs().max()) == 0.0                # no keys: zeros


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(4, 4, 64, 64, 16), (8, 2, 128, 128, 16), (5, 1, 80, 80, 7), (2, 2, 7, 9, 5)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (64, 4), (33, 70), (200, 0), (1000, 3)])
def test_one_new_token_behind_a_window_and_sinks(shape, dtype, window, sinks):
    lengths = [1, 5, 70, 300, 0, 411, 64, 65]
    cache = Cache(lengths, [1] * len(lengths), *shape, dtype, seed=window + sinks, window=window, sinks=sinks, uniform=True)
    cache.check(cache.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(4, 4, 64, 64, 16), (8, 2, 128, 128, 16), (6, 1, 80, 80, 24)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2), (100, 5)])
def test_a_few_rows_per_sequence_some_of_them_without_keys(shape, dtype, window, sinks):
    # counts of 0, rows before the first key, chunks of the whole length, rows of no sequence at the end
    lengths, counts = [300, 3, 5, 0, 77, 12, 130], [3, 5, 5, 2, 0, 1, 7]
    cache = Cache(lengths, counts, *shape, dtype, seed=3, window=window, sinks=sinks, extra_rows=2)
    got = cache.run()
    cache.check(got)
    assert float((got[-2:] + 7).abs().max()) == 0.0             # rows behind the last sequence stay as they were


@pytest.mark.parametrize("shape", [(4, 4, 64, 64, 16), (8, 2, 128, 128, 16), (16, 4, 64, 64, 64), (6, 2, 128, 128, 24), (3, 1, 80, 80, 32), (5, 5, 64, 64, 8),
                                   (8, 1, 96, 128, 48), (2, 1, 160, 160, 16), (4, 2, 64, 64, 5)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (130, 129), (300, 0)])
def test_prompts_of_ragged_rows(shape, window, sinks):
    lengths, counts = [200, 129, 500, 64, 30, 257], [200, 128, 131, 64, 40, 1]
    cache = Cache(lengths, counts, *shape, "bf16", seed=window + 1, window=window, sinks=sinks, extra_rows=3)
    got = cache.run()
    cache.check(got)
    assert float((got[-3:] + 7).abs().max()) == 0.0


@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 4)])
def test_long_prompts(window, sinks):
    cache = Cache([1500, 900], [700, 900], 2, 1, 128, 128, 64, "bf16", seed=9, window=window, sinks=sinks)
    cache.check(cache.run())
    cache = Cache([1111], [777], 4, 4, 64, 64, 16, "bf16", seed=10, window=window, sinks=sinks)
    cache.check(cache.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [7, 2, 11], [140, 60, 40]])
def test_windows_as_long_as_a_sequence_or_longer_than_any_position(counts, dtype):
    cache = Cache([210, 100, 77], counts, 4, 2, 64, 64, 16, dtype, seed=12)
    want = cache.run()
    cache.check(want)
    for window, sinks in ((211, 0), (256, 5), (0x7fffffff, 1), (0x80000000, 0), (0x80000003, 0xffffffff), (NONE, 3)):
        assert torch.equal(cache.run(window=window, sinks=sinks), want) or window == 211, window
        cache.check(cache.run(window=window, sinks=sinks))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 0, 1], [7, 2, 11], [140, 60, 40]])
def test_bounds_on_a_sequences_rows_that_are_far_above_them(counts, dtype):
    cache = Cache([210, 100, 77], counts, 4, 2, 64, 64, 16, dtype, seed=16, extra_rows=2)
    for chunk in (cache.rows, 1 << 20, NONE):
        cache.out.fill_(-7.0)
        got = cache.run(chunk=chunk)
        cache.check(got)
        assert float((got[-2:] + 7).abs().max()) == 0.0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
@pytest.mark.parametrize("shape", [(4, 2, 64, 64, 16), (2, 1, 160, 160, 16), (2, 2, 7, 9, 5)])
def test_scales_of_zero_and_below(shape, scale, dtype):
    cache = Cache([210, 100, 3], [70, 1, 5], *shape, dtype, seed=13)
    cache.scale = scale
    cache.check(cache.run())


def test_prompts_in_32_bits():
    cache = Cache([200, 129, 300], [200, 100, 31], 4, 2, 64, 64, 16, "f32", seed=1, window=50, sinks=2)
    cache.check(cache.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["heads", "gaps"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [150, 3, 90]])
def test_strides_of_pools_and_rows(dtype, layout, counts):
    cache = Cache([210, 100, 333], counts, 4, 2, 64, 64, 16, dtype, seed=2, layout=layout, pad=16)
    got = cache.run()
    cache.check(got[:, :cache.out_ld])
    # pitches and addresses that 16-byte copies cannot take
    cache = Cache([210, 100, 333], counts, 4, 2, 64, 64, 16, dtype, seed=2, layout=layout, pad=3)
    cache.check(cache.run())


def test_addresses_that_are_no_multiple_of_16_bytes():
    for counts in ([1, 1], [100, 70]):
        cache = Cache([210, 100], counts, 4, 2, 64, 64, 16, "bf16", seed=2)
        want = cache.run()
        room = torch.empty(cache.k_pool.numel() + 1, dtype=torch.bfloat16, device="cuda")
        room[1:] = cache.k_pool.reshape(-1)
        got = cache.run(k_pool=room.data_ptr() + 2)
        cache.check(got)
        _KEEP.append(room)
        assert float((got - want).abs().max()) <= 2 ** -7 * float(want.abs().max())


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("counts", [[1, 2], [3, 5], [140, 200]])
def test_what_is_hidden_from_a_row_does_not_reach_it(dim, counts):
    """NaN and infinity in keys and values that later rows see, and the type's lowest value in keys."""
    lengths = [150, 260]
    cache = Cache(lengths, counts, 4, 2, dim, dim, 16, "bf16", seed=5)
    clean = cache.run().clone()
    last = [n - 1 for n in lengths]
    table = cache.host_table
    for s, j in enumerate(last):
        page, r = int(table[s, j // 16]), j % 16
        cache.v_pool[page, r, 0, 3], cache.v_pool[page, r, 1, 5] = float("nan"), float("inf")
        cache.k_pool[page, r, 0] = torch.finfo(torch.bfloat16).min
        cache.k_pool[page, r, 1, 0] = float("nan")
    got = cache.run()
    for s in range(2):
        hidden = slice(int(cache.starts[s]), int(cache.starts[s + 1]) - 1)
        assert torch.equal(got[hidden], clean[hidden])
    # the last rows see them: head group 1 has a NaN score
    for s in range(2):
        assert bool(torch.isnan(got[int(cache.starts[s + 1]) - 1].view(4, dim)[2:]).all())


def test_keys_far_behind_in_a_pool_of_more_than_4_billion_values():
    heads, dim, page_rows = 2, 128, 64
    pages = (1 << 32) // (page_rows * heads * dim) + 40
    for counts in ([1, 1], [100, 33]):
        cache = Cache([150, 200], counts, 4, heads, dim, dim, page_rows, "bf16", seed=4, spare=0)
        far = np.where(cache.host_table == NONE, NONE, pages - 1 - cache.host_table.astype(np.int64)).astype(np.uint32)
        k, v = (torch.empty((pages, page_rows, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        k[pages - cache.pool_pages:] = cache.k_pool.flip(0)
        v[pages - cache.pool_pages:] = cache.v_pool.flip(0)
        cache.check(cache.run(k_pool=k.data_ptr(), v_pool=v.data_ptr(), table=u32(far).data_ptr(), pool_pages=pages))
        del k, v
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1] * 5, [2, 1, 3, 2, 2], [80, 33, 70, 90, 64]])
def test_bad_tables_and_lengths_are_reported_and_nothing_outside_is_read(dtype, counts):
    cache = Cache([100, 90, 70, 333, 64], counts, 4, 2, 64, 64, 16, dtype, seed=8)
    good = cache.run().clone()
    table = cache.host_table.copy()
    table[1, 2], table[3, 0] = cache.pool_pages, NONE - 5
    got = cache.run(status=4, table=u32(table).data_ptr())
    for s in (0, 2, 4):
        rows = slice(int(cache.starts[s]), int(cache.starts[s + 1]))
        assert torch.equal(got[rows], good[rows])
    assert bool(torch.isfinite(got).all())
    cache.status.zero_()
    lengths = np.array(cache.lengths, np.uint32)
    lengths[2] = 0xfffffff0
    table = cache.host_table.copy()
    table[2] = 0
    got = cache.run(status=3, lengths=u32(lengths).data_ptr(), table=u32(table).data_ptr())
    # where keys are cut, and with it the last bits, follows all lengths: within the tolerance, not to the bit
    want, tol = cache.expected()
    assert bool(((got.double() - want).abs() <= tol)[:int(cache.starts[2])].all())


def test_row_starts_that_lie_are_cut_to_the_rows_there_are():
    cache = Cache([100, 90, 70], [1, 2, 1], 4, 2, 64, 64, 16, "bf16", seed=8)
    good = cache.run().clone()
    # the last sequence claims rows past the end, more of them than a chunk
    got = cache.run(row_starts=u32([0, 1, 3, 50]).data_ptr())
    assert torch.equal(got, good)
    cache.run(status=3, row_starts=u32([0, 0, 4, 4]).data_ptr())        # four rows, chunk 2
    cache.status.zero_()
    cache.run(row_starts=u32([3, 2, 1, 0]).data_ptr())                   # backwards: nobody has rows


@pytest.mark.parametrize("counts", [[1] * 6, [4, 1, 2, 3, 1, 5], [70, 100, 5, 130, 64, 33]])
def test_same_bits_again_on_another_stream_in_a_graph_and_with_a_used_workspace(counts):
    cache = Cache([1200, 333, 20, 800, 64, 129], counts, 8, 2, 128, 128, 16, "bf16", seed=6, window=300, sinks=4)
    work = scratch(lib().tnsr_b200_paged_attention_workspace(128, 128, 1))
    want = cache.run(work).clone()
    cache.check(want)
    cache.out.fill_(-7.0)
    assert torch.equal(cache.run(work), want)
    cache.out.fill_(-7.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(cache.run(work), want)
    cache.out.fill_(-7.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    args = cache.args(work)
    with torch.cuda.graph(graph):
        ok(lib().tnsr_b200_paged_attention(C.byref(args), stream()))
    for _ in range(3):
        cache.out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.out[:cache.rows].float().cpu(), want)
    # undivided: sums in another order
    cache.out.fill_(-7.0)
    cache.check(cache.run(None))


@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_behind_one_another_whose_items_have_one_tile_or_two(dim):
    """Calls on two caches in turn, without waiting: blocks of the grid go from items of one tile to items of two, on shared memory of all kinds of contents."""
    caches = [Cache([1664, 512, 1280, 896, 2048], [259, 388, 648, 518, 777], 8, 2, dim, dim, 64, "bf16", seed=5, window=512, sinks=4),
              Cache([100, 400, 90], [100, 70, 33], 4, 4, dim, dim, 16, "bf16", seed=6)]
    want = [c.run().clone() for c in caches]
    caches[1].check(want[1])
    calls = [c.args() for c in caches]
    for _ in range(30):
        for c in caches:
            c.out.fill_(-7.0)
        for args in calls:
            ok(lib().tnsr_b200_paged_attention(C.byref(args), stream()))
        torch.cuda.synchronize()
        for c, w in zip(caches, want):
            assert torch.equal(c.out[:c.rows].float().cpu(), w)


# few prompts over long caches: the last round's keys are divided over the blocks, and a tile's parts joined
@pytest.mark.parametrize("shape", [(4, 2, 64, 64, 16), (2, 1, 128, 128, 64), (6, 2, 96, 40, 24)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1900, 5), (2047, 300)])
def test_few_prompts_over_long_caches(shape, window, sinks):
    cache = Cache([3000, 1700, 50, 2500], [100, 70, 60, 130], *shape, "bf16", seed=window + 2, window=window, sinks=sinks, extra_rows=2)
    got = cache.run()
    cache.check(got)
    assert float((got[-2:] + 7).abs().max()) == 0.0
    cache = Cache([2600, 40, 130], [150, 150, 150], *shape, "bf16", seed=window + 3, window=window, sinks=sinks, uniform=True)
    cache.check(cache.run())


@pytest.mark.parametrize("dim", [64, 128])
def test_few_prompts_over_long_caches_hide_what_is_hidden(dim):
    cache = Cache([3100, 2300], [90, 140], 4, 2, dim, dim, 16, "bf16", seed=8, window=2200, sinks=3)
    clean = cache.run().clone()
    table = cache.host_table
    seen = [[], []]
    for s, n in enumerate(cache.lengths):
        first = n - cache.counts[s]                  # position of the first new row: its window begins 2200 keys before
        for at in (n - 1, n - 30, first - 2200 + 20):
            if at < 3:
                continue
            page, r = int(table[s, at // 16]), at % 16
            cache.v_pool[page, r, 0, 3], cache.v_pool[page, r, 1, 5] = float("nan"), float("inf")
            seen[s].append(at)
    got = cache.run()
    for s, n in enumerate(cache.lengths):
        for i in range(cache.counts[s]):
            row, at = int(cache.starts[s]) + i, n - cache.counts[s] + i
            sees = any(j <= at and j > at - 2200 for j in seen[s])
            a, b = got[row].view(4, dim), clean[row].view(4, dim)
            if not sees:
                assert torch.equal(a, b), (s, i)
                continue
            # a value of NaN, or of infinity (its weight may have become 0, which makes NaN of it)
            assert bool(torch.isnan(a[:2, 3]).all()) and not bool(torch.isfinite(a[2:, 5]).any()), (s, i)
            others = [c for c in range(dim) if c not in (3, 5)]
            assert bool(torch.isfinite(a[:, others]).all()) and float((a[:, others] - b[:, others]).abs().max()) < 0.05


def test_few_prompts_over_long_caches_again_in_a_graph_and_behind_single_tokens():
    cache = Cache([3000, 1700, 50], [100, 70, 60], 8, 2, 128, 128, 16, "bf16", seed=14, window=0)
    tokens = Cache([700, 90], [1, 1], 8, 2, 128, 128, 16, "bf16", seed=15, uniform=True)
    work = scratch(lib().tnsr_b200_paged_attention_workspace(128, 128, 1))
    want, want_tokens = cache.run(work).clone(), tokens.run(work).clone()
    cache.check(want)
    tokens.check(want_tokens)
    graph = torch.cuda.CUDAGraph()
    args, token_args = cache.args(work), tokens.args(work)
    with torch.cuda.graph(graph):
        for _ in range(2):
            ok(lib().tnsr_b200_paged_attention(C.byref(args), stream()))
            ok(lib().tnsr_b200_paged_attention(C.byref(token_args), stream()))
    for _ in range(3):
        cache.out.fill_(-7.0)
        tokens.out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.out[:cache.rows].float().cpu(), want)
        assert torch.equal(tokens.out[:tokens.rows].float().cpu(), want_tokens)
    # the captured call follows its lengths: shorter ones, and back
    lengths = cache.d_lengths.clone()
    for smaller in ([1200, 900, 50], [100, 70, 60]):
        cache.d_lengths.copy_(u32(np.array(smaller)))
        graph.replay()
        torch.cuda.synchronize()
        # all but the rows behind the third sequence's 50 keys, whose places in the pool hold NaN
        assert int(cache.status[0]) == 0 and bool(torch.isfinite(cache.out[:int(cache.starts[2]) + 50].float()).all())
    cache.d_lengths.copy_(lengths)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cache.out[:cache.rows].float().cpu(), want)
    cache.out.fill_(-7.0)
    cache.check(cache.run(None))


def test_many_sequences_and_one_long_one_beside_short_ones():
    rng = np.random.default_rng(0)
    lengths = list(rng.integers(0, 40, 700)) + [5000]
    cache = Cache(lengths, [1] * len(lengths), 4, 1, 64, 64, 16, "bf16", seed=12, uniform=True)
    cache.check(cache.run())


# ---- appended rows -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,dim,vdim,page_rows,pad", [(2, 64, 64, 16, 0), (1, 7, 9, 5, 1), (4, 128, 32, 24, 16), (3, 20, 20, 1, 3)])
@pytest.mark.parametrize("layout", ["rows", "heads"])
def test_rows_are_appended_to_their_pages_and_nothing_else_changes(dtype, kv, dim, vdim, page_rows, pad, layout):
    lengths, counts = [100, 3, 40, 17, 5], [4, 3, 0, 17, 1]
    cache = Cache(lengths, counts, kv, kv, dim, vdim, page_rows, dtype, seed=1, layout=layout, extra_rows=2)
    t = DTYPES[dtype]
    k = torch.randn(cache.rows, kv * dim + pad, device="cuda").to(t)
    v = torch.randn(cache.rows, kv * vdim + pad, device="cuda").to(t)
    want_k, want_v = cache.k_pool.clone(), cache.v_pool.clone()
    for s, n in enumerate(lengths):
        for i in range(counts[s]):
            j, row = n - counts[s] + i, int(cache.starts[s]) + i
            for want, new, width in ((want_k, k, dim), (want_v, v, vdim)):
                at = want[int(cache.host_table[s, j // page_rows])]
                (at[j % page_rows] if layout == "rows" else at[:, j % page_rows]).copy_(new[row, :kv * width].view(kv, width))
    status = status_word()
    fields = dict(k=k.data_ptr(), v=v.data_ptr(), k_pool=cache.k_pool.data_ptr(), v_pool=cache.v_pool.data_ptr(), table=cache.table.data_ptr(),
                  lengths=cache.d_lengths.data_ptr(), row_starts=cache.d_starts.data_ptr(), d_status=status.data_ptr(), sequences=len(lengths),
                  chunk=cache.chunk, rows=cache.rows, k_ld=kv * dim + pad, v_ld=kv * vdim + pad, kv_heads=kv, dim=dim, vdim=vdim,
                  table_ld=cache.table_ld, page_rows=page_rows, pool_pages=cache.pool_pages, dtype=_native.DTYPE[dtype])
    fields.update(zip(("k_page", "k_row", "k_head", "v_page", "v_row", "v_head"), cache.strides))

    def same(x, y):
        return torch.equal(x.view(torch.int32 if dtype == "f32" else torch.int16), y.view(torch.int32 if dtype == "f32" else torch.int16))

    ok(lib().tnsr_b200_paged_append(C.byref(_native.PagedAppendArgs(**fields)), stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    assert same(cache.k_pool, want_k) and same(cache.v_pool, want_v)
    # a page outside the pool, and a sequence shorter than the rows it brings: left out and reported
    table = cache.host_table.copy()
    table[0] = cache.pool_pages
    fields["table"] = u32(table).data_ptr()
    ok(lib().tnsr_b200_paged_append(C.byref(_native.PagedAppendArgs(**fields)), stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == 4
    status.zero_()
    fields["table"], fields["lengths"] = cache.table.data_ptr(), u32([100, 2, 40, 17, 5]).data_ptr()
    ok(lib().tnsr_b200_paged_append(C.byref(_native.PagedAppendArgs(**{**fields, "row_starts": u32([0, 0, 3, 3, 3, 3]).data_ptr()})), stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == 3
