"""Attention of many rows over pages whose values hold infinities and NaN that rows of both tiles of an item see, or rows of one of them, or nobody."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import lib, ok, stream  # noqa: E402
from tests.paged_util import NONE, Cache  # noqa: E402


def spoil(cache, s, places):
    """Value `what` at key `at`, key/value head `h`, column `c` of sequence s, in the pool and in what expected() computes from (keys whose page is gone are nobody's)."""
    for at, h, c, what in places:
        if int(cache.host_table[s, at // cache.page_rows]) == NONE:
            continue
        cache.v_pool[int(cache.host_table[s, at // cache.page_rows]), at % cache.page_rows, h, c] = what
        cache.dense[s][1][at, h, c] = what


def check(cache, got, clean, odd):
    """Against 64 bits: elements that no odd value reaches within the tolerance (to the bit where the row sees none of them), the others of no finite number."""
    want, tol = cache.expected()
    got, finite = got.double(), torch.isfinite(want)
    assert not bool(torch.isfinite(got[~finite]).any())
    off = (got - want).abs()[finite] - tol[finite]
    assert bool(torch.isfinite(got[finite]).all()) and float(off.max()) <= 0
    for s, n in enumerate(cache.lengths):
        for i in range(cache.counts[s]):
            at = n - cache.counts[s] + i
            first = at - cache.window + 1 if cache.window else 0
            if not any(k <= at and (k >= first or k < cache.sinks) for k in odd[s]):
                row = int(cache.starts[s]) + i
                assert torch.equal(got[row].float(), clean[row]), (s, i)


# rows that are multiples of eight and the first columns are reached first by whoever looks through a block
PLACES = [[64, 72, 80, 128, 136, 184, 192, 256], [0, 1, 8, 127, 129], [120, 200, 201, 202, 203, 204, 205, 259]]


@pytest.mark.parametrize("workspace", [None, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("places", range(3))
@pytest.mark.parametrize("heads,kv,dim,page_rows", [(4, 2, 64, 16), (4, 2, 128, 64), (3, 1, 128, 16), (8, 1, 64, 8)])
def test_values_that_rows_of_both_tiles_see(heads, kv, dim, page_rows, places, window, sinks, workspace):
    cache = Cache([260, 203, 131], [200, 203, 1], heads, kv, dim, dim, page_rows, "bf16", seed=places, window=window, sinks=sinks)
    clean = cache.run(workspace).clone()
    odd = [[], [], []]
    for s, n in enumerate(cache.lengths):
        for j, at in enumerate(k for k in PLACES[places] if k < n):
            odd[s].append(at)
            spoil(cache, s, [(at, (j + s) % kv, j % 8, [float("nan"), float("inf"), -float("inf")][j % 3])])
    want = cache.run(workspace).clone()
    check(cache, want, clean, odd)
    for _ in range(10):
        assert torch.equal(cache.run(workspace).nan_to_num(7e30), want.nan_to_num(7e30))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2200, 3)])
def test_values_that_rows_of_both_tiles_see_in_divided_items(dim, window, sinks):
    cache = Cache([3100, 2300], [150, 140], 4, 2, dim, dim, 16, "bf16", seed=8, window=window, sinks=sinks)
    clean = cache.run().clone()
    odd = [[], []]
    for s, n in enumerate(cache.lengths):
        first = n - cache.counts[s]
        edges = [first + 8 - first % 8, first + 64, n - 80, n - 16] + ([first - window + 40 - first % 8, 1] if window else [])
        for j, at in enumerate(edges):
            odd[s].append(at)
            spoil(cache, s, [(at, h, j % 8, [float("nan"), float("inf")][j % 2]) for h in range(2)])
    want = cache.run().clone()
    check(cache, want, clean, odd)
    for _ in range(10):
        assert torch.equal(cache.run().nan_to_num(7e30), want.nan_to_num(7e30))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("many", [16, 17, 60])
def test_more_odd_keys_than_an_items_list_holds(dim, many):
    cache = Cache([300], [260], 4, 2, dim, dim, 16, "bf16", seed=1)
    for at in np.linspace(0, 290, many).astype(int):
        spoil(cache, 0, [(int(at), 0, int(at) % dim, float("nan"))])
    want, tol = cache.expected()
    got = cache.run().double()
    finite = torch.isfinite(want)
    assert not bool(torch.isfinite(got[~finite]).any()) and bool(torch.isfinite(got[finite]).all())
    assert float(((got - want).abs() - tol)[finite].max()) <= 0


@pytest.mark.parametrize("dim", [64, 128])
def test_items_of_one_tile_and_of_two_behind_one_another_with_odd_values_in_turn(dim):
    """Blocks of the grid go through items of one tile, of two, and of none that sees an odd value: no item takes another one's list."""
    counts = [70, 30, 128, 5, 129, 64, 1, 100] * 12
    lengths = [c + (37 * i) % 150 for i, c in enumerate(counts)]
    cache = Cache(lengths, counts, 8, 4, dim, dim, 16, "bf16", seed=3)
    clean = cache.run(None).clone()
    odd = [[] for _ in lengths]
    for s, n in enumerate(lengths):
        if s % 3 == 0:
            at = (n - counts[s] // 2 - 1) // 8 * 8
            odd[s].append(at)
            spoil(cache, s, [(at, h, h, float("inf")) for h in range(4)])
    want = cache.run(None).clone()
    check(cache, want, clean, odd)
    args = cache.args(None)
    for _ in range(20):
        ok(lib().tnsr_b200_paged_attention(C.byref(args), stream()))
    torch.cuda.synchronize()
    assert torch.equal(cache.out[:cache.rows].float().cpu().nan_to_num(7e30), want.nan_to_num(7e30))
