"""Rows of sequences whose lengths or counts cannot be: none of them is written, those of the others are."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import _KEEP, lib, ok, stream  # noqa: E402
from tests.paged_util import status_word, u32  # noqa: E402
from tnsr_b200 import _native  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [16, 7])
@pytest.mark.parametrize("lengths,starts,chunk,written", [
    ([10, 0xffffffff, 9], [0, 2, 4, 6], 2, [0, 2]),              # longer than its table row names
    ([10, 13, 9], [0, 2, 4, 6], 2, [0, 2]),
    ([10, 12, 9], [0, 1, 5, 6], 2, [0, 2]),                      # four rows of two
    ([10, 12, 9], [0, 1, 2, 600], 3, [0, 1]),                    # more rows than there are, more than a chunk
    ([10, 12, 9], [0, 2, 4, 600], 2, [0, 1, 2]),                 # more rows than there are: the others are a chunk
    ([4000000000, 12, 9], None, 2, [1, 2])])
def test_rows_of_sequences_that_cannot_be_are_left_out(lengths, starts, chunk, written, dim, dtype):
    page_rows, ld, rows, kv = 4, 3, 6, 2
    table = np.array([[8, 1, 5], [2, 7, 0], [3, 6, 4]])
    k_pool, v_pool = (torch.randn(9, page_rows, kv, dim, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(rows, kv, dim, device="cuda").to(dtype) for _ in range(2))
    status = status_word()
    want = [k_pool.clone(), v_pool.clone()]
    place = starts or [0, 2, 4, 6]
    for s in written:
        end = min(place[s + 1], rows)
        for row in range(place[s], end):
            j = lengths[s] - end + row
            want[0][table[s, j // page_rows], j % page_rows], want[1][table[s, j // page_rows], j % page_rows] = k[row], v[row]
    d_table, d_lengths, d_starts = u32(table), u32(np.array(lengths)), u32(np.array(starts)) if starts else None
    _KEEP.extend([k, v, k_pool, v_pool])
    args = _native.PagedAppendArgs(k=k.data_ptr(), v=v.data_ptr(), k_pool=k_pool.data_ptr(), v_pool=v_pool.data_ptr(), table=d_table.data_ptr(),
                                   lengths=d_lengths.data_ptr(), row_starts=d_starts.data_ptr() if starts else None, d_status=status.data_ptr(), sequences=3,
                                   chunk=chunk, rows=rows, k_ld=kv * dim, v_ld=kv * dim, kv_heads=kv, dim=dim, vdim=dim, table_ld=ld, page_rows=page_rows,
                                   pool_pages=9, dtype=0 if dtype == torch.float32 else 1)
    ok(lib().tnsr_b200_paged_append(C.byref(args), stream()))
    torch.cuda.synchronize()
    assert int(status[0]) == (0 if len(written) == 3 else 3)
    assert torch.equal(k_pool, want[0]) and torch.equal(v_pool, want[1])
