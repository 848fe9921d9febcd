"""What the operators of beam search and of caches in pages refuse, before any work on a device."""
import ctypes as C

import pytest

from tnsr_b200 import _native


@pytest.fixture(scope="module")
def library():
    from tnsr_b200 import build
    build.build()
    return _native.lib()


SOME = 0x1000        # an address that no refused call follows


def refuses(code, word, want=-1):
    assert code == want and word in _native.last_error(None), (code, _native.last_error(None))


def beam(**over):
    fields = dict(logits=SOME, scores=SOME, next_scores=SOME, tokens=SOME, parents=SOME, workspace=SOME, workspace_bytes=1 << 40, logits_ld=100, groups=2,
                  beams=4, vocab=100, keep=4, end_token=1, dtype=0)
    return _native.BeamSelectArgs(**{**fields, **over})


def test_selection_refuses(library):
    call = library.tnsr_b200_beam_select
    refuses(call(None, None), "null pointer")
    for name in ("logits", "scores", "next_scores", "tokens", "parents", "workspace"):
        refuses(call(C.byref(beam(**{name: None})), None), "null pointer")
    for over in (dict(beams=0), dict(beams=33), dict(keep=0), dict(keep=65), dict(vocab=0, logits_ld=0), dict(vocab=(1 << 26) + 1, logits_ld=1 << 27), dict(logits_ld=99),
                 dict(beams=1, vocab=3, keep=4), dict(groups=1 << 30)):
        refuses(call(C.byref(beam(**over)), None), "beams")
    refuses(call(C.byref(beam(dtype=2)), None), "dtype")
    need = library.tnsr_b200_beam_select_workspace(2, 4, 100, 4)
    assert need > 0
    refuses(call(C.byref(beam(workspace_bytes=need - 1)), None), "workspace")
    refuses(call(C.byref(beam(workspace=SOME + 8)), None), "workspace")
    assert call(C.byref(beam(groups=0)), None) == 0


def test_states_refuse(library):
    call = library.tnsr_b200_reorder_states
    one, size = (C.c_void_p * 1)(SOME), (C.c_uint64 * 1)(16)
    refuses(call(one, size, size, 1, None, 2, 4, None, None), "null pointer")
    refuses(call(None, size, size, 1, SOME, 2, 4, None, None), "null pointer")
    refuses(call((C.c_void_p * 1)(None), size, size, 1, SOME, 2, 4, None, None), "null")
    refuses(call(one, size, (C.c_uint64 * 1)(15), 1, SOME, 2, 4, None, None), "overlap")
    refuses(call(one, size, size, 1, SOME, 2, 0, None, None), "1 to 32")
    refuses(call(one, size, size, 1, SOME, 2, 33, None, None), "1 to 32")
    assert call(None, None, None, 0, SOME, 2, 4, None, None) == 0
    assert call(one, size, size, 1, SOME, 0, 4, None, None) == 0


def book(**over):
    fields = dict(table=SOME, lengths=SOME, holders=SOME, workspace=SOME, workspace_bytes=1 << 40, sequences=4, table_ld=8, page_rows=16, pool_pages=32)
    return _native.PageBook(**{**fields, **over})


def pools(**over):
    fields = dict(tensors=(C.c_void_p * 1)(SOME), page_bytes=(C.c_uint64 * 1)(64), count=1)
    return _native.PagePools(**{**fields, **over})


def test_books_refuse(library):
    calls = {"fork": lambda b: library.tnsr_b200_pages_fork(b, SOME, None),
             "reserve": lambda b: library.tnsr_b200_pages_reserve(b, C.byref(pools()), None, 1, None),
             "release": lambda b: library.tnsr_b200_pages_release(b, SOME, None),
             "compact": lambda b: library.tnsr_b200_pages_compact(b, C.byref(pools()), None, None)}
    need = library.tnsr_b200_pages_workspace(4, 32)
    for name, call in calls.items():
        refuses(call(None), name)
        for field in ("table", "lengths", "holders"):
            refuses(call(C.byref(book(**{field: None}))), "null pointer")
        for over in (dict(table_ld=0), dict(page_rows=0), dict(pool_pages=0), dict(pool_pages=1 << 30)):
            refuses(call(C.byref(book(**over))), "positive")
        refuses(call(C.byref(book(sequences=12289))), "12288")
        if name != "release":
            refuses(call(C.byref(book(workspace=None))), "null pointer")
            refuses(call(C.byref(book(workspace_bytes=need - 1))), "workspace")
            refuses(call(C.byref(book(workspace=SOME + 4))), "workspace")
    refuses(library.tnsr_b200_pages_fork(C.byref(book()), None, None), "null pointer")
    refuses(library.tnsr_b200_pages_release(C.byref(book()), None, None), "null pointer")
    for bad in (None, C.byref(pools(tensors=None)), C.byref(pools(page_bytes=None)), C.byref(pools(tensors=(C.c_void_p * 1)(None))),
                C.byref(pools(page_bytes=(C.c_uint64 * 1)(0)))):
        refuses(library.tnsr_b200_pages_reserve(C.byref(book()), bad, None, 1, None), "pool")
        refuses(library.tnsr_b200_pages_compact(C.byref(book()), bad, None, None), "pool")
        refuses(library.tnsr_b200_pages_copy(bad, SOME, SOME, 1, 4, None, None), "pool")
    refuses(library.tnsr_b200_pages_copy(C.byref(pools()), None, SOME, 1, 4, None, None), "null pointer")
    assert library.tnsr_b200_pages_copy(C.byref(pools()), None, None, 0, 4, None, None) == 0
    assert library.tnsr_b200_pages_fork(C.byref(book(sequences=0)), SOME, None) == 0


def append(**over):
    fields = dict(k=SOME, v=SOME, k_pool=SOME, v_pool=SOME, table=SOME, lengths=SOME, sequences=2, chunk=1, rows=2, k_ld=128, v_ld=128, kv_heads=2, dim=64, vdim=64,
                  table_ld=4, page_rows=16, pool_pages=8, dtype=1)
    return _native.PagedAppendArgs(**{**fields, **over})


def attend(**over):
    fields = dict(q=SOME, out=SOME, k_pool=SOME, v_pool=SOME, table=SOME, lengths=SOME, workspace=SOME, workspace_bytes=1 << 40, sequences=2, chunk=1, rows=2, q_ld=256,
                  out_ld=256, heads=4, kv_heads=2, dim=64, vdim=64, table_ld=4, page_rows=16, pool_pages=8, scale=0.125, dtype=1)
    return _native.PagedAttentionArgs(**{**fields, **over})


@pytest.mark.parametrize("make,entry", [(append, "tnsr_b200_paged_append"), (attend, "tnsr_b200_paged_attention")])
def test_rows_over_pages_refuse(library, make, entry):
    call = getattr(library, entry)
    refuses(call(None, None), "null pointer")
    for name in ("k_pool", "v_pool", "table", "lengths") + (("k", "v") if make is append else ("q", "out")):
        refuses(call(C.byref(make(**{name: None})), None), "null pointer")
    for name in ("chunk", "kv_heads", "dim", "vdim", "table_ld", "page_rows", "pool_pages"):
        refuses(call(C.byref(make(**{name: 0})), None), "positive")
    refuses(call(C.byref(make(dtype=2)), None), "dtype")
    refuses(call(C.byref(make(rows=3)), None), "row_starts")
    refuses(call(C.byref(make(kv_heads=1 << 26)), None), "2^31")
    refuses(call(C.byref(make(rows=1 << 31, row_starts=SOME)), None), "rows")
    assert call(C.byref(make(rows=0, sequences=0)), None) == 0
    if make is append:
        refuses(call(C.byref(make(k_ld=127)), None), "hold every head")
        refuses(call(C.byref(make(v_ld=127)), None), "hold every head")
    else:
        for over in (dict(heads=0), dict(heads=5), dict(q_ld=255), dict(out_ld=255)):
            refuses(call(C.byref(make(**over)), None), "heads")
        refuses(call(C.byref(make(dim=257, q_ld=2000)), None), "256", -8)
        refuses(call(C.byref(make(scale=float("nan"))), None), "scale")
        refuses(call(C.byref(make(sinks=3)), None), "sinks")
        need = library.tnsr_b200_paged_attention_workspace(64, 64, 1)
        refuses(call(C.byref(make(workspace_bytes=need - 1)), None), "workspace")
        refuses(call(C.byref(make(workspace=SOME + 8)), None), "workspace")


def test_a_selections_workspace_is_enough_for_smaller_ones(library):
    need = library.tnsr_b200_beam_select_workspace
    for vocab in (5, 2049, 9000, 130001):
        for beams in (1, 4, 7, 32):
            sizes = [need(groups, beams, vocab, 8) for groups in range(1, 200)]
            assert sizes == sorted(sizes)
    for big, small in (((40, 8, 50000, 16), (39, 3, 50000, 16)), ((40, 8, 50000, 16), (40, 8, 2048, 16)), ((40, 8, 50000, 16), (1, 1, 49999, 1))):
        assert need(*big) >= need(*small)


def test_more_rows_and_heads_than_a_grid_has_room_for_are_refused(library):
    for rows, heads, dim in ((1 << 30, 8, 1), (0x7fffffff, 5, 1), (1 << 25, 260, 7)):
        refuses(library.tnsr_b200_paged_attention(C.byref(attend(rows=rows, sequences=rows, heads=heads, kv_heads=1, dim=dim, vdim=dim, q_ld=heads * dim, out_ld=heads * dim)),
                                                  None), "too many rows")
