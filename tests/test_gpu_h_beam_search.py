"""Beam selection, reordered states and the management of pages against plain implementations, and all of them as a search uses them."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import _KEEP, lib, ok, ptr, stream  # noqa: E402
from tests.paged_util import DTYPES, NONE, host, scratch, status_word, u32  # noqa: E402
from tnsr_b200 import _native  # noqa: E402


# ---- selection -----------------------------------------------------------------------------------------------------------------------
def select(logits, scores, finished, groups, beams, keep, end, ld=None, work=None, offset=0):
    vocab = logits.shape[1]
    ld = ld or vocab
    room = torch.full((groups * beams * ld + offset,), float("nan"), dtype=logits.dtype, device="cuda")
    rows = room[offset:].view(groups * beams, ld)
    rows[:, :vocab] = logits.cuda()
    scores = scores.float().cuda()
    finished = None if finished is None else finished.to(torch.uint8).cuda()
    out = [torch.full((groups, keep), -7, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    done = torch.full((groups, keep), 7, dtype=torch.uint8, device="cuda")
    if work is None:
        work = scratch(lib().tnsr_b200_beam_select_workspace(groups, beams, vocab, keep))
    _KEEP.extend([room, scores, finished, work, done, *out])
    args = _native.BeamSelectArgs(logits=rows.data_ptr(), scores=scores.data_ptr(), finished=None if finished is None else finished.data_ptr(),
                                  next_scores=out[0].data_ptr(), tokens=out[1].data_ptr(), parents=out[2].data_ptr(), next_finished=done.data_ptr(),
                                  workspace=work.data_ptr(), workspace_bytes=work.numel(), logits_ld=ld, groups=groups, beams=beams, vocab=vocab, keep=keep,
                                  end_token=end, dtype=0 if logits.dtype == torch.float32 else 1)
    ok(lib().tnsr_b200_beam_select(C.byref(args), stream()))
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in out] + [done.cpu().numpy()]


def plain_select(logits, scores, finished, groups, beams, keep, end):
    """The rule of the header, candidate by candidate, in 64 bits."""
    x, c = logits.double().numpy(), scores.double().numpy()
    vocab = x.shape[1]
    result = []
    for g in range(groups):
        candidates = []
        for b in range(beams):
            row = g * beams + b
            over = finished is not None and bool(finished[row])
            with np.errstate(all="ignore"):
                top = np.max(x[row]) if not np.isnan(x[row]).any() else np.nan
                total = top + np.log(np.sum(np.exp(x[row] - top)))
            if over or not np.isfinite(total) or not np.isfinite(c[row]):
                s, order = np.full(vocab, -np.inf), np.zeros(vocab)
                if over and end < vocab and np.isfinite(c[row]):
                    s[end] = c[row]
            else:
                s, order = c[row] + (x[row] - total), np.where(np.isneginf(x[row]), 0.0, x[row])
            best = sorted(range(vocab), key=lambda t: (-s[t], -order[t], t))[:keep] if vocab < 3000 else list(np.lexsort((np.arange(vocab), -order, -s))[:keep])
            candidates += [(-s[t], b, i, t) for i, t in enumerate(best)]
        candidates.sort(key=lambda a: a[:3])
        result.append([(-s, t, g * beams + b) for s, b, _, t in candidates[:keep]])
    r = np.array(result)
    tokens, parents = r[..., 1].astype(np.int64), r[..., 2].astype(np.int64)
    done = tokens == end
    if finished is not None:
        done |= finished.numpy().astype(bool)[parents]
    return r[..., 0], tokens, parents, done


def check_select(got, want):
    scores, tokens, parents, done = got
    assert np.array_equal(tokens, want[1]) and np.array_equal(parents, want[2]) and np.array_equal(done, want[3])
    finite = np.isfinite(want[0])
    assert np.array_equal(np.isneginf(scores), ~finite)
    # the sum of exponentials: 32 terms at a time in f32 (32 steps), an exponential and its argument 2^-19 together; its logarithm is off by as
    # much, absolutely; then one rounding to f32
    off = np.abs(scores[finite] - want[0][finite])
    assert np.all(off <= 2.0 ** -18 + 2.0 ** -24 * np.abs(want[0][finite]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 12), (3, 4, 96, 8), (1, 4, 32000, 4), (2, 8, 2047, 16), (5, 1, 50021, 1),
                                                     (3, 32, 700, 64), (1, 5, 9000, 10), (40, 6, 8200, 12), (2, 2, 130001, 3), (1, 2, 64, 64), (70, 5, 33000, 9)])
def test_selection_equals_the_rule(dtype, groups, beams, vocab, keep):
    gen = torch.Generator().manual_seed(vocab + keep)
    rows = groups * beams
    logits = (torch.randn(rows, vocab, generator=gen) * 3).to(DTYPES[dtype])
    logits[torch.rand(rows, vocab, generator=gen) < 0.1] = -math.inf
    logits[:, vocab // 2] = 1.0
    scores = -torch.rand(rows, generator=gen) * 20
    finished = torch.rand(rows, generator=gen) < 0.3
    for end, over in ((vocab // 2, finished), (0xffffffff, None), (0, finished)):
        want = plain_select(logits, scores, over, groups, beams, keep, end)
        check_select(select(logits, scores, over, groups, beams, keep, end), want)
    # rows behind one another with a pitch, and at an odd address
    check_select(select(logits, scores, finished, groups, beams, keep, 0, ld=(vocab + 15) // 8 * 8), want)
    check_select(select(logits, scores, finished, groups, beams, keep, 0, ld=vocab + 1, offset=1), want)


@pytest.mark.parametrize("vocab", [40, 3000, 32000])
@pytest.mark.parametrize("keep", [1, 4, 13, 64])
def test_selection_among_equal_and_sorted_and_masked_logits(vocab, keep):
    groups, beams = 3, 4
    cases = {
        "equal": torch.zeros(12, vocab),
        "few values": torch.randint(0, 3, (12, vocab), generator=torch.Generator().manual_seed(1)).float(),
        "falling": -torch.arange(vocab).float().expand(12, vocab) * 0.01,
        "rising": torch.arange(vocab).float().expand(12, vocab) * 0.01,
        "one token": torch.full((12, vocab), -math.inf).index_fill(1, torch.tensor([vocab - 1]), 0.0),
        "blocks": torch.where(torch.arange(vocab) % 1024 < 16, torch.arange(vocab) * 1e-3, torch.tensor(-math.inf)).expand(12, vocab),
        "signed zeros": torch.where(torch.arange(vocab) % 2 == 0, -0.0, 0.0).expand(12, vocab),
    }
    scores = torch.tensor([-1.0, -1.0, -2.0, -1.0] * 3)
    for name, logits in cases.items():
        logits = logits.contiguous()
        want = plain_select(logits, scores, None, groups, beams, keep, 2)
        check_select(select(logits, scores, None, groups, beams, keep, 2), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_selection_with_beams_that_have_no_sum(dtype):
    gen = torch.Generator().manual_seed(5)
    vocab, keep = 4001, 24
    logits = torch.randn(8, vocab, generator=gen).to(DTYPES[dtype])
    logits[0, 17], logits[1, 4000], logits[2] = math.nan, math.inf, -math.inf
    scores = torch.tensor([0.0, 0.0, 0.0, -1.0, -math.inf, math.nan, -3.0, math.inf])
    finished = torch.tensor([False, False, True, False, True, False, True, False])
    for groups, beams, over in ((1, 8, finished), (2, 4, finished), (8, 1, None), (1, 8, torch.ones(8, dtype=torch.bool)), (4, 2, None)):
        want = plain_select(logits, scores, over, groups, beams, keep, 9)
        check_select(select(logits, scores, over, groups, beams, keep, 9), want)
    # the first step of a search: one beam counts
    first = torch.tensor([0.0] + [-math.inf] * 7)
    clean = torch.randn(1, vocab, generator=gen).to(DTYPES[dtype]).expand(8, vocab).contiguous()
    got = select(clean, first, None, 1, 8, 8, 0xffffffff)
    assert np.all(got[2] == 0)
    check_select(got, plain_select(clean, first, None, 1, 8, 8, 0xffffffff))
    # equal beams: all of an earlier one's equals come first
    same = torch.zeros(8)
    check_select(select(clean, same, None, 1, 8, 24, 0xffffffff), plain_select(clean, same, None, 1, 8, 24, 0xffffffff))


def test_selection_in_a_graph_follows_its_inputs():
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(12, 9000, generator=gen).cuda()
    scores = torch.zeros(12, device="cuda")
    out = [torch.zeros((3, 4), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    work = scratch(lib().tnsr_b200_beam_select_workspace(3, 4, 9000, 4))
    args = _native.BeamSelectArgs(logits=logits.data_ptr(), scores=scores.data_ptr(), next_scores=out[0].data_ptr(), tokens=out[1].data_ptr(),
                                  parents=out[2].data_ptr(), workspace=work.data_ptr(), workspace_bytes=work.numel(), logits_ld=9000, groups=3, beams=4,
                                  vocab=9000, keep=4, end_token=1, dtype=0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ok(lib().tnsr_b200_beam_select(C.byref(args), stream()))
    for _ in range(3):
        fresh = torch.randn(12, 9000, generator=gen)
        logits.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = plain_select(fresh, torch.zeros(12), None, 3, 4, 4, 1)
        assert np.array_equal(out[1].cpu().numpy(), want[1]) and np.array_equal(out[2].cpu().numpy(), want[2])


# ---- states ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 2), (3, 4), (5, 7), (2, 8), (3, 9), (1, 32), (7, 31)])
@pytest.mark.parametrize("sizes", [[(16, 16)], [(4096, 4096), (48, 64), (100000, 100016)], [(20, 24)], [(7, 9), (4096, 4097)], [(64, 64)] * 70])
def test_states_move_to_their_parents_places(groups, beams, sizes):
    rng = np.random.default_rng(groups * 100 + beams)
    rows = groups * beams
    tensors = [torch.from_numpy(rng.integers(0, 256, (rows, pitch), dtype=np.uint8)).cuda() for _, pitch in sizes]
    n = len(sizes)
    at = (C.c_void_p * n)(*[t.data_ptr() for t in tensors])
    nbytes, pitches = (C.c_uint64 * n)(*[s for s, _ in sizes]), (C.c_uint64 * n)(*[p for _, p in sizes])
    for _ in range(4):
        parents = rng.integers(0, beams, rows) + np.arange(rows) // beams * beams
        bad = rng.integers(0, 6) == 0 and rows > 1
        asked = parents.copy()
        if bad:
            asked[rows - 1], parents[rows - 1] = rows, rows - 1
        want = [torch.cat([t[torch.from_numpy(parents).cuda(), :s], t[:, s:]], 1) for t, (s, _) in zip(tensors, sizes)]
        status = status_word()
        ok(lib().tnsr_b200_reorder_states(at, nbytes, pitches, n, ptr(u32(asked)), groups, beams, ptr(status), stream()))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(tensors, want))
        assert int(status[0]) == (6 if bad and beams > 1 else 0)


# ---- pages ------------------------------------------------------------------------------------------------------------------------------
class Book:
    """A book on the device beside a model of it in Python, whose pages hold lists of what was written."""

    def __init__(self, sequences, table_ld, page_rows, pool_pages, page_bytes=(64, 32)):
        self.s, self.ld, self.r, self.pool = sequences, table_ld, page_rows, pool_pages
        self.table, self.lengths, self.holders = u32(np.full((sequences, table_ld), NONE)), u32(np.zeros(sequences)), u32(np.zeros(pool_pages))
        self.rng = np.random.default_rng(sequences * 7 + pool_pages)
        self.pools = [torch.from_numpy(self.rng.integers(0, 256, (pool_pages, b), dtype=np.uint8)).cuda() for b in page_bytes]
        self.work, self.status = scratch(lib().tnsr_b200_pages_workspace(sequences, pool_pages)), status_word()
        n = len(page_bytes)
        self.tensors, self.page_bytes = (C.c_void_p * n)(*[t.data_ptr() for t in self.pools]), (C.c_uint64 * n)(*page_bytes)
        self.c_pools = _native.PagePools(tensors=self.tensors, page_bytes=self.page_bytes, count=n)
        self.c_book = _native.PageBook(table=self.table.data_ptr(), lengths=self.lengths.data_ptr(), holders=self.holders.data_ptr(),
                                       workspace=self.work.data_ptr(), d_status=self.status.data_ptr(), workspace_bytes=self.work.numel(),
                                       sequences=sequences, table_ld=table_ld, page_rows=page_rows, pool_pages=pool_pages)
        self.m_pages, self.m_lengths = [[] for _ in range(sequences)], [0] * sequences
        self.m_pools = [p.cpu().numpy().copy() for p in self.pools]

    def held(self):
        count = np.zeros(self.pool, np.int64)
        for pages in self.m_pages:
            for p in pages:
                count[p] += 1
        return count

    def check(self, status=0):
        torch.cuda.synchronize()
        assert int(self.status[0]) == status
        self.status.zero_()
        assert host(self.lengths).tolist() == self.m_lengths
        table = host(self.table)
        for s, pages in enumerate(self.m_pages):
            assert table[s, :len(pages)].tolist() == pages, s
        assert np.array_equal(host(self.holders), self.held())
        live = self.held() > 0
        for p, m in zip(self.pools, self.m_pools):
            assert np.array_equal(p.cpu().numpy()[live], m[live])

    def fork(self, parents):
        ok(lib().tnsr_b200_pages_fork(C.byref(self.c_book), ptr(u32(parents)), stream()))
        self.m_pages, self.m_lengths = [list(self.m_pages[p]) for p in parents], [self.m_lengths[p] for p in parents]

    def reserve(self, rows, status=0):
        each = rows if isinstance(rows, int) else 0
        array = None if isinstance(rows, int) else u32(rows)
        ok(lib().tnsr_b200_pages_reserve(C.byref(self.c_book), C.byref(self.c_pools), ptr(array), each, stream()))
        rows = [rows] * self.s if isinstance(rows, int) else list(rows)
        if any(length + n > self.ld * self.r for length, n in zip(self.m_lengths, rows)):
            assert status == 3
            return
        held = self.held()
        writers = {}
        for s, n in enumerate(rows):
            if n and self.m_lengths[s] % self.r and held[self.m_pages[s][-1]] > 1:
                writers.setdefault(self.m_pages[s][-1], []).append(s)
        copies = {s for page, who in writers.items() for s in (who[1:] if len(who) == held[page] else who)}
        need = sum(-(-(length + n) // self.r) - -(-length // self.r) for length, n in zip(self.m_lengths, rows)) + len(copies)
        free = [p for p in range(self.pool) if held[p] == 0]
        if need > len(free):
            assert status == 5
            return
        for s, n in enumerate(rows):
            if s in copies:
                page = free.pop(0)
                for m in self.m_pools:
                    m[page] = m[self.m_pages[s][-1]]
                self.m_pages[s][-1] = page
            while len(self.m_pages[s]) * self.r < self.m_lengths[s] + n:
                self.m_pages[s].append(free.pop(0))
            self.m_lengths[s] += n

    def release(self, gone):
        flags = torch.zeros(self.s, dtype=torch.uint8)
        flags[list(gone)] = 3
        flags = flags.cuda()
        _KEEP.append(flags)
        ok(lib().tnsr_b200_pages_release(C.byref(self.c_book), ptr(flags), stream()))
        for s in gone:
            self.m_pages[s], self.m_lengths[s] = [], 0

    def compact(self):
        live = status_word()
        ok(lib().tnsr_b200_pages_compact(C.byref(self.c_book), C.byref(self.c_pools), ptr(live), stream()))
        held = self.held()
        n = int((held > 0).sum())
        to = [p for p in range(n) if held[p] == 0]
        moved = dict(zip([p for p in range(n, self.pool) if held[p]], to))
        for page, place in moved.items():
            for m in self.m_pools:
                m[place] = m[page]
        self.m_pages = [[moved.get(p, p) for p in pages] for pages in self.m_pages]
        torch.cuda.synchronize()
        assert int(live[0]) == n


@pytest.mark.parametrize("sequences,ld,page_rows,pool,page_bytes", [(1, 3, 1, 3, (16,)), (6, 12, 4, 60, (64, 32)), (24, 20, 7, 300, (48, 5, 3)), (64, 40, 16, 2000, (40000, 64)),
                                                                   (1100, 6, 3, 5000, (16,)), (5, 9, 2, 40000, (4,)), (1700, 4, 2, 6000, (32,)), (3, 5, 8, 20, ())])
def test_books_go_through_random_searches(sequences, ld, page_rows, pool, page_bytes):
    book = Book(sequences, ld, page_rows, pool, page_bytes)
    rng = book.rng
    for step in range(25):
        kind = rng.integers(0, 6)
        if kind <= 2:
            room = ld * page_rows - max(book.m_lengths)
            rows = rng.integers(0, min(room, 2 * page_rows) + 1, sequences) * (rng.random(sequences) < 0.7)
            free = int((book.held() == 0).sum())
            if int(rows.sum()) // page_rows + 2 * sequences > free or room == 0:
                book.release([int(s) for s in np.flatnonzero(rng.random(sequences) < 0.5)])
            elif rng.random() < 0.5:
                book.reserve(1)
            else:
                book.reserve([int(r) for r in rows])
        elif kind == 3:
            book.fork([int(p) for p in rng.integers(0, sequences, sequences)])
        elif kind == 4:
            book.release([int(s) for s in np.flatnonzero(rng.random(sequences) < 0.2)])
        else:
            book.compact()
        book.check()
        # a page's contents are its holders': change some
        for p, m in zip(book.pools, book.m_pools):
            at = int(rng.integers(0, pool))
            m[at] = step
            p[at] = step


def test_a_reserve_that_cannot_be_changes_nothing():
    book = Book(4, 3, 4, 8)
    book.reserve([5, 1, 0, 9])
    book.check()
    book.fork([0, 0, 0, 3])
    book.check()
    book.reserve(1)                      # two of three copies and 0, 1, 2 at row 5
    book.check()
    book.reserve([8, 0, 0, 0], status=3)
    book.check(status=3)
    book.reserve([3, 3, 3, 3], status=3)         # 13 rows of 12
    book.check(status=3)
    book.reserve([3, 3, 3, 1], status=5)         # three pages of one
    book.check(status=5)
    book.release([0, 1])
    book.check()
    book.reserve([3, 3, 3, 1])
    book.check()


def test_a_shared_page_is_copied_for_writers_beside_a_reader():
    book = Book(5, 4, 4, 30)
    book.reserve([6, 0, 0, 0, 0])
    book.fork([0, 0, 0, 0, 4])
    before = [list(p) for p in book.m_pages]
    book.reserve([1, 0, 1, 0, 0])        # 1 and 3 do not write: both writers get copies
    book.check()
    assert book.m_pages[1] == before[1] and book.m_pages[0][-1] != before[0][-1] != book.m_pages[2][-1]
    book.reserve([0, 1, 0, 1, 0])        # both holders write: the first keeps the page
    book.check()
    assert book.m_pages[1] == before[1] and book.m_pages[3][-1] != before[3][-1]


def test_bad_parents_and_pages_are_reported():
    book = Book(4, 3, 4, 12)
    book.reserve([5, 1, 3, 9])
    book.check()
    ok(lib().tnsr_b200_pages_fork(C.byref(book.c_book), ptr(u32([0, 9, 2, NONE])), stream()))
    book.check(status=6)
    table = host(book.table)
    table[1, 0] = 12
    book.table.copy_(u32(table))
    ok(lib().tnsr_b200_pages_reserve(C.byref(book.c_book), C.byref(book.c_pools), None, 1, stream()))
    torch.cuda.synchronize()
    assert int(book.status[0]) == 4 and host(book.lengths).tolist() == [5, 1, 3, 9]


@pytest.mark.parametrize("sequences", [4096, 4097, 12288])
def test_the_largest_books_fork(sequences):
    book = Book(sequences, 3, 2, 2 * sequences + 7)
    rng = np.random.default_rng(sequences)
    book.reserve([int(r) for r in rng.integers(0, 4, sequences)])
    book.fork([int(p) for p in rng.integers(0, sequences, sequences)])
    book.check()


def test_a_row_alone_stays_and_its_bad_parent_is_reported():
    t = torch.arange(3 * 8, dtype=torch.int32, device="cuda").view(3, 8)
    for parents, want in (([0, 1, 2], 0), ([0, 2, 2], 6)):
        status = status_word()
        one, size = (C.c_void_p * 1)(t.data_ptr()), (C.c_uint64 * 1)(32)
        ok(lib().tnsr_b200_reorder_states(one, size, size, 1, ptr(u32(parents)), 3, 1, ptr(status), stream()))
        torch.cuda.synchronize()
        assert int(status[0]) == want and t.flatten().tolist() == list(range(24))


def test_pages_are_copied_onto_others():
    book = Book(1, 1, 1, 50, (16, 33, 70000))
    pairs = [(3, 7), (9, 8), (3, 49), (0, 1)]
    status = status_word()
    before = [p.cpu().numpy().copy() for p in book.pools]
    for pairs, want in ((pairs, 0), ([(1, 2), (50, 3), (4, 4000000000)], 4), ([], 0)):
        for b in before:
            for x, y in pairs:
                if x < 50 and y < 50:
                    b[y] = b[x]
        status.zero_()
        ok(lib().tnsr_b200_pages_copy(C.byref(book.c_pools), ptr(u32([x for x, _ in pairs])), ptr(u32([y for _, y in pairs])), len(pairs), 50, ptr(status),
                                      stream()))
        torch.cuda.synchronize()
        assert int(status[0]) == want
        assert all(np.array_equal(p.cpu().numpy(), b) for p, b in zip(book.pools, before))


# ---- together -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_search_over_a_paged_cache_equals_one_that_keeps_whole_sequences(dtype, captured):
    """A two-layer toy model (token embedding -> q, k, v -> attention -> logits) decodes 40 steps of beam search; the plain search keeps every beam's tokens and
    recomputes its keys, and is told the choices that the search under test made, whose scores it checks."""
    t = DTYPES[dtype]
    groups, beams, heads, kv, dim, page_rows, vocab, steps = 3, 4, 4, 2, 64, 16, 311, 40
    rows, ld, pool, window, sinks = groups * beams, 4, 80, 20, 3
    gen = torch.Generator("cuda").manual_seed(3)
    weights = [tuple(torch.randn(vocab, n, dim, device="cuda", generator=gen).to(t) for n in (heads, kv, kv)) for _ in range(2)]
    head = torch.randn(2 * heads * dim, vocab, device="cuda", generator=gen) / 12
    table, lengths, holders = u32(np.full((rows, ld), NONE)), u32(np.zeros(rows)), u32(np.zeros(pool))
    pools = [torch.zeros(pool, page_rows, kv, dim, dtype=t, device="cuda") for _ in range(4)]
    state = torch.zeros(rows, 6, dtype=torch.int32, device="cuda")       # what a recurrent layer would keep: the last tokens
    work = scratch(lib().tnsr_b200_pages_workspace(rows, pool))
    attention_work = scratch(lib().tnsr_b200_paged_attention_workspace(dim, dim, _native.DTYPE[dtype]))
    select_work = scratch(lib().tnsr_b200_beam_select_workspace(groups, beams, vocab, beams))
    status = status_word()
    nbytes = page_rows * kv * dim * pools[0].element_size()
    c_pools = _native.PagePools(tensors=(C.c_void_p * 4)(*[p.data_ptr() for p in pools]), page_bytes=(C.c_uint64 * 4)(*[nbytes] * 4), count=4)
    book = _native.PageBook(table=table.data_ptr(), lengths=lengths.data_ptr(), holders=holders.data_ptr(), workspace=work.data_ptr(), d_status=status.data_ptr(),
                            workspace_bytes=work.numel(), sequences=rows, table_ld=ld, page_rows=page_rows, pool_pages=pool)
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") // beams
    parents = torch.arange(rows, dtype=torch.int32, device="cuda")
    scores = torch.tensor([0.0] + [-math.inf] * (beams - 1), device="cuda").repeat(groups)
    next_scores, out = torch.empty_like(scores), torch.empty(2, rows, heads * dim, dtype=t, device="cuda")
    state_at, state_bytes = (C.c_void_p * 1)(state.data_ptr()), (C.c_uint64 * 1)(24)
    L = lib()

    def step():
        s = stream()
        ok(L.tnsr_b200_pages_fork(C.byref(book), parents.data_ptr(), s))
        ok(L.tnsr_b200_pages_reserve(C.byref(book), C.byref(c_pools), None, 1, s))
        ok(L.tnsr_b200_reorder_states(state_at, state_bytes, state_bytes, 1, parents.data_ptr(), groups, beams, status.data_ptr(), s))
        state.copy_(torch.cat([state[:, 1:], tokens[:, None]], 1))
        for layer, (wq, wk, wv) in enumerate(weights):
            q, k, v = (w[tokens.long()].contiguous() for w in (wq, wk, wv))
            common = dict(table=table.data_ptr(), lengths=lengths.data_ptr(), d_status=status.data_ptr(), sequences=rows, chunk=1, rows=rows, kv_heads=kv,
                          dim=dim, vdim=dim, table_ld=ld, page_rows=page_rows, pool_pages=pool, dtype=_native.DTYPE[dtype],
                          k_pool=pools[2 * layer].data_ptr(), v_pool=pools[2 * layer + 1].data_ptr())
            ok(L.tnsr_b200_paged_append(C.byref(_native.PagedAppendArgs(k=k.data_ptr(), v=v.data_ptr(), k_ld=kv * dim, v_ld=kv * dim, **common)), s))
            ok(L.tnsr_b200_paged_attention(C.byref(_native.PagedAttentionArgs(
                q=q.data_ptr(), out=out[layer].data_ptr(), workspace=attention_work.data_ptr(), workspace_bytes=attention_work.numel(), q_ld=heads * dim,
                out_ld=heads * dim, heads=heads, window=window, sinks=sinks, scale=0.125, **common)), s))
            _KEEP.extend([q, k, v])
        logits = (out.transpose(0, 1).reshape(rows, -1).float() @ head).contiguous()
        _KEEP.append(logits)
        ok(L.tnsr_b200_beam_select(C.byref(_native.BeamSelectArgs(
            logits=logits.data_ptr(), scores=scores.data_ptr(), next_scores=next_scores.data_ptr(), tokens=tokens.data_ptr(), parents=parents.data_ptr(),
            workspace=select_work.data_ptr(), workspace_bytes=select_work.numel(), logits_ld=vocab, groups=groups, beams=beams, vocab=vocab, keep=beams,
            end_token=0xffffffff, dtype=0)), s))
        scores.copy_(next_scores)

    history = [[r // beams] for r in range(rows)]
    plain_scores = [0.0 if r % beams == 0 else -math.inf for r in range(rows)]
    graph = None
    for i in range(steps):
        if captured and i == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        if graph is not None:
            graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        assert int(status[0]) == 0
        # every beam's logits from its whole history, in 64 bits
        want = []
        for h in history:
            at = torch.tensor(h, device="cuda")
            j = torch.arange(len(h), device="cuda")
            seen = (j > len(h) - 1 - window) | (j < sinks)
            o = []
            for wq, wk, wv in weights:
                q, k, v = wq[at[-1]].double(), wk[at].double()[seen].repeat_interleave(heads // kv, 1), wv[at].double()[seen].repeat_interleave(heads // kv, 1)
                w = torch.softmax(0.125 * torch.einsum("hd,jhd->hj", q, k), 1)
                o.append(torch.einsum("hj,jhd->hd", w, v).reshape(-1))
            want.append(torch.log_softmax(torch.cat(o) @ head.double(), 0).cpu())
        chosen, from_, got = host(tokens), host(parents), scores.cpu()
        # attention in bf16 is off by 2^-7 of a value, of size 3 at the most, in 512 terms of weight 1/12 that do not all err the same way
        room = 2e-3 if dtype == "f32" else 0.25
        for r in range(rows):
            assert from_[r] // beams == r // beams
            expect = plain_scores[from_[r]] + float(want[from_[r]][chosen[r]])
            assert abs(float(got[r]) - expect) <= room
        # nothing better was left out
        for g in range(groups):
            every = torch.cat([plain_scores[r] + want[r] for r in range(g * beams, (g + 1) * beams)])
            best = torch.topk(every, beams).values
            assert float((got[g * beams:(g + 1) * beams].double() - best).abs().max()) <= room
        history = [history[from_[r]] + [int(chosen[r])] for r in range(rows)]
        plain_scores = [float(x) for x in got]
    held = np.bincount(np.concatenate([host(table)[r, :-(-steps // page_rows)] for r in range(rows)]), minlength=pool)
    assert np.array_equal(host(holders), held)
    # the state that travelled with the beams holds what they decoded before the last choice
    final = host(state)
    before = [h[:-1] for h in history]
    parents_now = host(parents)
    for r in range(rows):
        assert final[parents_now[r]].tolist()[-6:] == before[r][-6:]
