"""Workspaces that are zeroed once and serve calls of different sizes one after the other."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import lib  # noqa: E402
from tests.paged_util import scratch  # noqa: E402
from tests.test_gpu_h_beam_search import Book, check_select, plain_select, select  # noqa: E402

# groups, beams, vocab, keep: joined by a group's last block or by a launch of its own (32 x 700, and 1100 groups), one run of a row or many
SELECTIONS = [(48, 6, 9001, 12), (47, 6, 9001, 12), (2, 4, 32000, 4), (1, 4, 32000, 4), (3, 32, 700, 64), (1, 4, 32000, 8), (5, 1, 50021, 1), (1100, 2, 90, 3), (64, 4, 600, 4),
              (1024, 1, 70, 2), (1, 1, 5, 5), (1025, 1, 70, 2), (7, 3, 4100, 13)]


@pytest.mark.parametrize("order", ["as listed", "backwards", "shuffled"])
def test_one_workspace_serves_selections_of_all_sizes(order):
    work = scratch(max(lib().tnsr_b200_beam_select_workspace(*s) for s in SELECTIONS))
    assert int(work.max()) == 0
    sizes = {"as listed": SELECTIONS, "backwards": SELECTIONS[::-1], "shuffled": SELECTIONS * 2}[order]
    if order == "shuffled":
        sizes = [sizes[i] for i in np.random.default_rng(0).permutation(len(sizes))]
    gen = torch.Generator().manual_seed(1)
    for groups, beams, vocab, keep in sizes:
        logits = torch.randn(groups * beams, vocab, generator=gen) * 3
        logits[torch.rand(groups * beams, vocab, generator=gen) < 0.1] = -math.inf
        scores = -torch.rand(groups * beams, generator=gen) * 20
        check_select(select(logits, scores, None, groups, beams, keep, 0, work=work), plain_select(logits, scores, None, groups, beams, keep, 0))


def test_a_search_whose_groups_finish_one_after_the_other():
    beams, vocab, keep = 4, 5000, 8
    work = scratch(lib().tnsr_b200_beam_select_workspace(12, beams, vocab, keep))
    gen = torch.Generator().manual_seed(2)
    assert all(lib().tnsr_b200_beam_select_workspace(g, beams, vocab, keep) <= work.numel() for g in range(1, 13))
    for groups in list(range(12, 0, -1)) + [3, 12]:
        logits, scores = torch.randn(groups * beams, vocab, generator=gen), -torch.rand(groups * beams, generator=gen)
        check_select(select(logits, scores, None, groups, beams, keep, 0, work=work), plain_select(logits, scores, None, groups, beams, keep, 0))


@pytest.mark.parametrize("sizes", [[(8, 60), (6, 33), (8, 300)], [(40, 4000), (3, 17), (12, 90), (40, 4001)]])
def test_one_workspace_serves_books_of_all_sizes(sizes):
    """Searches step by step in turn: last pages that several beams hold and write to, or that a beam which does not write holds beside them."""
    books = [Book(sequences, 6, 4, pool) for sequences, pool in sizes]
    work = scratch(max(lib().tnsr_b200_pages_workspace(*s) for s in sizes))
    for book in books:
        book.c_book.workspace, book.c_book.workspace_bytes = work.data_ptr(), work.numel()
        book.reserve([2] + [0] * (book.s - 1))
        book.check()
    for step in range(12):
        for book in books:
            rng = book.rng
            if step % 4 == 3:
                book.compact()
                book.release([s for s in range(book.s) if book.m_lengths[s] > 12 or rng.random() < 0.2])
                if not any(book.m_lengths):
                    book.reserve([3] + [0] * (book.s - 1))
            live = [s for s in range(book.s) if book.m_lengths[s]]
            book.fork([live[int(i)] for i in rng.integers(0, min(2, len(live)), book.s)])
            book.check()
            if max(book.m_lengths) < 20 and int((book.held() == 0).sum()) >= book.s:
                book.reserve([int(r) for r in rng.random(book.s) < 0.7])
            book.check()
