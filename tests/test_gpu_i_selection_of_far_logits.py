"""Beam selection where finite logits lie far apart: masks by large negative numbers, and logits whose exponential or whose product with log2(e) no f32 holds."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.paged_util import DTYPES  # noqa: E402
from tests.test_gpu_h_beam_search import check_select, select  # noqa: E402

MASKS = {"f32 lowest": torch.finfo(torch.float32).min, "bf16 lowest": torch.finfo(torch.bfloat16).min, "-1e30": -1e30, "-1e20": -1e20, "-1e10": -1e10,
         "-1e6": -1e6, "-1e4": -1e4}


def want_select(logits, scores, finished, groups, beams, keep, end):
    """The rule in 64 bits, with a row's largest logit taken off first: beside one of 1e20 the sum's logarithm would be lost.  Order within a beam is by the logits themselves."""
    x, c = logits.double().numpy(), scores.double().numpy()
    vocab = x.shape[1]
    result = []
    for g in range(groups):
        candidates = []
        for b in range(beams):
            row = g * beams + b
            over, top = finished is not None and bool(finished[row]), x[row].max()
            if over or np.isneginf(top):
                s, order = np.full(vocab, -np.inf), np.zeros(vocab)
                if over:
                    s[end] = c[row]
            else:
                below = x[row] - top
                s, order = c[row] + (below - np.log(np.sum(np.exp(below)))), np.where(np.isneginf(x[row]), 0.0, x[row])
            best = np.lexsort((np.arange(vocab), -order, -s))[:keep]
            candidates += [(-s[t], b, i, t) for i, t in enumerate(best)]
        candidates.sort(key=lambda a: a[:3])
        result.append([(-s, t, g * beams + b) for s, b, _, t in candidates[:keep]])
    r = np.array(result)
    tokens, parents = r[..., 1].astype(np.int64), r[..., 2].astype(np.int64)
    done = tokens == end
    if finished is not None:
        done |= finished.numpy()[parents]
    # scores are ranked in 64 bits and returned in 32: what is below all of those is -inf
    with np.errstate(over="ignore"):
        best = np.where(np.isneginf(r[..., 0].astype(np.float32)), -np.inf, r[..., 0])
    return best, tokens, parents, done


def check(logits, scores, finished, groups, beams, keep, end=0xffffffff, **how):
    check_select(select(logits, scores, finished, groups, beams, keep, end, **how), want_select(logits, scores, finished, groups, beams, keep, end))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("vocab", [7, 200, 4100, 32000])
def test_logits_masked_by_large_negative_numbers(vocab, mask, dtype):
    if dtype == "bf16" and mask == "f32 lowest":
        pytest.skip("rounds to -inf")
    gen = torch.Generator().manual_seed(vocab)
    groups, beams = 3, 4
    rows = groups * beams
    scores = -torch.rand(rows, generator=gen) * 5
    base = (torch.randn(rows, vocab, generator=gen) * 3).to(DTYPES[dtype])
    order = torch.rand(rows, vocab, generator=gen).argsort(1)
    for allowed in (0, 1, min(300, vocab // 2), vocab - 1):
        # any tokens, the first ones, the last ones: whole runs are masked
        for places in (order, torch.arange(vocab).expand(rows, vocab), torch.arange(vocab - 1, -1, -1).expand(rows, vocab)):
            logits = base.clone().scatter_(1, places[:, allowed:].contiguous(), MASKS[mask])
            check(logits, scores, None, groups, beams, 4)
            check(logits, scores, None, groups, beams, 13)
    # some rows masked, some not, some with -inf beside the mask or instead of it
    logits = base.clone()
    logits[1] = MASKS[mask]
    logits[2] = -math.inf
    logits[3].scatter_(0, order[3, 1:], MASKS[mask])
    logits[4, ::2], logits[4, 1::2] = MASKS[mask], -math.inf
    logits[5].scatter_(0, order[5, vocab // 2:], MASKS[mask])
    logits[5].scatter_(0, order[5, vocab - vocab // 4:], -math.inf)
    finished = torch.tensor([False] * 6 + [True] + [False] * 5)
    for end in (0, vocab - 1):
        check(logits, scores, finished, groups, beams, 7, end, ld=vocab + 1, offset=1)
        check(logits, scores, finished, 1, rows, 24, end)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [7, 200, 4100, 32000])
def test_logits_of_any_finite_size(vocab, dtype):
    gen = torch.Generator().manual_seed(vocab + 1)
    t, rows = DTYPES[dtype], 8
    largest = torch.finfo(t).max
    scores = -torch.rand(rows, generator=gen) * 5
    logits = torch.zeros(rows, vocab, dtype=t)
    logits[0, ::3] = largest                                   # many of the largest
    logits[1, vocab // 2] = largest                            # one, all others zero
    logits[2] = -largest
    logits[2, vocab // 3] = largest                            # both ends
    logits[3] = (torch.randn(vocab, generator=gen) * 1e12).to(t)
    logits[4] = (torch.randn(vocab, generator=gen) * 1e37).to(t)
    logits[5] = (2.0 ** (torch.rand(vocab, generator=gen) * 250 - 126)).to(t)
    logits[6] = -logits[5]
    logits[7] = (1e7 + torch.randn(vocab, generator=gen) * 4).to(t)      # far from zero, near each other
    for keep in (1, 4, 7):
        check(logits, scores, None, rows, 1, keep)
        check(logits, scores, None, 2, 4, keep)


def test_far_logits_do_not_bring_other_rows_to_notice():
    """A row's candidates are what they are beside rows that are masked whole, partly or not at all."""
    gen = torch.Generator().manual_seed(9)
    clean = torch.randn(4, 9000, generator=gen)
    scores = torch.tensor([0.0, -40.0, -40.0, -40.0])
    alone = select(clean, scores, None, 1, 4, 4, 0xffffffff)
    for mask in MASKS.values():
        masked = clean.clone()
        masked[1], masked[2, 100:] = mask, mask
        got = select(masked, scores, None, 1, 4, 4, 0xffffffff)
        assert all(np.array_equal(a, b) for a, b in zip(alone, got))
