"""The status word of beam selection, with waits that may give up."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.gpu_util import lib, ok, stream  # noqa: E402
from tests.paged_util import scratch, status_word  # noqa: E402
from tests.test_gpu_h_beam_search import check_select, plain_select  # noqa: E402
from tnsr_b200 import _native  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_waits_that_give_up_are_told_and_the_next_call_is_whole(dtype):
    groups, beams, vocab, keep = 20, 5, 40001, 6
    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(groups * beams, vocab, generator=gen).to(dtype)
    scores = -torch.rand(groups * beams, generator=gen)
    want = plain_select(logits, scores, None, groups, beams, keep, 1)
    d_logits, d_scores, status = logits.cuda(), scores.cuda(), status_word()
    out = [torch.zeros((groups, keep), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    done = torch.zeros((groups, keep), dtype=torch.uint8, device="cuda")
    work = scratch(lib().tnsr_b200_beam_select_workspace(groups, beams, vocab, keep))
    args = _native.BeamSelectArgs(logits=d_logits.data_ptr(), scores=d_scores.data_ptr(), next_scores=out[0].data_ptr(), tokens=out[1].data_ptr(),
                                  parents=out[2].data_ptr(), next_finished=done.data_ptr(), workspace=work.data_ptr(), workspace_bytes=work.numel(), logits_ld=vocab,
                                  groups=groups, beams=beams, vocab=vocab, keep=keep, end_token=1, dtype=0 if dtype == torch.float32 else 1,
                                  d_status=status.data_ptr())
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")

    def call(limit):
        flush.zero_()                       # the logits come from memory
        status.zero_()
        torch.cuda.synchronize()
        assert lib().tnsr_b200_set_wait_limit_ns(limit) == 0
        try:
            ok(lib().tnsr_b200_beam_select(C.byref(args), stream()))
            torch.cuda.synchronize()
        finally:
            assert lib().tnsr_b200_set_wait_limit_ns(2_000_000_000) == 0
        assert int(status[0]) in ((0, 2) if limit == 1000 else (0,))
        if int(status[0]) == 0:             # nothing is wrong in silence
            check_select([t.cpu().numpy() for t in out] + [done.cpu().numpy()], want)
        else:
            assert np.all(out[2].cpu().numpy() // beams == np.arange(groups)[:, None])
        return int(status[0])

    for _ in range(8):
        call(1000)
        call(2_000_000_000)
