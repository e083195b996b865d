"""GPU: eos ids outside 32 bits are what they say, not their low half."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_eos_ids_that_do_not_fit():
    from vault_b200 import beam_select
    from vault_b200._lib import EngineError
    g = torch.Generator().manual_seed(1)
    logits, scores = torch.randn(2, 3, 500, generator=g).cuda(), torch.zeros(2, 3, device="cuda")
    finished = torch.zeros(2, 3, dtype=torch.uint8, device="cuda")
    finished[0, 1] = 1
    for eos in (500, 2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 64 + 7):
        with pytest.raises(EngineError, match="eos_id"):
            beam_select(logits, scores, finished, eos)
    want = beam_select(logits, scores, finished, -1)
    for eos in (-2, -2 ** 31, 7 - 2 ** 32, 7 - 2 ** 64):
        assert all(torch.equal(a, b) for a, b in zip(beam_select(logits, scores, finished, eos), want))
