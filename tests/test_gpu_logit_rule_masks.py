"""The allow mask is words of bits: a mask of numbers is refused."""
import pytest
import torch

from rec_b200 import sampling

pytestmark = pytest.mark.gpu


def test_masks_of_numbers_are_refused():
    logits = torch.randn(2, 64, device="cuda")
    words = torch.full((2, 2), -1, device="cuda", dtype=torch.int32)
    for allow in (words, words.view(torch.uint32)):
        assert torch.equal(sampling.process_logits(logits, allow=allow), logits)
    for allow in (torch.ones(2, 64, device="cuda"), words.float(), torch.ones(2, 64, device="cuda", dtype=torch.bool)):
        with pytest.raises(ValueError, match="words"):
            sampling.process_logits(logits, allow=allow)
