"""Words are words: fp32 tensors, 32 bits too, are refused where codes or
masks are wanted."""
import pytest
import torch

from rec_b200 import paged

pytestmark = pytest.mark.gpu


def test_code_words():
    scales = [torch.zeros(2, 1, 16, 1, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    words = torch.zeros(2, 1, 16, 16, device="cuda", dtype=torch.int32)
    for k, v in ((words, words), (words.view(torch.uint32), words.view(torch.uint32)), (words, words.view(torch.uint32))):
        assert paged.PagedKV(k, v, *scales).bits == (8, 8)
    for k, v in ((words.float(), words.float()), (words, words.float()), (words.float(), words),
                 (words.view(torch.float32), words.view(torch.float32))):
        with pytest.raises(ValueError, match="code words"):
            paged.PagedKV(k, v, *scales)
