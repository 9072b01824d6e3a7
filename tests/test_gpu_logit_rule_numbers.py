"""Rules given as plain numbers (process_logits) equal the same rules given as
tensors, bit for bit: the lengths as well as the penalties."""
import pytest
import torch

from rec_b200 import sampling

pytestmark = pytest.mark.gpu


def inputs(B=3, V=500, n=40):
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randn(B, V, device="cuda", generator=g)
    return logits, torch.randint(0, V, (B, n), device="cuda", generator=g, dtype=torch.int32)


@pytest.mark.parametrize("rules", [dict(history_len=10, prompt_len=4, repetition=1.1),
                                   dict(history_len=25, frequency=0.3, presence=0.2),
                                   dict(prompt_len=7, repetition=1.3, frequency=0.5),
                                   dict(history_len=0, repetition=2.0),
                                   dict(history_len=33, prompt_len=12, repetition=1.2, frequency=0.4, presence=0.1)],
                         ids=str)
def test_numbers_equal_tensors(rules):
    logits, history = inputs()
    B = len(logits)
    tensors = {name: torch.full((B,), x, device="cuda", dtype=torch.int32 if name.endswith("_len") else torch.float32)
               for name, x in rules.items()}
    want = sampling.process_logits(logits, history=history, **tensors)
    assert torch.equal(sampling.process_logits(logits, history=history, **rules), want)


def test_a_number_as_length_stops_there():
    """Only the ids before it are penalised."""
    logits, history = inputs()
    out = sampling.process_logits(logits, history=history, history_len=10, prompt_len=4, repetition=1.1)
    for b in range(len(logits)):
        changed = set(torch.nonzero(out[b] != logits[b]).flatten().tolist())
        assert changed == set(history[b, :10].tolist())
