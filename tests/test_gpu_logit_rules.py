"""Per-row logits rules on the GPU (process_logits).

Every output equals, bit for bit, the rules in fp32 steps (one rounding each,
in the documented order) rounded once to the logits' type.  fp32 logits are
also held to a float64 form: at most six fp32 operations, 6 * 2^-24 of the
largest magnitude that enters a value, and the final rounding, 2^-24."""
import numpy as np
import pytest
import torch

from rec_b200 import sampling
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def case(dtype, B, V, n, m, *, mask, seed=0, spread=None, in_place=False, offset=0):
    rng = np.random.default_rng(seed)
    wide = torch.from_numpy(5 * rng.standard_normal((B, V + 13)).astype(np.float32)).cuda().to(dtype)
    logits = wide[:, offset:offset + V]
    hist = rng.integers(-2, spread or V + 2, (B, n)).astype(np.int32)
    hl = rng.integers(0, n + 1, B).astype(np.int32)
    pl = (hl * rng.random(B)).astype(np.int32)
    rep, freq, pres = (rng.random(B).astype(np.float32) + o for o in (0.7, 0.0, -0.5))
    rep, freq, pres = (x.astype(np.float32) for x in (rep, freq, pres))
    ids = rng.integers(-1, min(V, 50) + 1, (B, m)).astype(np.int32)
    val = rng.standard_normal((B, m)).astype(np.float32)
    words = (V + 31) // 32 + 1
    allow = rng.integers(0, 2 ** 32, (B, words), dtype=np.uint32)
    if mask:
        allow[0] = 0  # a row with nothing allowed
    before = logits.double().cpu().numpy()
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    out = sampling.process_logits(
        logits, history=t(hist), history_len=t(hl), prompt_len=t(pl), repetition=t(rep), frequency=t(freq),
        presence=t(pres), bias_ids=t(ids) if m else None, bias_values=t(val) if m else None,
        allow=t(allow.view(np.int32)) if mask else None, out=logits if in_place else None)
    got = out.double().cpu().numpy()
    for b in range(B):
        ok = ((allow[b][:, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(-1)[:V].astype(bool) if mask else None
        want = ref.logit_rules(before[b], hist[b, :hl[b]].tolist(), int(pl[b]), float(rep[b]), float(freq[b]),
                               float(pres[b]), list(zip(ids[b].tolist(), val[b].tolist())), ok)
        steps = ref.logit_rules(before[b], hist[b, :hl[b]].tolist(), int(pl[b]), rep[b], freq[b], pres[b],
                                list(zip(ids[b].tolist(), val[b].tolist())), ok, np.float32)
        assert torch.equal(out[b].cpu(), torch.from_numpy(steps).to(dtype))
        if dtype == torch.float32:
            inf = np.isinf(want)
            assert (got[b][inf] == want[inf]).all()
            top = np.abs(before[b]).max() * 2 + n + 8
            assert (np.abs(got[b] - want)[~inf] <= (np.abs(want) + 6 * top)[~inf] * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 31, 32, 1000, 8192, 8193, 50257])
@pytest.mark.parametrize("mask", [False, True])
def test_rules(dtype, V, mask):
    case(dtype, 3, V, 40, 6, mask=mask, seed=V)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_rows_at_any_alignment(dtype, offset):
    case(dtype, 4, 4099, 100, 20, mask=True, offset=offset, in_place=True, seed=offset)
    case(dtype, 4, 4099, 100, 20, mask=False, offset=offset, seed=offset)


@pytest.mark.parametrize("n,spread", [(0, None), (1, 1), (5000, 3), (20000, None), (20000, 100)])
def test_histories(n, spread):
    """Empty, one id, long, and ids that repeat thousands of times."""
    case(torch.float32, 2, 3001, n, 0, mask=False, spread=spread, seed=n)


@pytest.mark.parametrize("m", [0, 1, 300, 8190])
def test_biases(m):
    """Entries of the same id: the last one counts."""
    case(torch.float32, 2, 3001, 10, m, mask=False, seed=m)


@pytest.mark.parametrize("B", [1, 7, 64, 200])
def test_batches(B):
    case(torch.bfloat16, B, 2000, 64, 4, mask=True, seed=B)


def test_special_values():
    """Infinities stay, NaN stays unless it is not allowed, and -inf + bias is -inf."""
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), float("nan"), 1.0, -1.0]], device="cuda")
    i32 = dict(device="cuda", dtype=torch.int32)
    out = sampling.process_logits(x, history=torch.tensor([[0, 1, 2, 4, 5, 5]], **i32), repetition=2.0, frequency=0.5,
                                  presence=0.25, bias_ids=torch.tensor([[1]], **i32),
                                  bias_values=torch.full((1, 1), 9.0, device="cuda"),
                                  allow=torch.tensor([[0b110111]], **i32))
    o = out.cpu()[0]
    assert o[0] == float("inf") and o[1] == float("-inf") and torch.isnan(o[2]) and o[3] == float("-inf")
    assert o[4] == 1.0 / 2 - 0.5 - 0.25 and o[5] == -2.0 - 1.0 - 0.25


def test_numbers_equal_tensors_and_nothing_is_a_copy():
    x = torch.randn(3, 777, device="cuda").bfloat16()
    h = torch.randint(0, 777, (3, 50), device="cuda", dtype=torch.int32)
    full = lambda v: torch.full((3,), v, device="cuda")  # noqa: E731
    a = sampling.process_logits(x, history=h, repetition=1.3, frequency=0.2, presence=0.1)
    b = sampling.process_logits(x, history=h, repetition=full(1.3), frequency=full(0.2), presence=full(0.1))
    assert torch.equal(a, b) and torch.equal(sampling.process_logits(x), x)
    assert torch.equal(sampling.process_logits(x, history=h), x)


def test_same_ids_as_the_sampler():
    """Penalties and mask here, then the sampler without them, against the
    sampler's own (one rule for all rows), on fp32-exact values."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randint(-64, 65, (4, 5000), device="cuda", generator=g).float() / 8).bfloat16()
    h = torch.randint(0, 5000, (4, 300), device="cuda", dtype=torch.int32, generator=g)
    allow = torch.randint(-2 ** 31, 2 ** 31, (4, 157), device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    want = sampling.sample_logits(x, sampling.params(repetition_penalty=2.0, presence_penalty=0.5), history=h, allow=allow)
    got = sampling.sample_logits(sampling.process_logits(x, history=h, repetition=2.0, presence=0.5, allow=allow),
                                 sampling.params())
    assert torch.equal(got, want)
