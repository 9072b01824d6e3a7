"""The example that runs append, attention, eviction, the logits' rules and
the sampler together.

Without eviction its logits are those of the same weights in float64 over the
whole history.  What differs: q, k, v and the attention's output are rounded
to bf16 (2^-9 relatively), the rest is fp32.  A score of size |s| moves by at
most 2 * 2^-9 |s|, with |s| below 8 here, so a weight by 2^-5 and the
attention's branch by 2^-5 plus the roundings of v and o; both layers' branches
are no larger than the stream that they join, hence 2^-3 for the two, of which
the errors' signs leave a small part: the bound is 2^-4 in the 2-norm."""
import pytest
import torch

from rec_b200 import paged, sampling

pytestmark = pytest.mark.gpu


def plain_logits(model, tokens):
    """float64, one session, all tokens at once; logits of the last."""
    positions = torch.arange(len(tokens), device="cuda")
    x = model.embedding.double()[torch.tensor(tokens, device="cuda")]
    causal = positions[None, :] > positions[:, None]
    for block in model.blocks:
        wide = {name: w.double() for name, w in block.items()}
        q, k, v = model.qkv(wide, x, positions)
        k, v = (t.repeat_interleave(model.heads // model.kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * model.head_dim ** -0.5
        assert float(s.abs().max()) < 8
        p = torch.softmax(s.masked_fill(causal, -torch.inf), -1)
        x = model.finish(wide, x, torch.einsum("hqk,khd->qhd", p, v))
    return 2.0 * model.norm(x[-1]) @ model.head.double().T


def test_equals_the_whole_history():
    from examples.paged_batch import Decoder, PagedBatch
    model = Decoder(seed=1)
    prompts = [[3], [7, 8, 9], list(range(100, 170))]
    batch = PagedBatch(model, 3, 500, slack=8)
    ids = batch.generate(prompts, 40, temperature=0.0, banned=(5, 6)).tolist()
    for b, p in enumerate(prompts):
        want = plain_logits(model, p + ids[b][:-1])
        assert float(torch.linalg.norm(batch.logits[b].double() - want) / torch.linalg.norm(want)) <= 2.0 ** -4
        assert not {5, 6} & set(ids[b])


@pytest.mark.parametrize("kv", ["bf16", "k8v8", "k8v4", "k4v4"])
def test_stays_within_its_budget(kv):
    from examples.paged_batch import Decoder, PagedBatch
    model = Decoder(seed=2)
    prompts = [[1], list(range(60)), list(range(200, 330))]
    batch = PagedBatch(model, 3, 64, slack=16, kv=kv, recent=20, first=3)
    ids = batch.generate(prompts, 90, seed=5)
    again = PagedBatch(model, 3, 64, slack=16, kv=kv, recent=20, first=3).generate(prompts, 90, seed=5)
    assert torch.equal(ids, again)
    assert ids.shape == (3, 90) and int(ids.min()) >= 0 and int(ids.max()) < 1000
    assert batch.positions.tolist() == [len(p) + 89 for p in prompts]
    assert max(batch.lengths.tolist()) < 64 + 16
    table = batch.table.tolist()
    for b, n in enumerate(batch.lengths.tolist()):
        for places in batch.places:
            for h in range(model.kv_heads):
                have = [int(places[table[b][t // 16], h, t % 16]) for t in range(n)]
                now = int(batch.positions[b])
                assert len(set(have)) == n
                assert set(range(3)) | set(range(now - 20, now)) <= set(have) <= set(range(now))


def test_bias_and_frequency_reach_the_sampler():
    from examples.paged_batch import Decoder, PagedBatch
    model = Decoder(seed=3)
    ids = PagedBatch(model, 2, 100).generate([[1], [2, 3]], 12, temperature=0.0, bias={17: 100.0, 18: 90.0},
                                             repetition=1.0, frequency=3.0, presence=0.0)
    # 17 leads by 10 and loses 3 an occurrence, so after its fourth 18 leads, and they take turns
    for row in ids.tolist():
        assert row[:3] == [17] * 3 and set(row) == {17, 18}


def test_refusals():
    from examples.paged_batch import Decoder, PagedBatch
    model = Decoder(layers=1)
    for bad in (dict(kv="k3v3"), dict(recent=100), dict(slack=0)):
        with pytest.raises(ValueError):
            PagedBatch(model, 2, 64, **bad)
    with pytest.raises(ValueError):
        PagedBatch(model, 2, 64).prefill([[1], []])


def test_positions_of_appended_rows():
    """first_positions gives the tokens' positions, the slots stay those of starts."""
    cache = paged.PagedKV.allocate(4, 2, 8, 64)
    k = torch.randn(5, 2, 64, device="cuda").bfloat16()
    i32 = dict(device="cuda", dtype=torch.int32)
    pos = torch.full((4, 2, 8), -1, **i32)
    paged.paged_append(cache, k, k, torch.tensor([[2, 0], [1, 3]], **i32), torch.tensor([6, 0], **i32),
                       torch.tensor([0, 3, 5], **i32), positions=pos, first_positions=torch.tensor([100, 2 ** 30], **i32))
    paged.check_status()
    want = torch.full((4, 2, 8), -1, **i32)
    want[2, :, 6], want[2, :, 7], want[0, :, 0] = 100, 101, 102
    want[1, :, 0], want[1, :, 1] = 2 ** 30, 2 ** 30 + 1
    assert torch.equal(pos, want)
    with pytest.raises(ValueError):
        paged.paged_append(cache, k, k, torch.zeros(2, 2, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32),
                           positions=pos, first_positions=torch.zeros(3, **i32))


def test_one_allow_mask_for_every_row():
    logits = torch.randn(5, 1003, device="cuda").bfloat16()
    words = torch.randint(-2 ** 31, 2 ** 31, (1, 32), device="cuda").int()
    assert torch.equal(sampling.process_logits(logits, allow=words.expand(5, -1)),
                       sampling.process_logits(logits, allow=words.repeat(5, 1)))
