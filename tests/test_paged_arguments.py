"""Arguments of the batched calls that the Python side answers for, on the CPU
with a stand-in for the library."""
import types

import pytest
import torch

from rec_b200 import abi, paged


class Library:
    def __init__(self):
        self.attn, self.evicted = [], []

    def rec_paged_attn_workspace_bytes(self, kv, table, hq, weights, counters):
        counters._obj.value = 64
        return 512

    def rec_paged_evict_workspace_bytes(self, kv, table, budget):
        return 512

    def rec_paged_attn_decode(self, kv, table, a, *rest):
        self.attn.append(abi.RecPagedAttn.from_buffer_copy(a))
        return 0

    def rec_paged_evict(self, kv, table, e, *rest):
        self.evicted.append(abi.RecPagedEvict.from_buffer_copy(e))
        return 0


class Torch:
    """torch, with devices on the CPU; counts what it allocates."""

    def __init__(self):
        self.made = 0

    def __getattr__(self, name):
        return getattr(torch, name)

    def device(self, *_):
        return torch.device("cpu")

    def empty(self, *a, **k):
        self.made += 1
        return torch.empty(*a, **k)

    def zeros(self, *a, **k):
        self.made += 1
        return torch.zeros(*a, **k)


@pytest.fixture
def fake(monkeypatch):
    library = Library()
    library.torch = Torch()
    for name, x in dict(lib=lambda: library, torch=library.torch, _scratch={}, _sizes={}, _capturing=lambda: False,
                        _current_device=lambda: -1, _raw_stream=lambda i: 0, _status_ptr=lambda i: None).items():
        monkeypatch.setattr(paged, name, x)
    return library


CACHE = types.SimpleNamespace(_index=-1, head_dim=8, dtype=torch.bfloat16, shape=(4, 1, 16), bits=(16, 16), _desc=b"")


def attend(batch=2, width=4, heads=8, q=None, **over):
    q = torch.zeros(batch, heads, 8, dtype=torch.bfloat16) if q is None else q
    return paged.paged_attn_decode(CACHE, q, torch.zeros(batch, width, dtype=torch.int32),
                                   torch.zeros(batch, dtype=torch.int32), **over)


def evict(budget, batch=2, **over):
    return paged.paged_evict(CACHE, torch.zeros(batch, 4, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32), budget,
                             torch.zeros(4, 1, 16), **over)


@pytest.mark.parametrize("call", [lambda: attend(window=2 ** 31), lambda: attend(window=-2 ** 40), lambda: evict(2 ** 31),
                                  lambda: evict(-2 ** 31 - 1), lambda: evict(4, keep_below=2 ** 33)])
def test_numbers_out_of_range_are_value_errors(fake, call):
    with pytest.raises(ValueError, match="out of range"):
        call()
    assert not fake.attn and not fake.evicted


def test_the_largest_numbers_pass(fake):
    attend(window=2 ** 31 - 1, scale=1e30)
    evict(2 ** 31 - 1, keep_below=2 ** 31 - 1)
    assert fake.attn[0].window == fake.evicted[0].budget == fake.evicted[0].keep_below == 2 ** 31 - 1


def test_an_eviction_has_no_counters(fake, monkeypatch):
    """Under capture they would be cleared by every replay for nothing."""
    lengths = torch.zeros(2, dtype=torch.int32)
    for capturing in (False, True):
        monkeypatch.setattr(paged, "_capturing", lambda: capturing)
        fake.torch.made = 0
        evict(16, lengths_out=lengths)
        # the workspace, and the tensors that this file's `evict` makes through torch itself are not counted
        assert fake.torch.made == 1


@pytest.mark.parametrize("batch,heads,strides", [(1, 8, (3, 8, 1)), (2, 1, (8, 5, 1)), (1, 1, (3, 5, 1)), (2, 8, (64, 8, 1))])
def test_strides_that_no_address_uses_are_not_checked(fake, batch, heads, strides):
    """A dimension of one entry may have any stride (a slice, an expanded
    view); the library wants multiples of 8 elements."""
    q, out = (torch.zeros(256, dtype=torch.bfloat16).as_strided((batch, heads, 8), strides) for _ in range(2))
    attend(batch=batch, q=q, out=out)
    a = fake.attn[0]
    for got in ((a.q_batch_stride, a.q_head_stride), (a.out_batch_stride, a.out_head_stride)):
        assert got == (strides[0] if batch > 1 else 0, strides[1] if heads > 1 else 0)


def test_an_empty_batch_is_nothing_to_do(fake):
    """As for process_logits; arguments that do not match are still refused."""
    assert attend(batch=0).shape == (0, 8, 8)
    assert evict(16, batch=0).shape == (0,)
    rows = torch.zeros(0, 1, 8, dtype=torch.bfloat16)
    none, cu = torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    paged.paged_append(CACHE, rows, rows, torch.zeros(0, 4, dtype=torch.int32), none, cu)
    assert not fake.attn and not fake.evicted and fake.torch.made == 0
    with pytest.raises(ValueError):
        attend(batch=0, lse=torch.zeros(1, 8))
    with pytest.raises(ValueError):
        evict(2 ** 40, batch=0)


def test_the_remembered_sizes_are_bounded(fake):
    for width in range(5000):
        attend(batch=1, width=width + 1, heads=1)
    assert 0 < len(paged._sizes) <= 4096 and len(fake.attn) == 5000


def test_a_captured_call_takes_what_it_needs(fake, monkeypatch):
    """Not the size of the largest call so far, which a graph would keep."""
    sizes = []
    monkeypatch.setattr(fake, "rec_paged_evict_workspace_bytes", lambda kv, table, budget: 1000 * budget)
    monkeypatch.setattr(fake, "rec_paged_evict", lambda kv, table, e, ws, n, *rest: sizes.append(n) or 0)
    evict(900)
    evict(5)
    monkeypatch.setattr(paged, "_capturing", lambda: True)
    evict(5)
    assert sizes == [900000, 900000, 5000]
