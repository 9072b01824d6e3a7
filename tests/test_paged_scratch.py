"""The scratch of the batched calls, on the CPU with a stand-in for the
library: it stays alive until the call's launches, and two threads on one
stream do not meet in it."""
import threading
import types
import weakref

import pytest
import torch

from rec_b200 import paged


class Torch:
    """torch, with devices on the CPU; keeps weak references to what it allocates."""

    def __init__(self):
        self.made = {}

    def __getattr__(self, name):
        return getattr(torch, name)

    def device(self, *_):
        return torch.device("cpu")

    def _keep(self, t):
        self.made[t.data_ptr()] = weakref.ref(t)
        return t

    def empty(self, *a, **k):
        return self._keep(torch.empty(*a, **k))

    def zeros(self, *a, **k):
        return self._keep(torch.zeros(*a, **k))

    def alive(self, at):
        return self.made[at]() is not None


class Library:
    """Two launches a call, as the real one makes; `between` runs after the
    first of them."""

    def __init__(self):
        self.inside, self.most, self.seen = 0, 0, []
        self.between = lambda: None

    def rec_paged_attn_workspace_bytes(self, kv, table, hq, weights, counters):
        counters._obj.value = 5000 * hq
        return 10000 * hq

    def rec_paged_evict_workspace_bytes(self, kv, table, budget):
        return 1000 * budget

    def rec_paged_attn_decode(self, kv, table, a, ws, ws_bytes, counters, counter_bytes, status, stream):
        return self._run(ws, counters)

    def rec_paged_evict(self, kv, table, e, ws, ws_bytes, status, stream):
        return self._run(ws)

    def _run(self, *buffers):
        self.inside += 1
        self.most = max(self.most, self.inside)
        self.between()
        self.seen.append(all(self.torch.alive(b) for b in buffers))
        self.inside -= 1
        return 0


@pytest.fixture
def fake(monkeypatch):
    library = Library()
    library.torch = Torch()
    for name, x in dict(lib=lambda: library, torch=library.torch, _scratch={}, _sizes={}, _capturing=lambda: False,
                        _current_device=lambda: -1, _raw_stream=lambda i: 0, _status_ptr=lambda i: None).items():
        monkeypatch.setattr(paged, name, x)
    return library


CACHE = types.SimpleNamespace(_index=-1, head_dim=8, dtype=torch.bfloat16, shape=(4, 1, 16), bits=(16, 16), _desc=b"")
TABLE, LENGTHS = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


def attend(hq):
    paged.paged_attn_decode(CACHE, torch.zeros(2, hq, 8, dtype=torch.bfloat16), TABLE, LENGTHS)


def evict(budget):
    paged.paged_evict(CACHE, TABLE, LENGTHS, budget, torch.zeros(4, 1, 16))


@pytest.mark.parametrize("call", [attend, evict])
def test_a_larger_call_of_another_thread_waits(fake, call):
    call(8)
    other = threading.Thread(target=call, args=(64,))

    def between():
        if not other.ident:
            other.start()
            other.join(0.3)  # it must not get through meanwhile

    fake.between = between
    call(8)
    other.join(10)
    assert not other.is_alive()
    assert fake.most == 1 and fake.seen == [True, True, True]


@pytest.mark.parametrize("call", [attend, evict])
def test_a_captured_call_holds_its_own(fake, monkeypatch, call):
    monkeypatch.setattr(paged, "_capturing", lambda: True)
    call(8)
    call(64)
    assert fake.seen == [True, True] and not paged._scratch


def test_a_refusal_leaves_the_lock_open(fake, monkeypatch):
    monkeypatch.setattr(fake, "between", lambda: 1 / 0)
    for _ in range(2):
        with pytest.raises(ZeroDivisionError):
            attend(8)
