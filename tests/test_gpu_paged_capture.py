"""Bad pages under stream capture: recorded by every replay, when a PagedKV
was made before."""
import pytest
import torch

from rec_b200 import paged

pytestmark = pytest.mark.gpu


def inputs():
    k = torch.randn(4, 1, 16, 64, device="cuda").bfloat16()
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    table = torch.tensor([[0, 9]], device="cuda", dtype=torch.int32)  # page 9 is not there
    return k, q, table, torch.tensor([30], device="cuda", dtype=torch.int32)


def capture(call):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def test_a_first_call_under_capture_is_recorded(monkeypatch):
    monkeypatch.setattr(paged, "_status", {})
    k, q, table, n = inputs()
    cache, out = paged.PagedKV(k, k), torch.zeros_like(q)
    graph = capture(lambda: paged.paged_attn_decode(cache, q, table, n, out=out))
    paged.check_status()
    for _ in range(2):
        graph.replay()
        graph.replay()
        with pytest.raises(RuntimeError, match="status 5"):
            paged.check_status()
        paged.check_status()
    assert bool(out.any())


def test_a_capture_without_a_record_warns(monkeypatch):
    monkeypatch.setattr(paged, "_status", {})
    k, q, table, n = inputs()
    out = torch.zeros_like(q)
    with pytest.warns(RuntimeWarning, match="not recorded"):
        graph = capture(lambda: paged.paged_attn_decode(paged.PagedKV(k, k), q, table, n, out=out))
    graph.replay()
    paged.check_status()
    assert bool(out.any())
