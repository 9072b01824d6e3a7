"""One to three units of a head's slots, whole in a block or split and joined:
the sizes on both sides of that choice, against float64 forms."""
import pytest

from tests.test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,d,unit", [("bf16", 64, 192), ("fp16", 128, 192), ("bf16", 256, 128), ("k8v8", 128, 384),
                                         ("k4v4", 64, 384), ("k8v4", 256, 128)])
@pytest.mark.parametrize("units", [1, 2, 3, 4])
def test_sizes_around_whole_heads(kind, d, unit, units):
    for n in (units * unit - 1, units * unit, units * unit + 1):
        check_attention(kind, 8, 2, d, 64, [n], seed=n, sinks=True, weights=True)
        check_attention(kind, 8, 2, d, 64, [n, 3, n // 2], seed=n, window=unit + 1)
