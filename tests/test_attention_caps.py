"""Capped scores at caps of every size: softcap * tanh(score / softcap) of a cap far above the
scores is the score itself, and of one far below them the cap."""
import pytest

torch = pytest.importorskip("torch")

import kv_helpers  # noqa: E402
from bybylang_b200 import _lib  # noqa: E402
from test_attention_accuracy import check  # noqa: E402

pytestmark = pytest.mark.gpu
GEMV, TC, SIMT = _lib.ROUTE_GEMV, _lib.ROUTE_TC, _lib.ROUTE_SIMT


@pytest.mark.parametrize("route,dtype", [(GEMV, torch.bfloat16), (GEMV, torch.float32), (TC, torch.bfloat16), (SIMT, torch.bfloat16),
                                         (SIMT, torch.float32)])
@pytest.mark.parametrize("cap", [1e-40, 1e-30, 1e-3, 0.7, 3.0, 50.0, 250.0, 260.0, 1e3, 1e4, 1e5, 1e6, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("spread", [1.0, 6.0])
def test_caps(cap, spread, route, dtype):
    """Scores of order 1, and of order 6 with some beyond 20: on both sides of where a cap bends."""
    for lens, dim in (([(1, 900), (1, 65)], 128), ([(3, 40), (70, 300)], 64)):
        bt = kv_helpers.Batch(lens, page=16, heads=8, kv_heads=2, dim=dim, seed=int(spread) + dim, spread=spread)
        check(bt, route, dtype, size=spread, softcap=cap)


@pytest.mark.parametrize("route", [GEMV, TC, SIMT])
def test_caps_with_a_negative_scale_and_slopes(route):
    bt = kv_helpers.Batch([(2, 300), (90, 200)], page=32, heads=4, kv_heads=1, dim=64, seed=5)
    for cap in (2.0, 1e6):
        check(bt, route, torch.bfloat16, size=2.0, softcap=cap, scale=-0.2)
        check(bt, route, torch.bfloat16, softcap=cap, slopes=torch.tensor([0.5, 0.1, 0.01, 0.0]))


@pytest.mark.parametrize("route,dtype", [(GEMV, torch.bfloat16), (GEMV, torch.float32), (TC, torch.bfloat16), (SIMT, torch.float32)])
@pytest.mark.parametrize("cap", [1e-40, 1e-3, 1e38])
def test_scores_of_zero(cap, route, dtype):
    """A query of zeros sees the mean of the values under any cap, 1 / cap in range or not."""
    bt = kv_helpers.Batch([(1, 70), (50, 200)], page=16, heads=4, kv_heads=2, dim=64, seed=6)
    bt.q = torch.zeros_like(bt.q)
    check(bt, route, dtype, softcap=cap)
