"""Launches sized for many row tiles."""
import pytest

torch = pytest.importorskip("torch")

import kv_helpers  # noqa: E402
from bybylang_b200 import _lib  # noqa: E402
from test_attention_accuracy import check  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV])
def test_more_row_tiles_than_a_grid_has_rows(route):
    """A call sized for 32768 new tokens of 4 heads a kv head, 32 kv heads: 65536 tiles of 64 rows."""
    bt = kv_helpers.Batch([(40, 300), (1, 20)], page=16, heads=128, kv_heads=32, dim=64, seed=2)
    check(bt, route, torch.float32, max_q=32768, max_kv=40000)
    bt = kv_helpers.Batch([(3, 30)], page=16, heads=32, kv_heads=16, dim=256, seed=3)
    check(bt, route, torch.bfloat16, max_q=131072, max_kv=131072)


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV, _lib.ROUTE_TC])
def test_a_bound_on_the_new_tokens_may_be_any(route):
    bt = kv_helpers.Batch([(3, 40), (70, 200)], page=16, heads=8, kv_heads=2, dim=64, seed=8)
    for max_q in (73, 1 << 20, 2 ** 31 - 1):
        check(bt, route, torch.bfloat16, max_q=max_q)
