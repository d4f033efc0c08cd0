"""Launches of many row tiles or sequences."""
import pytest

torch = pytest.importorskip("torch")

import kv_helpers  # noqa: E402
from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402
from rounding_helpers import scores_off  # noqa: E402
from test_attention_accuracy import check  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV])
def test_more_row_tiles_than_a_grid_has_rows(route):
    """A call sized for 32768 new tokens of 4 heads a kv head, 32 kv heads: 65536 tiles of 64 rows."""
    bt = kv_helpers.Batch([(40, 300), (1, 20)], page=16, heads=128, kv_heads=32, dim=64, seed=2)
    check(bt, route, torch.float32, max_q=32768, max_kv=40000)
    bt = kv_helpers.Batch([(3, 30)], page=16, heads=32, kv_heads=16, dim=256, seed=3)
    check(bt, route, torch.bfloat16, max_q=131072, max_kv=131072)


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_sequences_than_a_grid_has_layers(route, dtype):
    """70000 sequences of one token: each gives its own value."""
    n, dim = 70000, 8
    v = torch.randn(n, 1, 1, dim, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    k, q = torch.ones_like(v), torch.ones(n, 1, dim, dtype=torch.bfloat16, device=DEV)
    table = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=DEV)[:, None]
    starts = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    out = kv.paged_attention(q, k, v, table, starts, torch.ones(n, dtype=torch.int32, device=DEV), max_q=1, max_kv=1, out_dtype=dtype, route=route)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert torch.equal(out[:, 0], v[:, 0, 0].flip(0).to(dtype))


@pytest.mark.parametrize("dim,heads,tokens", [(8, 64, 65537), (136, 32, 131073)])
def test_prompts_of_more_row_tiles_than_a_grid_has_rows(dim, heads, tokens):
    """Tokens x heads in tiles of 64 rows, past 65535 of them, under a window: the tensor-core-free
    routes against each other."""
    page, n = 64, -(-tokens // 64)
    g = torch.Generator(device=DEV).manual_seed(7)
    k, v = (torch.randn(n, 1 if dim > 128 else heads, page, dim, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(tokens, heads, dim, generator=g, device=DEV).to(torch.bfloat16)
    ints = dict(dtype=torch.int32, device=DEV)
    batch = k, v, torch.randperm(n, generator=g, device=DEV).to(torch.int32)[None], torch.tensor([0, tokens], **ints), torch.tensor([tokens], **ints)
    got, want = (kv.paged_attention(q, *batch, max_q=tokens, max_kv=tokens, window=9, out_dtype=torch.float32, route=r)
                 for r in (_lib.ROUTE_AUTO, _lib.ROUTE_SIMT))
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    # both exact to fp32: scores_off of each, of values up to 6
    assert float((got - want).abs().max()) <= 2 * scores_off(1.0) * 6
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV, _lib.ROUTE_TC])
def test_a_bound_on_the_new_tokens_may_be_any(route):
    bt = kv_helpers.Batch([(3, 40), (70, 200)], page=16, heads=8, kv_heads=2, dim=64, seed=8)
    for max_q in (73, 1 << 20, 2 ** 31 - 1):
        check(bt, route, torch.bfloat16, max_q=max_q)


@pytest.mark.parametrize("route", [_lib.ROUTE_GEMV, _lib.ROUTE_TC, _lib.ROUTE_SIMT])
def test_the_last_positions_of_the_longest_table(route):
    """What a window sees does not depend on where it lies: the same cache 2^31 - 12000 positions on."""
    page, pages = 4096, 524285
    bt = kv_helpers.Batch([(1, 4000), (40, 4090)], page=page, heads=8, kv_heads=2, dim=64, seed=9)
    call = dict(max_q=40, window=300, out_dtype=torch.bfloat16, route=route)
    want = kv.paged_attention(bt.q, *bt.args(), max_kv=4096, **call)
    table = torch.full((2, pages), -1, dtype=torch.int32, device=DEV)
    table[:, -1] = bt.table[:, 0]
    far = bt.kv_lens + (pages - 1) * page
    got = kv.paged_attention(bt.q, bt.k, bt.v, table, bt.q_start, far, max_kv=pages * page, **call)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert torch.equal(got, want) and torch.isfinite(got).all() and got.any()


@pytest.mark.parametrize("route", [_lib.ROUTE_AUTO, _lib.ROUTE_GEMV, _lib.ROUTE_SIMT])
def test_one_query_for_every_token(route):
    """q expanded over the tokens (stride 0): the tensor-core route cannot step by it and is not taken."""
    bt = kv_helpers.Batch([(70, 200), (3, 40)], page=16, heads=8, kv_heads=2, dim=64, seed=10)
    bt.q = bt.q[:1].expand(bt.tokens, 8, 64)
    assert bt.q.stride(0) == 0
    check(bt, route, torch.bfloat16)


def test_one_query_for_every_token_is_refused_on_the_tensor_cores():
    bt = kv_helpers.Batch([(70, 200)], page=16, heads=8, kv_heads=2, dim=64, seed=10)
    with pytest.raises(_lib.BybyCudaError, match="token stride of q"):
        kv.paged_attention(bt.q[:1].expand(70, 8, 64), *bt.args(), max_q=70, max_kv=200, route=_lib.ROUTE_TC)
    one = kv_helpers.Batch([(1, 200)], page=16, heads=8, kv_heads=2, dim=64, seed=10)     # a single token needs none
    one.q = one.q.as_strided((1, 8, 64), (0, 64, 1))
    check(one, _lib.ROUTE_TC, torch.bfloat16)
