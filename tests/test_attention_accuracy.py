"""paged_attention within what its roundings can do, element by element: lost or doubled keys in
long caches, caps of any size, and launches sized for far more than there is."""
import pytest

torch = pytest.importorskip("torch")

import kv_helpers  # noqa: E402
from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402
from rounding_helpers import bf16_bound, exact_and_spread, f32_bound  # noqa: E402

DEV = "cuda:0"
AUTO, GEMV, TC, SIMT = _lib.ROUTE_AUTO, _lib.ROUTE_GEMV, _lib.ROUTE_TC, _lib.ROUTE_SIMT


def check(bt, route, dtype, max_q=None, max_kv=None, size=1.0, **mods):
    out = torch.full((bt.tokens, bt.heads, bt.dim), float("nan"), dtype=dtype, device=DEV)
    kw = dict(mods)
    prefix = kw.pop("prefix", None)
    if prefix is not None:
        kw["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32, device=DEV)
    if kw.get("slopes") is not None:
        kw["slopes"] = kw["slopes"].to(DEV)
    kv.paged_attention(bt.q, *bt.args(), max_q=max_q or bt.max_q, max_kv=max_kv or bt.max_kv, out=out, route=route, **kw)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    want, total, spread = exact_and_spread(bt, **mods)
    bound = (bf16_bound if dtype == torch.bfloat16 else f32_bound)(want, total, spread, size)
    over = (out.cpu().double() - want).abs() - bound
    assert (over <= 0).all(), f"{float(over.max()):.2e} above the bound, {int((over > 0).sum())} of {over.numel()}"


# ---- lost keys -----------------------------------------------------------------------------

LONG = [dict(lens=[(1, 9000), (2, 700), (1, 3)], page=16, heads=8, kv_heads=1, dim=64, seed=13),
        dict(lens=[(40, 5000)], page=64, heads=8, kv_heads=2, dim=128, seed=12),
        dict(lens=[(1, 20000)], page=32, heads=4, kv_heads=4, dim=128, seed=14),
        dict(lens=[(130, 4000), (5, 8000)], page=128, heads=8, kv_heads=1, dim=64, seed=15)]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{len(c['lens'])}x{c['lens'][0][1]}")
def test_the_bounds_see_a_lost_block(case, monkeypatch):
    """On the CPU: a kernel that lost 128 keys anywhere in a cache would be outside of both bounds."""
    monkeypatch.setattr(kv_helpers, "DEV", "cpu")
    bt = kv_helpers.Batch(**case)
    want, total, spread = exact_and_spread(bt)
    b = max(range(len(bt.lens)), key=lambda i: bt.lens[i][1])
    rows = slice(bt.starts[b], bt.starts[b + 1])
    for first in (0, bt.lens[b][1] // 2, bt.lens[b][1] - bt.lens[b][0] - 128):
        lost = exact_and_spread(bt, drop=(b, first, first + 128))[0]
        for bound in (bf16_bound, f32_bound):
            over = (lost - want).abs() > bound(want, total, spread)
            assert over[rows].flatten(1).any(1).all()       # in every row


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("route", [AUTO, GEMV, TC, SIMT])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{len(c['lens'])}x{c['lens'][0][1]}")
def test_long_caches(case, route, dtype):
    if route == TC and dtype == torch.float32:
        pytest.skip("no tensor-core form of an fp32 output")
    bt = kv_helpers.Batch(**case)
    check(bt, route, dtype)
    check(bt, route, dtype, window=2500)
    check(bt, route, dtype, softcap=25.0)


@pytest.mark.gpu
@pytest.mark.parametrize("route", [AUTO, GEMV, TC])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 128, 128), (8, 1, 64, 32), (6, 2, 96, 16)])
def test_long_prompts(heads, kv_heads, dim, page, route):
    bt = kv_helpers.Batch([(700, 3000), (257, 257), (300, 1500)], page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=dim)
    check(bt, route, torch.bfloat16)
    check(bt, route, torch.bfloat16, window=900, prefix=[40, 100, 0])
