"""The paged-cache operators against their definitions in 64 bits: rotary append, paged attention,
page copies, beam selection, at the sizes, layouts and masks where they can go wrong."""
import math

import pytest

torch = pytest.importorskip("torch")

from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402
from kv_helpers import DEV, Batch, attention64  # noqa: E402

pytestmark = pytest.mark.gpu

AUTO, GEMV, TC, SIMT = _lib.ROUTE_AUTO, _lib.ROUTE_GEMV, _lib.ROUTE_TC, _lib.ROUTE_SIMT


# ---- paged attention -----------------------------------------------------------------------
# Tolerances.  fp32 output: the score of a pair is an fp32 sum of products that are exact in fp32
# (|error| <= dim * 2^-24 * sum |q k| * scale, about 1e-5 at these sizes), which moves a
# probability by that relative amount; probabilities keep 16 bits at least (2^-16), their sum is
# fp32.  Together below 6e-5 of the largest value the row can see.  bf16 (8 significant bits, so a
# rounding is up to 2^-8 of the value) output: each probability and the output are rounded once.
F32_TOL = 6e-5
BF16_TOL = 2.0 ** -7 + F32_TOL


def tc_runs(bt, out_dtype):
    return bt.dim <= 128 and out_dtype == torch.bfloat16 and bt.page % 8 == 0 and (128 % bt.page == 0 or bt.page % 128 == 0)


def check(bt, route, out_dtype=torch.float32, **mods):
    kw = dict(mods)
    if kw.get("slopes") is not None:
        kw["slopes"] = kw["slopes"].to(DEV)
    if route == TC and not tc_runs(bt, out_dtype):
        pytest.skip("no tensor-core form of this shape")
    prefix = kw.pop("prefix", None)
    if prefix is not None:
        kw["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32, device=DEV)
    out = torch.full((bt.tokens, bt.heads, bt.dim), float("nan"), dtype=out_dtype, device=DEV)
    kv.paged_attention(bt.q, *bt.args(), max_q=bt.max_q, max_kv=bt.max_kv, out=out, route=route, **kw)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    want = attention64(bt, **mods)
    top = max([1e-30] + [float(v.abs().max()) for v in bt.values if v.numel()])
    err = float((out.cpu().double() - want).abs().max()) if bt.tokens else 0.0
    assert err <= (F32_TOL if out_dtype == torch.float32 else BF16_TOL) * top, f"{err:.3e} of {top:.2f}"
    return out


RAGGED = [(5, 37), (0, 11), (1, 1), (64, 64), (17, 300), (3, 0), (130, 131), (1, 257)]
DECODE = [(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 0)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("route", [AUTO, GEMV, SIMT, TC])
@pytest.mark.parametrize("dim,page,heads,kv_heads", [(64, 16, 8, 2), (128, 64, 4, 4), (128, 16, 8, 1), (8, 1, 3, 1),
                                                     (80, 7, 6, 2), (96, 48, 5, 5), (256, 128, 2, 1), (40, 256, 4, 2)])
@pytest.mark.parametrize("lens", [RAGGED, DECODE], ids=["ragged", "decode"])
def test_attention_lengths_and_layouts(lens, dim, page, heads, kv_heads, route, out_dtype):
    for token_major in (False, True):
        bt = Batch(lens, page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=dim + page, token_major=token_major,
                   pad_pages=3, q_pad=2 if token_major else 0)
        out = check(bt, route, out_dtype)
        for b, (n, c) in enumerate(lens):
            if c <= 0 and n:   # rows that see nothing
                assert not out[bt.starts[b]:bt.starts[b + 1]].any()


MODS = [dict(softcap=5.0), dict(softcap=30.0, window=40), dict(window=1), dict(window=33), dict(prefix=[0, 5, 1, 64, 290, 0, 200, 3]),
        dict(slopes=True), dict(slopes=True, softcap=20.0, prefix=[37] * 8, window=100), dict(scale=0.0), dict(scale=-0.3)]


@pytest.mark.parametrize("route", [AUTO, GEMV, SIMT, TC])
@pytest.mark.parametrize("dim,page,heads,kv_heads", [(64, 16, 8, 2), (128, 64, 4, 4), (80, 7, 6, 2), (128, 32, 24, 1)])
@pytest.mark.parametrize("mods", MODS, ids=lambda m: "-".join(m))
def test_attention_masks_and_scores(mods, dim, page, heads, kv_heads, route):
    mods = dict(mods)
    if mods.get("slopes"):
        mods["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads)
    bt = Batch(RAGGED, page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=3)
    dtype = torch.bfloat16 if route == TC else torch.float32
    check(bt, route, dtype, **mods)
    one = dict(mods)
    if one.get("prefix"):
        one["prefix"] = (one["prefix"] * 2)[:len(DECODE)]
    check(Batch(DECODE, page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=4), route, dtype, **one)


@pytest.mark.parametrize("route", [AUTO, GEMV, SIMT, TC])
@pytest.mark.parametrize("lens", [[(1, 400), (1, 90)], [(40, 400), (200, 390)]], ids=["decode", "chunk"])
def test_attention_pages_before_the_window_are_gone(lens, route):
    """A freed page (-1 in the table, its memory someone else's NaN) before the window is not touched."""
    bt = Batch(lens, page=16, heads=4, kv_heads=2, dim=64, seed=9)
    for b, (n, c) in enumerate(lens):
        for pg in range(max(0, c - n - 49) // 16):
            first = int(bt.table[b, pg])
            bt.k[first] = float("nan")
            bt.v[first] = float("nan")
            bt.table[b, pg] = -1
    check(bt, route, torch.bfloat16 if route == TC else torch.float32, window=50)


@pytest.mark.parametrize("route", [AUTO, GEMV, SIMT, TC])
def test_attention_large_scores(route):
    """Scores in the hundreds: the running maximum carries the sums, whatever order the keys come in."""
    bt = Batch([(1, 700), (70, 700)], page=64, heads=4, kv_heads=1, dim=64, seed=5, spread=40.0)
    # the score error scales with the scores: 64 * 2^-24 * sum|qk| * scale <= 2e-3 here
    out = torch.empty((bt.tokens, 4, 64), dtype=torch.bfloat16 if route == TC else torch.float32, device=DEV)
    kv.paged_attention(bt.q, *bt.args(), max_q=bt.max_q, max_kv=bt.max_kv, out=out, route=route)
    want = attention64(bt)
    assert torch.isfinite(out).all()
    assert float((out.cpu().double() - want).abs().max()) <= (2e-3 + (2.0 ** -7 if route == TC else 0.0)) * max(float(v.abs().max()) for v in bt.values)


@pytest.mark.parametrize("route", [AUTO, GEMV, TC])
@pytest.mark.parametrize("dim,page,heads,kv_heads", [(64, 16, 12, 4), (128, 128, 4, 4), (96, 32, 7, 1), (128, 8, 32, 1)])
@pytest.mark.parametrize("mods", [dict(), dict(window=200), dict(softcap=20.0, prefix=[300, 700, 0])], ids=["plain", "window", "capped"])
def test_attention_prompts(mods, dim, page, heads, kv_heads, route):
    """Many tiles of rows and blocks of keys: chunks that start inside a cache and end anywhere."""
    bt = Batch([(300, 300), (257, 900), (33, 1111)], page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=11)
    check(bt, route, torch.bfloat16, **mods)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("route", [AUTO, GEMV, TC])
def test_attention_split_caches(route, out_dtype):
    """Few rows over a long cache: the keys split across the grid and joined."""
    bt = Batch([(40, 5000)], page=64, heads=8, kv_heads=2, dim=128, seed=12)
    check(bt, route, out_dtype)
    check(bt, route, out_dtype, window=3000)
    bt = Batch([(1, 9000), (2, 700), (1, 3)], page=16, heads=8, kv_heads=1, dim=64, seed=13)
    check(bt, route, out_dtype)


def test_attention_bad_metadata_is_recorded_not_followed():
    bt = Batch([(1, 40), (1, 60)], page=16, heads=4, kv_heads=4, dim=64, seed=6)
    good = kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=60)
    bt.table[0, 1] = bt.n_pages          # a page that does not exist
    out = kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=60)
    torch.cuda.synchronize()
    assert _lib.device_error() == 9
    assert torch.equal(out[1], good[1]) and torch.isfinite(out).all()
    bt.table[0, 1] = -7
    kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=60)
    assert _lib.device_error() == 9
    bt.table[0, 1] = 0
    kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=59)
    assert _lib.device_error() == 10
    bt.kv_lens[1] = 1 << 20              # past the table
    kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=1 << 21)
    assert _lib.device_error() == 10
    assert _lib.device_error() == 0


def test_attention_on_another_stream_and_in_a_graph():
    from bybylang_b200 import gpubackend as gb
    gb.ensureGpuInit(gb.GpuBackend.gbCuda, 0)
    bt = Batch([(1, 900)] * 3, page=16, heads=8, kv_heads=2, dim=128, seed=8)
    want = kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=900)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=900, stream=s)
    s.synchronize()
    assert torch.equal(out, want)
    out = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv.paged_attention(bt.q, *bt.args(), max_q=1, max_kv=900, out=out)
    for _ in range(2):
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert _lib.device_error() == 0


# ---- rotary append -------------------------------------------------------------------------

def rope64(x, pos, turns, layout, magnitude=1.0):
    """x [tokens, heads, dim] fp64 on the CPU, turned."""
    r = 2 * turns.numel()
    a = 2 * math.pi * (pos.double()[:, None] * turns[None])
    cs, sn = magnitude * torch.cos(a)[:, None], magnitude * torch.sin(a)[:, None]
    x = x.double()
    i = torch.arange(r // 2)
    u, w = (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)
    y = x.clone()
    y[..., u] = x[..., u] * cs - x[..., w] * sn
    y[..., w] = x[..., u] * sn + x[..., w] * cs
    return y


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,pairs,page,heads,kv_heads,fused", [(128, 64, 16, 8, 2, True), (128, 32, 64, 4, 4, False), (64, 31, 7, 3, 1, True),
                                                                 (8, 1, 1, 1, 1, False), (256, 128, 48, 2, 1, True), (80, 0, 16, 5, 5, False),
                                                                 (96, 48, 16, 33, 3, True)])
def test_rope_append(dim, pairs, page, heads, kv_heads, fused, layout, dtype):
    lens = [(5, 37), (0, 11), (1, 1), (64, 64), (3, 0), (2, 1), (1, 100000 if dim == 128 and page == 64 else 300)]
    g = torch.Generator().manual_seed(dim + pairs)
    bt = Batch([(n, min(c, 400)) for n, c in lens], page=page, heads=heads, kv_heads=kv_heads, dim=dim, seed=1, pad_pages=1)
    long = lens[-1][1] > 400
    turns = kv.rope_frequencies(2 * pairs, 10000.0, device=DEV)
    total = heads + 2 * kv_heads + (1 if fused and dim != 8 else 0)
    wide = torch.randn(bt.tokens, total, dim, generator=g).to(dtype)
    d = wide.to(DEV)
    if fused:
        q, k, v = d[:, :heads], d[:, heads:heads + kv_heads], d[:, heads + kv_heads:heads + 2 * kv_heads]
    else:
        q, k, v = (x.contiguous() for x in (d[:, :heads], d[:, heads:heads + kv_heads], d[:, heads + kv_heads:heads + 2 * kv_heads]))
    before = bt.k.clone(), bt.v.clone()
    pos = torch.cat([torch.arange(c - n, c) for n, c in bt.lens])
    turn_by = None
    if long:   # far positions without a cache of that length
        turn_by = pos.clone()
        turn_by[-1] = 99999
    q_out = kv.rope_append(q, k, v, *bt.args(), turns, layout=layout, magnitude=1.25,
                           positions=None if turn_by is None else turn_by.to(torch.int32).to(DEV))
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    by = pos if turn_by is None else turn_by
    c = wide.double()
    wq = rope64(c[:, :heads], by, turns.cpu(), layout, 1.25)
    wk = rope64(c[:, heads:heads + kv_heads], by, turns.cpu(), layout, 1.25)
    wv = c[:, heads + kv_heads:heads + 2 * kv_heads]
    wq[pos < 0] = 0
    # one bf16 rounding (8 significant bits: 2^-8) of an fp32 value whose products and angle are good to 2^-20 of the pair
    def close(got, want, pair):
        assert (got.cpu().double() - want).abs().le(2.0 ** -8 * want.abs() + 2.0 ** -20 * pair + 1e-38).all()
    close(q_out, wq, float(c.abs().max()) * 2.5)
    want_k, want_v = before[0].cpu().double(), before[1].cpu().double()
    t = 0
    for b, (n, ctx) in enumerate(bt.lens):
        for i in range(n):
            p = ctx - n + i
            if p >= 0:
                want_k[bt.table[b, p // page], :, p % page] = wk[t]
                want_v[bt.table[b, p // page], :, p % page] = wv[t]
            t += 1
    for got, want in ((bt.k, want_k), (bt.v, want_v)):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        close(got[ok], want[ok], float(c.abs().max()) * 2.5)


def test_rope_append_rows_of_no_sequence_and_bad_pages():
    bt = Batch([(2, 20), (1, 5)], page=16, heads=2, kv_heads=2, dim=64, seed=2)
    x = torch.randn(6, 6, 64, device=DEV)
    q, k, v = x[:, :2], x[:, 2:4], x[:, 4:]
    starts = torch.tensor([1, 3, 4], dtype=torch.int32, device=DEV)
    out = torch.full((6, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    turns = kv.rope_frequencies(64, device=DEV)
    kv.rope_append(q, k, v, bt.k, bt.v, bt.table, starts, bt.kv_lens, turns, q_out=out)
    assert _lib.device_error() == 0
    assert (out[[0, 4, 5]] == 7.0).all() and not (out[[1, 2, 3]] == 7.0).all()
    before = bt.k.clone()
    bt.table[1, 0] = bt.n_pages + 5
    bt.table[0, 1] = -1
    kv.rope_append(q, k, v, bt.k, bt.v, bt.table, starts, bt.kv_lens, turns, q_out=out)
    assert _lib.device_error() == 9
    assert torch.equal(bt.k.view(torch.int16), before.view(torch.int16))


def test_rope_frequencies():
    base = kv.rope_frequencies(64, 10000.0, device=DEV).cpu()
    want = torch.tensor([10000.0 ** (-i / 32) / (2 * math.pi) for i in range(32)], dtype=torch.float64)
    assert torch.allclose(base, want, rtol=1e-14, atol=0)
    assert torch.allclose(kv.rope_frequencies(64, scaling="linear", factor=4.0, device=DEV).cpu(), want / 4, rtol=1e-14, atol=0)
    b = kv.rope_frequencies(64, scaling="base", factor=4.0, device=DEV).cpu()
    assert abs(b[0] / want[0] - 1) < 1e-14 and abs(b[-1] / want[-1] * 4 - 1) < 1e-12
    p = kv.rope_frequencies(64, scaling="by-parts", factor=4.0, original_context=4096, device=DEV).cpu()
    turns = want * 4096
    assert torch.equal(p[turns > 32], want[turns > 32]) and torch.allclose(p[turns < 1], want[turns < 1] / 4, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((p < want) & (p > want / 4))[mid].all()


# ---- page copies ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,pages,heads,page,dim,n", [(1, 3, 1, 1, 8, 1), (4, 40, 2, 16, 64, 13), (2, 2500, 1, 1, 8, 1200), (3, 9, 8, 128, 128, 4)])
def test_copy_pages(layers, pages, heads, page, dim, n, dtype):
    g = torch.Generator().manual_seed(n)
    k = torch.randn(layers, pages, heads, page, dim, generator=g).to(dtype).to(DEV)
    v = torch.randn(layers, pages, heads, page, dim, generator=g).to(dtype).to(DEV)
    order = torch.randperm(pages, generator=g)
    dst = order[:n]
    src = order[n:][torch.randint(0, pages - n, (n,), generator=g)]     # one page may go to several
    pairs = torch.stack([src, dst], 1).to(torch.int32)
    want_k, want_v = k.clone(), v.clone()
    want_k[:, dst.to(DEV)] = k[:, src.to(DEV)]
    want_v[:, dst.to(DEV)] = v[:, src.to(DEV)]
    kv.copy_pages(k, v, pairs)
    torch.cuda.synchronize()
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    kv.copy_pages(k, None, [(int(src[0]), int(dst[0]))])
    kv.copy_pages(k[0], v[0], [])
    # token-major pages and padded page strides are dense blocks too
    room = torch.zeros(layers, pages, 2 * page, heads, dim, dtype=dtype, device=DEV)
    kt = room[:, :, :page].transpose(2, 3)
    kt.copy_(want_k)
    kv.copy_pages(kt, None, pairs)
    torch.cuda.synchronize()
    assert torch.equal(kt, want_k)
    assert not room[:, :, page:].any()


# ---- beam selection ------------------------------------------------------------------------

def beams64(logits, scores, keep):
    groups, beams = scores.shape
    x = logits.cpu().double().view(groups, beams, -1)
    s = scores.cpu().double()[..., None] + torch.log_softmax(x, -1)
    s = torch.where(torch.isnan(s), -math.inf, s)
    return s


def check_beams(logits, scores, keep):
    got, b, t = kv.beam_select(logits, scores, keep)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    groups, beams = scores.shape
    V = logits.shape[1]
    s = beams64(logits, scores, keep)
    flat = s.view(groups, -1)
    place = b.cpu().long() * V + t.cpu().long()
    assert (b.cpu() >= 0).all() and (b.cpu() < beams).all() and (t.cpu() >= 0).all() and (t.cpu() < V).all()
    at = torch.gather(flat, 1, place)
    top = torch.sort(flat, 1, descending=True).values[:, :keep]
    got = got.cpu().double()
    # log-softmax in fp32: a sum of exponentials good to 2^-20 and one rounding of each of three terms
    tol = 1e-5 * (1 + torch.where(torch.isfinite(top), top.abs(), 0.0))
    fin = torch.isfinite(top)
    assert torch.equal(got == -math.inf, top == -math.inf)
    assert ((got - top).abs()[fin] <= tol[fin]).all() and ((got - at).abs()[fin] <= tol[fin]).all()
    assert ((at == -math.inf) == (top == -math.inf)).all()
    for g in range(groups):
        assert len(set(place[g].tolist())) == keep
    # exact order inside a beam: logits fall, equal logits by the lower token, none skipped
    x = logits.cpu().float().view(groups, beams, V)
    for g in range(groups):
        for beam in range(beams):
            mine = [int(q) for q, w in zip(t[g].tolist(), b[g].tolist()) if w == beam]
            if not mine:
                continue
            dead = not bool(torch.isfinite(s[g, beam]).any())
            want = list(range(len(mine))) if dead else \
                torch.sort(x[g, beam], descending=True, stable=True).indices[:len(mine)].tolist()
            assert mine == want, (g, beam)
    return got, b, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,beams,vocab,keep", [(1, 1, 1, 1), (1, 4, 128256, 8), (3, 2, 1000, 4), (2, 5, 33, 64), (1, 64, 7, 64), (2, 8, 8193, 16),
                                                     (40, 8, 32000, 16), (1, 1, 20000, 64), (5, 3, 257, 6), (1, 3, 65, 33)])
def test_beam_select(groups, beams, vocab, keep, dtype):
    g = torch.Generator().manual_seed(vocab)
    x = 3 * torch.randn(groups * beams, vocab + 5, generator=g)
    s = -5 * torch.rand(groups, beams, generator=g)
    x = x.to(dtype).to(DEV)
    check_beams(x[:, :vocab], s.to(DEV), keep)            # rows apart: scalar loads
    check_beams(x[:, :vocab].contiguous(), s.to(DEV), keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 5000, 128256])
@pytest.mark.parametrize("what", ["constant", "masked", "one left", "rising", "falling", "dead beams", "all dead", "nan", "inf", "first", "blocks"])
def test_beam_select_hard_rows(what, vocab, dtype):
    g = torch.Generator().manual_seed(7)
    beams, keep = 4, 8
    x = torch.randn(2 * beams, vocab, generator=g)
    s = -torch.rand(2, beams, generator=g)
    if what == "constant":
        x[:] = 0.25
    elif what == "masked":
        x[:, : vocab - 9] = -math.inf
    elif what == "one left":
        x[:, 1:] = -math.inf
    elif what == "rising":
        x[:] = torch.arange(vocab) / vocab * 40
    elif what == "falling":
        x[:] = -torch.arange(vocab) / vocab * 40
    elif what == "dead beams":
        x[0], x[5] = -math.inf, -math.inf
    elif what == "all dead":
        x[:] = -math.inf
    elif what == "nan":
        x[1, vocab // 2] = math.nan
        x[4] = math.nan
        s[0, 3] = math.nan
    elif what == "inf":
        x[2, 3] = math.inf
        x[4, :20] = math.inf
    elif what == "first":
        s[:, 1:] = -math.inf
        x[0, 1:], x[4, 5:] = -math.inf, -math.inf
    elif what == "blocks":     # whole warps' tokens masked, the rest all above them
        x = torch.where((torch.arange(vocab) // 128) % 8 == 3, -math.inf, x + 10)
    check_beams(x.to(dtype).to(DEV), s.to(DEV), keep)


# ---- together, and at the edges of the address space ----------------------------------------

def test_beam_search_example():
    """The example's found sequences, scored again without a cache in fp32: q, k, v, the attention
    output and the activations of the 4-bit products are rounded to 8..15 bits on the way, which at
    these widths moves a log-probability by some 1e-2; a wrong page, position or parent by whole
    units."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "beam_search.py")
    spec = importlib.util.spec_from_file_location("beam_search_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    model, prompts, found = mod.main(["--beams", "3", "--tokens", "20", "--prompts", "2"])
    assert _lib.device_error() == 0
    assert model.pool.free_pages == model.pool.n_pages          # every page came back
    for prompt, beams in zip(prompts, found):
        assert [s for s, _ in beams] == sorted((s for s, _ in beams), reverse=True)
        assert len({tuple(t) for _, t in beams}) == len(beams)
        for score, text in beams:
            assert abs(score - model.check(prompt, text)) < 0.2


def test_offsets_past_32_bits():
    """Pages that start 2^31 elements and more into the cache."""
    page, heads, dim = 64, 8, 128
    per = page * heads * dim
    n = (1 << 31) // per + 40
    k = torch.empty(n, heads, page, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(n, heads, page, dim, dtype=torch.bfloat16, device=DEV)
    lens = [(1, 200), (70, 100)]
    bt = Batch(lens, page=page, heads=16, kv_heads=heads, dim=dim, seed=3)
    for i in range(bt.n_pages):     # the same cache, far out
        k[n - 1 - i], v[n - 1 - i] = bt.k[i], bt.v[i]
    bt.table = torch.where(bt.table >= 0, n - 1 - bt.table, bt.table)
    bt.k, bt.v = k, v
    for route in (GEMV, TC, SIMT):
        check(bt, route, torch.bfloat16)
    x = torch.randn(71, 32, dim, device=DEV)
    q, kk, vv = x.split([16, 8, 8], 1)
    kv.rope_append(q, kk, vv, *bt.args(), kv.rope_frequencies(0, device=DEV))     # no pair turns: a plain append
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    assert torch.equal(k[bt.table[0, 3].long(), :, 199 % page], kk[0].to(torch.bfloat16))
    assert torch.equal(v[bt.table[1, 1].long(), :, 99 % page], vv[70].to(torch.bfloat16))
    pairs = [(n - 1, 0), (1, n - 20)]
    k[1].fill_(3.0)
    kv.copy_pages(k, v, pairs)
    torch.cuda.synchronize()
    assert torch.equal(k[0].view(torch.int16), k[n - 1].view(torch.int16)) and (k[n - 20] == 3.0).all()


@pytest.mark.parametrize("route", [GEMV, TC, SIMT])
def test_attention_groups_and_rows_that_do_not_divide(route):
    for heads, kv_heads, dim in ((100, 1, 64), (9, 3, 128), (127, 1, 32)):
        bt = Batch([(3, 40), (20, 333), (1, 5)], page=16, heads=heads, kv_heads=kv_heads, dim=dim, seed=heads)
        check(bt, route, torch.bfloat16)
    bt = Batch([(3, 40), (2, 200)], page=16, heads=200, kv_heads=1, dim=64, seed=1)
    if route == TC:
        with pytest.raises(_lib.BybyCudaError, match="128 heads a group"):
            kv.paged_attention(bt.q, *bt.args(), max_q=3, max_kv=200, route=TC)
    else:
        check(bt, route, torch.bfloat16)


@pytest.mark.parametrize("route", [GEMV, TC, SIMT])
def test_attention_nan_reaches_only_rows_that_see_it(route):
    """A NaN key is a NaN row for every row that sees it, in whatever half or step of a block, and
    nothing for the others; so is one behind a tanh cap."""
    for softcap in (0.0, 20.0):
        for at in (3, 37, 70, 127, 128, 199):
            bt = Batch([(200, 200), (60, 200)], page=16, heads=2, kv_heads=1, dim=64, seed=at)
            bt.k[bt.table[0, at // 16], 0, at % 16, 5] = float("nan")
            out = kv.paged_attention(bt.q, *bt.args(), max_q=200, max_kv=200, softcap=softcap, out_dtype=torch.bfloat16, route=route)
            torch.cuda.synchronize()
            bad = torch.isnan(out).any(-1).any(-1)
            want = torch.zeros(260, dtype=torch.bool, device=DEV)
            want[at:200] = True
            assert torch.equal(bad, want)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("route", [GEMV, TC, SIMT])
def test_attention_is_the_same_every_time(route):
    for lens in ([(1, 9000)], [(1, 700)] * 3, [(300, 2000), (64, 64)]):
        bt = Batch(lens, page=64, heads=8, kv_heads=2, dim=128, seed=2)
        outs = [kv.paged_attention(bt.q, *bt.args(), max_q=bt.max_q, max_kv=bt.max_kv, route=route) for _ in range(3)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_python_refusals():
    bt = Batch([(1, 20)], page=16, heads=4, kv_heads=2, dim=64, seed=1)
    call = dict(max_q=1, max_kv=20)
    with pytest.raises(_lib.BybyCudaError, match="torch.bfloat16"):
        kv.paged_attention(bt.q.float(), *bt.args(), **call)
    with pytest.raises(_lib.BybyCudaError, match="torch.float32"):
        kv.paged_attention(bt.q, *bt.args(), slopes=torch.zeros(3, device=DEV), **call)
    with pytest.raises(_lib.BybyCudaError, match="torch.int32"):
        kv.paged_attention(bt.q, *bt.args(), prefix_lens=torch.zeros(1, device=DEV), **call)
    with pytest.raises(_lib.BybyCudaError, match="not \\[1, 4, 64\\]"):
        kv.paged_attention(bt.q, *bt.args(), out=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV), **call)
    with pytest.raises(_lib.BybyCudaError, match="float32 or bfloat16"):
        kv.paged_attention(bt.q, *bt.args(), out_dtype=torch.float16, **call)
    with pytest.raises(_lib.BybyCudaError, match="16-byte aligned"):
        odd = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(1, 4, 64)
        kv.paged_attention(odd, *bt.args(), **call)
    with pytest.raises(_lib.BybyCudaError, match="tensor-core route"):
        kv.paged_attention(bt.q, *bt.args(), out_dtype=torch.float32, route=TC, **call)
    q3 = torch.zeros(1, 3, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(_lib.BybyCudaError, match="3 query heads over 2"):
        kv.paged_attention(q3, *bt.args(), **call)
    turns = kv.rope_frequencies(64, device=DEV)
    kk = torch.zeros(1, 2, 64, device=DEV)
    with pytest.raises(_lib.BybyCudaError, match="unknown layout"):
        kv.rope_append(kk.expand(1, 2, 64), kk, kk, *bt.args(), turns, layout="other")
    with pytest.raises(_lib.BybyCudaError, match="torch.float64"):
        kv.rope_append(kk, kk, kk, *bt.args(), turns.float())
    with pytest.raises(_lib.BybyCudaError, match="k must be"):
        kv.rope_append(kk, kk.bfloat16(), kk, *bt.args(), turns)
    with pytest.raises(_lib.BybyCudaError, match="dense block"):
        kv.copy_pages(bt.k[:, :, :8], bt.v[:, :, :8], [(0, 1)])
    with pytest.raises(_lib.BybyCudaError, match="scores must be contiguous"):
        kv.beam_select(torch.zeros(2, 9, device=DEV), torch.zeros(1, 2, dtype=torch.float64, device=DEV), 2)
    with pytest.raises(_lib.BybyCudaError, match="unknown scaling"):
        kv.rope_frequencies(64, scaling="x", device=DEV)
    assert _lib.device_error() == 0
