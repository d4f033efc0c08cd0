"""The paged-cache operators without a GPU: what they refuse before any device work, and the page
pool's bookkeeping."""
import ctypes as C
import random

import pytest

from bybylang_b200 import _lib
from bybylang_b200.kvcache import PagePool, copy_pages, paged_attention

P = 1 << 20   # an aligned address that is never followed


def cache(**kw):
    d = dict(k=P, v=P, page_stride=4 * 16 * 64, head_stride=16 * 64, token_stride=64, page_table=P, table_stride=8, q_start=P,
             kv_lens=P, n_pages=10, page_size=16, kv_heads=4, head_dim=64, max_pages=8, n_seqs=2, n_tokens=3, reserved=0)
    d.update(kw)
    return _lib.PagedKv(*[d[n] for n, _ in _lib.PagedKv._fields_])


def rope(**kw):
    d = dict(q=P, k=P, v=P, q_out=P, q_token_stride=512, q_head_stride=64, k_token_stride=256, k_head_stride=64, v_token_stride=256,
             v_head_stride=64, out_token_stride=512, out_head_stride=64, turns=P, positions=None, in_dtype=1, q_heads=8, pairs=32,
             interleaved=0, magnitude=1.0, reserved=0)
    d.update(kw)
    return _lib.Rope(*[d[n] for n, _ in _lib.Rope._fields_])


def attention(**kw):
    d = dict(q=P, out=P, q_token_stride=512, q_head_stride=64, out_token_stride=512, out_head_stride=64, slopes=None, prefix_lens=None,
             out_dtype=1, q_heads=8, max_q=2, max_kv=100, window=0, route=0, scale=0.125, softcap=0.0)
    d.update(kw)
    return _lib.Attention(*[d[n] for n, _ in _lib.Attention._fields_])


def refused(rc, code, text):
    assert rc == code, (rc, _lib.last_error())
    got, message = _lib.last_error()
    assert got == code and text in message, message


CACHE_REFUSALS = [
    (dict(head_dim=60), _lib.ERR_SHAPE, "head dimension"), (dict(head_dim=264), _lib.ERR_SHAPE, "head dimension"),
    (dict(kv_heads=0), _lib.ERR_SHAPE, "heads=0"), (dict(page_size=0), _lib.ERR_SHAPE, "page=0"), (dict(n_tokens=-1), _lib.ERR_SHAPE, "tokens=-1"),
    (dict(max_pages=1 << 28), _lib.ERR_SHAPE, "2^31"), (dict(k=0), _lib.ERR_ARGS, "missing"), (dict(page_table=0), _lib.ERR_ARGS, "missing"),
    (dict(v=P + 8), _lib.ERR_ARGS, "misaligned"), (dict(token_stride=60), _lib.ERR_ARGS, "multiples of 8"),
    (dict(table_stride=7), _lib.ERR_ARGS, "max_pages"), (dict(token_stride=32), _lib.ERR_ARGS, "overlap"),
    (dict(head_stride=512), _lib.ERR_ARGS, "overlap"), (dict(page_stride=1024), _lib.ERR_ARGS, "overlap"), (dict(reserved=1), _lib.ERR_ARGS, "reserved"),
]


@pytest.mark.parametrize("kw,code,text", CACHE_REFUSALS)
def test_cache_refusals(kw, code, text):
    lib = _lib.load()
    refused(lib.bybycu_rope_append(cache(**kw), rope(), None), code, text)
    refused(lib.bybycu_paged_attention(cache(**kw), attention(), None), code, text)


def test_null_structs():
    lib = _lib.load()
    refused(lib.bybycu_rope_append(None, rope(), None), _lib.ERR_ARGS, "cache is NULL")
    refused(lib.bybycu_rope_append(cache(), None, None), _lib.ERR_ARGS, "arguments are NULL")
    refused(lib.bybycu_paged_attention(cache(), None, None), _lib.ERR_ARGS, "arguments are NULL")


@pytest.mark.parametrize("kw,code,text", [
    (dict(in_dtype=2), _lib.ERR_ARGS, "F32 or BF16"), (dict(pairs=33), _lib.ERR_SHAPE, "33 pairs"), (dict(pairs=-1), _lib.ERR_SHAPE, "pairs"),
    (dict(q_heads=0), _lib.ERR_SHAPE, "query heads"), (dict(q=0), _lib.ERR_ARGS, "missing"), (dict(turns=None), _lib.ERR_ARGS, "missing"),
    (dict(turns=P + 4), _lib.ERR_ARGS, "misaligned"), (dict(q_head_stride=32), _lib.ERR_ARGS, "strides"),
    (dict(v_token_stride=-1), _lib.ERR_ARGS, "strides"), (dict(reserved=3), _lib.ERR_ARGS, "reserved")])
def test_rope_refusals(kw, code, text):
    refused(_lib.load().bybycu_rope_append(cache(), rope(**kw), None), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(out_dtype=5), _lib.ERR_ARGS, "F32 or BF16"), (dict(q_heads=6), _lib.ERR_SHAPE, "6 query heads over 4"),
    (dict(max_q=-1), _lib.ERR_SHAPE, "max_q=-1"), (dict(window=-2), _lib.ERR_SHAPE, "window=-2"), (dict(scale=float("nan")), _lib.ERR_ARGS, "scale"),
    (dict(softcap=-1.0), _lib.ERR_ARGS, "softcap"), (dict(route=99), _lib.ERR_ARGS, "unknown route"), (dict(q=0), _lib.ERR_ARGS, "missing"),
    (dict(out=P + 2), _lib.ERR_ARGS, "16-byte"), (dict(q_token_stride=516), _lib.ERR_ARGS, "16-byte"), (dict(q_head_stride=56), _lib.ERR_ARGS, "overlap")])
def test_attention_refusals(kw, code, text):
    refused(_lib.load().bybycu_paged_attention(cache(), attention(**kw), None), code, text)


def test_empty_batches_need_no_device():
    lib = _lib.load()
    for kw in (dict(n_tokens=0), dict(n_seqs=0)):
        assert lib.bybycu_rope_append(cache(**kw), rope(), None) == 0
        assert lib.bybycu_paged_attention(cache(**kw), attention(), None) == 0


def pairs(*p):
    return (C.c_int32 * (2 * len(p)))(*[x for q in p for x in q])


@pytest.mark.parametrize("kw,code,text", [
    (dict(p=[(0, 8)]), _lib.ERR_RANGE, "outside the 8 pages"), (dict(p=[(-1, 2)]), _lib.ERR_RANGE, "outside"),
    (dict(p=[(3, 3)]), _lib.ERR_ARGS, "destination"), (dict(p=[(0, 1), (2, 1)]), _lib.ERR_ARGS, "page 1"),
    (dict(p=[(0, 1), (1, 2)]), _lib.ERR_ARGS, "page 1"), (dict(p=[(1, 2), (0, 1)]), _lib.ERR_ARGS, "page 1"),
    (dict(page_bytes=24), _lib.ERR_SHAPE, "page bytes=24"), (dict(k=0), _lib.ERR_ARGS, "missing"), (dict(k=P + 4), _lib.ERR_ARGS, "16 bytes"),
    (dict(page_stride=32), _lib.ERR_ARGS, "page_bytes apart"), (dict(layers=0), _lib.ERR_SHAPE, "layers=0")])
def test_copy_refusals(kw, code, text):
    d = dict(k=P, v=P, layers=2, layer_stride=1 << 16, page_stride=64, page_bytes=64, pages=8, p=[(0, 1)])
    d.update(kw)
    rc = _lib.load().bybycu_copy_pages(d["k"], d["v"], d["layers"], d["layer_stride"], d["page_stride"], d["page_bytes"], d["pages"],
                                       pairs(*d["p"]), len(d["p"]), None)
    refused(rc, code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=3), _lib.ERR_ARGS, "F32 or BF16"), (dict(keep=65), _lib.ERR_SHAPE, "keep=65"), (dict(keep=0), _lib.ERR_SHAPE, "keep=0"),
    (dict(beams=65), _lib.ERR_SHAPE, "beams=65"), (dict(beams=1, vocab=3, keep=4), _lib.ERR_SHAPE, "keep=4"), (dict(vocab=0), _lib.ERR_SHAPE, "vocab=0"),
    (dict(vocab=1 << 21), _lib.ERR_SHAPE, "vocab"), (dict(groups=20000, beams=4), _lib.ERR_SHAPE, "65535"), (dict(stride=99), _lib.ERR_ARGS, "overlap"),
    (dict(logits=P + 2), _lib.ERR_ARGS, "misaligned"), (dict(scores=0), _lib.ERR_ARGS, "missing")])
def test_beam_refusals(kw, code, text):
    d = dict(logits=P, dtype=0, stride=None, scores=P, groups=2, beams=4, vocab=100, keep=8)
    d.update(kw)
    rc = _lib.load().bybycu_beam_select(d["logits"], d["dtype"], d["stride"] or d["vocab"] if d["stride"] is None else d["stride"], d["scores"],
                                        d["groups"], d["beams"], d["vocab"], d["keep"], P, P, P, None)
    refused(rc, code, text)


def test_python_refusals_on_the_host():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, 4, dtype=torch.int32)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    starts, lens = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    with pytest.raises(_lib.BybyCudaError, match="on the device"):
        paged_attention(q, k, k, i, starts, lens, max_q=1, max_kv=1)
    with pytest.raises(_lib.BybyCudaError, match="bfloat16"):
        paged_attention(q, k.float(), k, i, starts, lens, max_q=1, max_kv=1)
    with pytest.raises(_lib.BybyCudaError, match="int32"):
        paged_attention(q, k, k, i.long(), starts, lens, max_q=1, max_kv=1)
    with pytest.raises(_lib.BybyCudaError, match="2 starts"):
        paged_attention(q, k, k, i, starts[:1], lens, max_q=1, max_kv=1)
    with pytest.raises(_lib.BybyCudaError, match="on the device"):
        copy_pages(k, k, [(0, 1)])


# ---- PagePool -----------------------------------------------------------------------------

class Shadow:
    """The pool's contents as a plain simulation: what every slot of every page holds."""

    def __init__(self, n_pages, page):
        self.pool, self.page = PagePool(n_pages, page), page
        self.mem = [[None] * page for _ in range(n_pages)]
        self.texts = {}

    def copy(self, pairs):
        src = [list(self.mem[a]) for a, _ in pairs]
        assert len({b for _, b in pairs}) == len(pairs) and not {a for a, _ in pairs} & {b for _, b in pairs}
        for s, (_, b) in zip(src, pairs):
            self.mem[b] = s

    def write(self, seq, items):
        n = self.pool.length(seq)
        self.copy(self.pool.extend(seq, len(items)))
        pages = self.pool.pages(seq)
        for i, x in enumerate(items):
            self.mem[pages[(n + i) // self.page]][(n + i) % self.page] = x
        self.texts[seq] = self.texts[seq] + items

    def check(self):
        pool, held = self.pool, {}
        for seq, text in self.texts.items():
            pages = pool.pages(seq)
            assert pool.length(seq) == len(text) and len(pages) == -(-len(text) // self.page)
            assert [self.mem[pages[i // self.page]][i % self.page] for i in range(len(text))] == text
            for p in pages:
                held[p] = held.get(p, 0) + 1
        assert all(pool._refs[p] == held.get(p, 0) for p in range(pool.n_pages))
        assert sorted(pool._free) == [p for p in range(pool.n_pages) if p not in held]


@pytest.mark.parametrize("page", [1, 4, 16])
def test_page_pool_against_a_simulation(page):
    rng = random.Random(page)
    s = Shadow(60, page)
    for step in range(600):
        act = rng.choice(["new", "write", "write", "write", "fork", "free", "compact", "reorder"])
        seqs = sorted(s.texts)
        try:
            if act == "new" or not seqs:
                s.texts[s.pool.new()] = []
            elif act == "write":
                s.write(rng.choice(seqs), [step * 1000 + i for i in range(rng.randrange(0, 3 * page))])
            elif act == "fork" and len(seqs) < 12:
                a = rng.choice(seqs)
                s.texts[s.pool.fork(a)] = list(s.texts[a])
            elif act == "free":
                a = rng.choice(seqs)
                s.pool.free(a)
                del s.texts[a]
            elif act == "compact":
                s.copy(s.pool.compact())
                used = s.pool.n_pages - s.pool.free_pages
                assert all(p < used for q in s.texts for p in s.pool.pages(q))
            elif act == "reorder":
                some = rng.sample(seqs, min(len(seqs), 3))
                parents = [rng.randrange(len(some)) for _ in some]
                new = s.pool.reorder(some, parents)
                old = [s.texts.pop(q) for q in some]
                for q, p in zip(new, parents):
                    s.texts[q] = list(old[p])
        except _lib.BybyCudaError as e:   # full: nothing may have changed
            assert e.code == _lib.ERR_RANGE
        s.check()


def test_page_pool_refusals_and_tables():
    torch = pytest.importorskip("torch")
    with pytest.raises(_lib.BybyCudaError):
        PagePool(0, 16)
    pool = PagePool(4, 16)
    a = pool.new()
    pool.extend(a, 40)
    with pytest.raises(_lib.BybyCudaError, match="2 pages wanted, 1 free"):
        pool.extend(a, 40)
    with pytest.raises(_lib.BybyCudaError, match="unknown sequence"):
        pool.free(99)
    b = pool.fork(a)
    assert pool.extend(b, 1) == [(2, 3)] and pool.free_pages == 0
    table, lens = pool.table([a, b], device="cpu", width=5)
    assert table.tolist() == [[0, 1, 2, -1, -1], [0, 1, 3, -1, -1]] and lens.tolist() == [40, 41]
    assert table.dtype == lens.dtype == torch.int32
    with pytest.raises(_lib.BybyCudaError, match="more than 2"):
        pool.table([a], device="cpu", width=2)
    pool.free(a)
    assert pool.free_pages == 1
    with pytest.raises(_lib.BybyCudaError):
        pool.length(a)
