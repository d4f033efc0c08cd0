"""The cases that the serving operators of bybylang_b200.kvcache are timed on.

Four operators make up one step of a decoder beside the quantised projections: rope_append (rotary positions, and the new
keys and values into their pages), paged_attention (a chunk of new tokens, or one, over a paged cache), beam_select (the
best continuations of the LM head's logits) and copy_pages (forked and compacted pages).  With `own` false `run` computes
them with elementary torch operations in 32 bits; with `own` true it calls the framework.
"""
import math
import random

import torch

own = False

DEV = "cuda"
HEAD_VOCAB = 128256   # the framework's LM-head benchmark: 128256 rows


# ---- the cases ---------------------------------------------------------------------------

def _rope(**k):
    return dict(op="rope", heads=32, kv_heads=8, dim=128, page=16, layout="half", rotary=128, base=500000.0, stretch=1.0,
                in_dtype="bf16", **k) if not k else {**_rope(), **k}


def _attn(**k):
    base = dict(op="attention", heads=32, kv_heads=8, dim=128, page=64, out_dtype="bf16", softcap=0.0, alibi=False, window=0,
                prefix=0)
    return {**base, **k}


def listed():
    return [
        # one token of one sequence: what a step costs when there is nothing to do but to get through it (32 heads of 128, the 7B layer's)
        _rope(name="append-1", heads=32, kv_heads=32, seqs=1, chunk=1, context=1000, ragged=1, base=10000.0),
        # a batch of 256 sequences deep in long contexts, frequencies stretched fourfold
        _rope(name="append-decode-256", seqs=256, chunk=1, context=32000, ragged=2, stretch=4.0),
        # ragged prompts, fp32 projections, adjacent pairs, half of each head turned
        _rope(name="append-prompts", seqs=8, chunk=1536, context=1600, ragged=3, page=64, layout="interleaved", rotary=64, in_dtype="f32"),
        # one token over a short context, every head with keys of its own
        _attn(name="decode-1", kv_heads=32, seqs=1, chunk=1, context=1023, ragged=0, page=16),
        # a serving batch: 64 sequences of all lengths up to 8K
        _attn(name="decode-64", seqs=64, chunk=1, context=8192, ragged=4),
        # one token over a very long context, fp32 out for the asymmetric-Q4 projection
        _attn(name="decode-long", seqs=1, chunk=1, context=131071, ragged=0, out_dtype="f32"),
        # chunks of ragged prompts over what is cached: capped scores, a window, heads of 64
        _attn(name="chunk-capped-window", seqs=6, chunk=700, context=9000, ragged=5, dim=64, page=32, softcap=30.0, window=4096),
        # the largest: two prompts of 4096 at once, 32 heads of 128
        _attn(name="prompt-4096", kv_heads=32, seqs=2, chunk=4096, context=4096, ragged=0, page=128),
        # four beams' last pages, all layers of a small cache: the copy of a fork
        dict(name="fork-4", op="copy", layers=8, pages=64, page=16, kv_heads=8, dim=128, pairs=4),
        # the cache's upper half moved down into holes
        dict(name="compact-256", op="copy", layers=8, pages=640, page=64, kv_heads=8, dim=128, pairs=256),
        # the first step of a search: one live beam of four
        dict(name="beams-1x4", op="beam", groups=1, beams=4, vocab=HEAD_VOCAB, keep=8, dtype="f32", first=True),
        # a batch of searches, bf16 logits (ties), part of the vocabulary masked
        dict(name="beams-32x8", op="beam", groups=32, beams=8, vocab=HEAD_VOCAB, keep=16, dtype="bf16", first=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "attention", "copy", "beam"])
    if op == "rope":
        seqs = _spread(rng, 1, 256)
        chunk = 1 if rng.random() < 0.5 else _spread(rng, 1, max(1, 12288 // seqs))
        dim = rng.choice([64, 128])
        c = _rope(seqs=seqs, chunk=chunk, context=max(chunk, _spread(rng, 100, 32000)), ragged=rng.randrange(1, 1 << 20), dim=dim,
                  kv_heads=rng.choice([1, 4, 8, 16]), heads=rng.choice([16, 32]), page=rng.choice([16, 32, 64, 128]),
                  layout=rng.choice(["half", "interleaved"]), rotary=rng.choice([dim, dim // 2]), in_dtype=rng.choice(["bf16", "f32"]),
                  base=rng.choice([10000.0, 500000.0]), stretch=rng.choice([1.0, 4.0]))
        while _slots(c) * c["kv_heads"] * dim > 300_000_000:
            c["context"] = max(c["chunk"], c["context"] // 2)
            if c["context"] == c["chunk"]:
                break
        return c
    if op == "attention":
        decode = rng.random() < 0.5
        seqs = _spread(rng, 1, 64 if decode else 8)
        chunk = rng.choice([1, 1, 1, 2, 4]) if decode else _spread(rng, 16, 4096)
        context = max(chunk, _spread(rng, 300, 131071 if seqs == 1 else 16384))
        kv_heads = rng.choice([1, 4, 8, 16, 32])
        c = _attn(seqs=seqs, chunk=chunk, context=context, ragged=rng.randrange(1, 1 << 20), dim=rng.choice([64, 128]), kv_heads=kv_heads,
                  heads=32, page=rng.choice([16, 32, 64, 128]), out_dtype=rng.choice(["bf16", "f32"]))
        mod = rng.choice(["none", "none", "softcap", "alibi", "window", "prefix"])
        c["softcap"] = 30.0 if mod == "softcap" else 0.0
        c["alibi"] = mod == "alibi"
        c["window"] = _spread(rng, 128, 4096) if mod == "window" else 0
        c["prefix"] = _spread(rng, 16, max(17, context)) if mod == "prefix" else 0
        top = max(_cost(x) for x in listed())
        while _cost(c) > top or c["seqs"] * 32 * c["chunk"] * c["context"] > 1_100_000_000 or \
                c["seqs"] * c["kv_heads"] * c["context"] * c["dim"] > 600_000_000:
            c["seqs"], c["context"], c["chunk"] = max(1, c["seqs"] * 2 // 3), max(c["context"] * 2 // 3, 16), max(1, c["chunk"] * 2 // 3)
            c["context"] = max(c["context"], c["chunk"])
        return c
    if op == "copy":
        pages = _spread(rng, 32, 640)
        return dict(op="copy", layers=rng.choice([1, 2, 4, 8]), pages=pages, page=rng.choice([16, 32, 64]), kv_heads=rng.choice([1, 4, 8]),
                    dim=rng.choice([64, 128]), pairs=_spread(rng, 1, pages * 2 // 5))
    groups, beams = _spread(rng, 1, 32), rng.randrange(1, 9)
    return dict(op="beam", groups=groups, beams=beams, vocab=_spread(rng, 1000, HEAD_VOCAB), keep=rng.choice([beams, 2 * beams]),
                dtype=rng.choice(["f32", "bf16"]), first=rng.random() < 0.3)


def _lengths(c):
    """[(new tokens, tokens in the cache with them)] of a case's sequences: the whole sizes, or ragged ones up to them."""
    if not c["ragged"]:
        return [(c["chunk"], c["context"])] * c["seqs"]
    r = random.Random(c["ragged"])
    got = []
    for _ in range(c["seqs"]):
        n = 1 if c["chunk"] == 1 else max(1, _spread(r, max(1, c["chunk"] // 8), c["chunk"]))
        got.append((n, max(n, _spread(r, max(1, c["context"] // 16), c["context"]))))
    got[0] = (c["chunk"], c["context"])
    return got


def _slots(c):
    return sum(-(-kv // c["page"]) for _, kv in _lengths(c)) * c["page"]


def _visible(c, n, kv):
    """(keys that some new token sees, pairs of a new token and a key that it sees) of one sequence."""
    low, pairs = kv, 0
    for i in range(n):
        p = kv - n + i
        lo = max(0, p - c["window"] + 1) if c["window"] else 0
        low = min(low, lo)
        pairs += max(p + 1, min(kv, c["prefix"])) - lo
    return kv - low, pairs


def work(c):
    if c["op"] == "rope":
        tokens = sum(n for n, _ in _lengths(c))
        size = 2 if c["in_dtype"] == "bf16" else 4
        values = tokens * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": values * (size + 2), "flops": 3 * tokens * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if c["op"] == "attention":
        size = 2 if c["out_dtype"] == "bf16" else 4
        tokens = keys = pairs = 0
        for n, kv in _lengths(c):
            k, p = _visible(c, n, kv)
            tokens, keys, pairs = tokens + n, keys + k, pairs + p
        return {"bytes": tokens * c["heads"] * c["dim"] * (2 + size) + keys * c["kv_heads"] * c["dim"] * 4,
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if c["op"] == "copy":
        return {"bytes": 2 * 2 * c["pairs"] * c["layers"] * c["page"] * c["kv_heads"] * c["dim"] * 2, "flops": 0}
    rows = c["groups"] * c["beams"]
    return {"bytes": rows * c["vocab"] * (4 if c["dtype"] == "f32" else 2) + c["groups"] * c["keep"] * 12, "flops": 4 * rows * c["vocab"]}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


# ---- inputs ------------------------------------------------------------------------------

def _paged(c, g):
    """The page table, lengths and a cache whose pages are handed out in no order; slots that hold no token keep old values."""
    lens = _lengths(c)
    need = [-(-kv // c["page"]) for _, kv in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(c["seqs"], max(need), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    shape = (n_pages, c["kv_heads"], c["page"], c["dim"])
    k = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    v = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    return dict(page_table=table, q_start=torch.tensor(starts, dtype=torch.int32, device=DEV),
                kv_lens=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV), k_cache=k, v_cache=v,
                max_q=max(n for n, _ in lens), max_kv=max(kv for _, kv in lens), tokens=starts[-1])


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "rope":
        s.update(_paged(c, g))
        dt = torch.bfloat16 if c["in_dtype"] == "bf16" else torch.float32
        # the fused projection's output: q, k and v of a token beside one another
        wide = torch.randn(s["tokens"], c["heads"] + 2 * c["kv_heads"], c["dim"], generator=g, device=DEV).to(dt)
        s["q"], s["k"], s["v"] = wide.split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
        i = torch.arange(c["rotary"] // 2, dtype=torch.float64, device=DEV)
        s["turns"] = c["base"] ** (-2 * i / c["rotary"]) / c["stretch"] / (2 * math.pi)   # turns a position
    elif c["op"] == "attention":
        s.update(_paged(c, g))
        s["q"] = torch.randn(s["tokens"], c["heads"], c["dim"], generator=g, device=DEV).to(torch.bfloat16)
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, c["heads"] + 1, device=DEV, dtype=torch.float32) / c["heads"]) if c["alibi"] else None
        s["prefix"] = torch.clamp(s["kv_lens"], max=c["prefix"]).to(torch.int32) if c["prefix"] else None
    elif c["op"] == "copy":
        shape = (c["layers"], c["pages"], c["kv_heads"], c["page"], c["dim"])
        s["k_cache"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
        s["v_cache"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
        r = random.Random(seed)
        ids = r.sample(range(c["pages"]), 2 * c["pairs"])
        s["pairs"] = torch.tensor(list(zip(ids[:c["pairs"]], ids[c["pairs"]:])), dtype=torch.int32)   # the allocator's list, on the host
    else:
        logits = 2.0 * torch.randn(c["groups"] * c["beams"], c["vocab"], generator=g, device=DEV)
        logits[:, :: 7] = -math.inf   # tokens that a constraint rules out
        s["logits"] = logits.to(torch.float32 if c["dtype"] == "f32" else torch.bfloat16)
        s["scores"] = -4.0 * torch.rand(c["groups"], c["beams"], generator=g, device=DEV)
        if c["first"]:
            s["scores"][:, 1:] = -math.inf
            s["scores"][:, 0] = 0.0
    return s


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from bybylang_b200 import kvcache as kv
    c = s["case"]
    if c["op"] == "rope":
        q = kv.rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_lens"], s["turns"],
                           layout=c["layout"])
        return [q, s["k_cache"], s["v_cache"]]
    if c["op"] == "attention":
        return kv.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_lens"], max_q=s["max_q"],
                                  max_kv=s["max_kv"], softcap=c["softcap"], slopes=s["slopes"], window=c["window"], prefix_lens=s["prefix"],
                                  out_dtype=torch.bfloat16 if c["out_dtype"] == "bf16" else torch.float32)
    if c["op"] == "copy":
        kv.copy_pages(s["k_cache"], s["v_cache"], s["pairs"])
        return [s["k_cache"], s["v_cache"]]
    return list(kv.beam_select(s["logits"], s["scores"], c["keep"]))


def _tokens_of(s):
    """Each new token's sequence and its position in that sequence's cache."""
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["q_start"][1:], t, right=True)
    return t, b, s["kv_lens"][b] - s["q_start"][b + 1] + t


def _run_plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return _plain_rope(s, c)
    if c["op"] == "attention":
        return _plain_attention(s, c)
    if c["op"] == "copy":
        src, dst = s["pairs"].to(DEV).long().unbind(1)
        s["k_cache"][:, dst] = s["k_cache"][:, src]
        s["v_cache"][:, dst] = s["v_cache"][:, src]
        return [s["k_cache"], s["v_cache"]]
    return _plain_beams(s, c)


def _plain_rope(s, c):
    _, b, pos = _tokens_of(s)
    # the angle's whole turns are taken off in 64 bits: at position 30000 a 32-bit product has lost three digits of it
    turn = pos[:, None].double() * s["turns"][None]
    ang = (turn - torch.floor(turn)).float()[:, None] * (2 * math.pi)
    cos, sin = torch.cos(ang), torch.sin(ang)
    r = c["rotary"]

    def turned(x):
        x = x.float()
        if c["layout"] == "half":
            a, z = x[..., :r // 2], x[..., r // 2:r]
            return torch.cat([a * cos - z * sin, a * sin + z * cos, x[..., r:]], -1)
        a, z = x[..., 0:r:2], x[..., 1:r:2]
        return torch.cat([torch.stack([a * cos - z * sin, a * sin + z * cos], -1).flatten(-2), x[..., r:]], -1)

    page = s["page_table"][b, torch.div(pos, c["page"], rounding_mode="floor").long()].long()[:, None]
    slot, head = (pos % c["page"]).long()[:, None], torch.arange(c["kv_heads"], device=DEV)[None]
    s["k_cache"][page, head, slot] = turned(s["k"]).to(torch.bfloat16)
    s["v_cache"][page, head, slot] = s["v"].to(torch.bfloat16)
    return [turned(s["q"]).to(torch.bfloat16), s["k_cache"], s["v_cache"]]


def _plain_attention(s, c):
    B, H, Hk, D = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    nq, nk = s["max_q"], s["max_kv"]
    pages = s["page_table"][:, : -(-nk // c["page"])].long()
    k = s["k_cache"][pages].transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :nk].float()
    v = s["v_cache"][pages].transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :nk].float()
    j = torch.arange(nk, device=DEV, dtype=torch.int32)
    kv_len = s["kv_lens"][:, None]
    v = torch.where((j[None] < kv_len)[:, None, :, None], v, 0.0)
    i = torch.arange(nq, device=DEV, dtype=torch.int32)
    n = (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    at = torch.where(i[None] < n, s["q_start"][:-1, None] + i[None], 0).long()
    q = s["q"][at].float().view(B, nq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    score = torch.matmul(q, k.transpose(2, 3)).view(B, H, nq, nk)
    score *= D ** -0.5
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    pos = kv_len - n + i[None]                       # [B, nq]
    dist = pos[:, :, None] - j[None, None]           # [B, nq, nk]
    if s["slopes"] is not None:
        score -= s["slopes"].view(1, H, 1, 1) * dist.abs()[:, None].float()
    seen = dist >= 0
    if s["prefix"] is not None:
        seen = seen | (j[None, None] < s["prefix"][:, None, None])
    if c["window"]:
        seen = seen & (dist < c["window"])
    seen = seen & (j[None] < kv_len)[:, None]
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top == -math.inf, 0.0, top)
    score.exp_()
    total = score.sum(-1)
    out = torch.matmul(score.view(B, Hk, -1, nk), v).view(B, H, nq, D)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    t, b, _ = _tokens_of(s)
    out = out.transpose(1, 2)[b, (t - s["q_start"][b]).long()]
    return out.to(torch.bfloat16 if c["out_dtype"] == "bf16" else torch.float32)


def _plain_beams(s, c):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    score = s["scores"].reshape(-1, 1) + (x - lse)
    score = torch.where(torch.isnan(score), -math.inf, score).view(c["groups"], -1) + 0.0
    # one whole number a candidate, ordered by score and then by the lower place
    bits = score.view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = order * (1 << 32) + ((1 << 32) - 1 - torch.arange(score.shape[1], device=DEV))
    at = (1 << 32) - 1 - (torch.topk(key, c["keep"]).values & ((1 << 32) - 1))
    return [torch.gather(score, 1, at), torch.div(at, c["vocab"], rounding_mode="floor").to(torch.int32), (at % c["vocab"]).to(torch.int32)]


# ---- the same from the definitions, in 64 bits -------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "copy":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        for a, b in s["pairs"].tolist():
            k[:, b], v[:, b] = k[:, a].clone(), v[:, a].clone()
        return [k, v]
    if c["op"] == "beam":
        logp = torch.log_softmax(s["logits"].double(), -1).view(c["groups"], c["beams"], -1) + s["scores"].double()[..., None]
        logp = torch.nan_to_num(logp, nan=-math.inf, neginf=-math.inf)
        return [torch.sort(logp.flatten(1), -1, descending=True).values[:, :c["keep"]], None, None]
    starts, table, page = s["q_start"].tolist(), s["page_table"].long(), c["page"]
    if c["op"] == "rope":
        k, v, q = s["k_cache"].double(), s["v_cache"].double(), []
        r = c["rotary"]
        for b, (n, kv) in enumerate(_lengths(c)):
            pos = torch.arange(kv - n, kv, device=DEV)
            z = torch.polar(torch.ones(n, r // 2, dtype=torch.float64, device=DEV), 2 * math.pi * (pos[:, None] * s["turns"][None]))[:, None]
            new = []
            for x in (s["q"], s["k"]):
                x = x[starts[b]:starts[b + 1]].double()
                if c["layout"] == "half":
                    y = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * z
                    new.append(torch.cat([y.real, y.imag, x[..., r:]], -1))
                else:
                    y = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * z
                    new.append(torch.cat([torch.view_as_real(y).flatten(-2), x[..., r:]], -1))
            q.append(new[0])
            k[table[b, pos // page], :, pos % page] = new[1]
            v[table[b, pos // page], :, pos % page] = s["v"][starts[b]:starts[b + 1]].double()
        return [torch.cat(q), k, v]
    out = torch.zeros(s["tokens"], c["heads"], c["dim"], dtype=torch.float64, device=DEV)
    per = c["heads"] // c["kv_heads"]
    for b, (n, kv) in enumerate(_lengths(c)):
        pos = torch.arange(kv, device=DEV)
        keys = s["k_cache"][table[b, pos // page], :, pos % page]
        values = s["v_cache"][table[b, pos // page], :, pos % page]
        mine = torch.arange(kv - n, kv, device=DEV)[:, None]
        seen = pos[None] <= mine
        if s["prefix"] is not None:
            seen = seen | (pos[None] < s["prefix"][b])
        if c["window"]:
            seen = seen & (mine - pos[None] < c["window"])
        for h in range(c["heads"]):
            x = s["q"][starts[b]:starts[b + 1], h].double() @ keys[:, h // per].double().T / math.sqrt(c["dim"])
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            if s["slopes"] is not None:
                x = x - s["slopes"][h].double() * (mine - pos[None]).abs()
            x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            out[starts[b]:starts[b + 1], h] = x @ values[:, h // per].double()
    return out
