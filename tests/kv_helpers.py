"""A paged batch in no particular order and the definitions of the paged-cache operators in 64 bits."""
import math

import torch

DEV = "cuda:0"


class Batch:
    """lens: [(new tokens, cached tokens)].  Every slot that holds no token, and a spare page, is
    NaN; table entries past a sequence's pages are -1; pages and rows come in random order."""

    def __init__(self, lens, *, page, heads, kv_heads, dim, seed=0, token_major=False, pad_pages=0, q_pad=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.heads, self.kv_heads, self.dim = lens, page, heads, kv_heads, dim
        need = [max(0, -(-kv // page)) for _, kv in lens]
        self.n_pages = sum(need) + 2
        width = max([1] + need) + pad_pages
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = order.pop()
        shape = (self.n_pages, page, kv_heads, dim) if token_major else (self.n_pages, kv_heads, page, dim)
        k = torch.full(shape, float("nan"), dtype=torch.bfloat16)
        v = torch.full(shape, float("nan"), dtype=torch.bfloat16)
        if token_major:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.keys, self.values = [], []
        for b, (_, kv) in enumerate(lens):
            kk = torch.randn(max(kv, 0), kv_heads, dim, generator=g).mul(spread).to(torch.bfloat16)
            vv = torch.randn(max(kv, 0), kv_heads, dim, generator=g).to(torch.bfloat16)
            for j in range(kv):
                k[table[b, j // page], :, j % page] = kk[j]
                v[table[b, j // page], :, j % page] = vv[j]
            self.keys.append(kk)
            self.values.append(vv)
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.starts, self.tokens = starts, starts[-1]
        self.table = table.to(DEV)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.kv_lens = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
        # the strides survive the copy to the device
        self.k = torch.empty_strided(k.shape, k.stride(), dtype=k.dtype, device=DEV).copy_(k)
        self.v = torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device=DEV).copy_(v)
        wide = torch.randn(self.tokens, heads + q_pad, dim, generator=g).to(torch.bfloat16)
        self.q = wide.to(DEV)[:, :heads]
        self.max_q = max([0] + [n for n, _ in lens])
        self.max_kv = max([0] + [kv for _, kv in lens])

    def args(self):
        return self.k, self.v, self.table, self.q_start, self.kv_lens


def attention64(bt, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None):
    """The operator's definition on the CPU in 64 bits: [tokens, heads, dim]."""
    scale = bt.dim ** -0.5 if scale is None else scale
    per = bt.heads // bt.kv_heads
    out = torch.zeros(bt.tokens, bt.heads, bt.dim, dtype=torch.float64)
    q = bt.q.cpu().double()
    for b, (n, kv) in enumerate(bt.lens):
        if not n or kv <= 0:
            continue
        pos = torch.arange(kv - n, kv)[:, None]
        j = torch.arange(kv)[None]
        seen = j <= pos
        if prefix is not None:
            seen = seen | (j < prefix[b])
        if window:
            seen = seen & (pos - j < window)
        seen = seen & (pos >= 0)
        keys = bt.keys[b].double().repeat_interleave(per, 1)
        values = bt.values[b].double().repeat_interleave(per, 1)
        s = torch.einsum("ihd,jhd->hij", q[bt.starts[b]:bt.starts[b + 1]], keys) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.cpu().double()[:, None, None] * (pos - j).abs()
        s = s.masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        p = torch.where(seen, p, 0.0)   # a row that sees nothing
        out[bt.starts[b]:bt.starts[b + 1]] = torch.einsum("hij,jhd->ihd", p, values)
    return out
