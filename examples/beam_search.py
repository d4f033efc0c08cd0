"""Beam search with a small decoder on 4-bit weights: what the operators of bybylang_b200.kvcache are for.

    python examples/beam_search.py [--beams 4] [--tokens 12] [--prompts 3]

One step is, per layer: the Q4B32 projection of q, k and v; rope_append (turned queries, new keys
and values into their pages); paged_attention; the output and feed-forward projections.  The LM
head's logits go to beam_select, PagePool.reorder forks the surviving beams, and copy_pages gives
each beam that writes into a shared page one of its own.  Weights are random, so the text means
nothing; ``check`` scores the found sequences again without a cache, in fp32 torch.
"""
import argparse
import math
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from bybylang_b200 import gpubackend as gb  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402
from bybylang_b200.session_vm import TileFormatQ4B32  # noqa: E402

DEV = "cuda:0"


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


class Decoder:
    """A pre-norm decoder with grouped heads, rotary positions and a gated feed-forward block."""

    def __init__(self, *, vocab=1000, hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=512, page_size=16, pages=256, seed=0):
        g = torch.Generator().manual_seed(seed)

        def weights(n, k):
            nib = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
            scales = torch.full((n, k // 32), 0.25 / math.sqrt(k)).to(torch.float16)
            return gb.Q4B32Weights(nib, scales, device=DEV)

        self.heads, self.kv_heads, self.dim, self.vocab = heads, kv_heads, head_dim, vocab
        self.embed = torch.randn(vocab, hidden, generator=g).to(DEV)
        self.qkv = [weights((heads + 2 * kv_heads) * head_dim, hidden) for _ in range(layers)]
        self.out = [weights(hidden, heads * head_dim) for _ in range(layers)]
        self.gate = [weights(ffn, hidden) for _ in range(layers)]
        self.up = [weights(ffn, hidden) for _ in range(layers)]
        self.down = [weights(hidden, ffn) for _ in range(layers)]
        self.head = weights(vocab, hidden)
        self.turns = kv.rope_frequencies(head_dim, 10000.0, device=DEV)
        self.cache = kv.PagedKvCache(layers, pages, kv_heads, head_dim, page_size, device=DEV)
        self.pool = kv.PagePool(pages, page_size)

    def step(self, seqs, tokens):
        """Logits of each sequence's last new token; `tokens` has a list of new tokens for each."""
        for s, t in zip(seqs, tokens):
            pairs = self.pool.extend(s, len(t))
            if pairs:
                self.cache.copy(pairs)
        table, kv_lens = self.pool.table(seqs, device=DEV)
        ends = torch.tensor([len(t) for t in tokens]).cumsum(0)
        q_start = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).to(DEV)
        batch = table, q_start, kv_lens
        max_q, max_kv = max(map(len, tokens)), max(self.pool.length(s) for s in seqs)
        x = self.embed[torch.tensor([t for ts in tokens for t in ts], device=DEV)]
        for i in range(len(self.qkv)):
            qkv = self.qkv[i].matmul(norm(x)).view(-1, self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            q = kv.rope_append(q, k, v, *self.cache.layer(i), *batch, self.turns)
            a = kv.paged_attention(q, *self.cache.layer(i), *batch, max_q=max_q, max_kv=max_kv)
            x = x + self.out[i].matmul(a.flatten(1))
            h = norm(x)
            x = x + self.down[i].matmul(torch.nn.functional.silu(self.gate[i].matmul(h)) * self.up[i].matmul(h))
        return self.head.matmul(norm(x[ends.to(DEV) - 1]))

    def beam_search(self, prompts, beams, n_tokens):
        """[(score, new tokens) of each beam, best first] for each prompt."""
        groups = len(prompts)
        seqs = [self.pool.new() for _ in prompts]
        logits = self.step(seqs, prompts)
        # every group starts from its prompt alone
        scores, _, token = kv.beam_select(logits, torch.zeros(groups, 1, device=DEV), beams)
        live = [[self.pool.fork(s) for _ in range(beams)] for s in seqs]
        for s in seqs:
            self.pool.free(s)
        texts = [[[t] for t in row] for row in token.tolist()]
        for _ in range(n_tokens - 1):
            flat = [s for group in live for s in group]
            logits = self.step(flat, [[t[-1]] for row in texts for t in row])
            scores, parent, token = kv.beam_select(logits, scores.contiguous(), beams)
            parent, token = parent.tolist(), token.tolist()
            live = [self.pool.reorder(group, p) for group, p in zip(live, parent)]
            texts = [[row[p] + [t] for p, t in zip(ps, ts)] for row, ps, ts in zip(texts, parent, token)]
        for group in live:
            for s in group:
                self.pool.free(s)
        return [list(zip(sc, row)) for sc, row in zip(scores.tolist(), texts)]

    def check(self, prompt, text):
        """The log-probability of `text` after `prompt`, recomputed without a cache in fp32."""
        def dense(w):
            return gb.dequant(TileFormatQ4B32, w.packed, torch.empty(w.N, w.K, device=DEV), K=w.K, N=w.N, scale_base=w.scale_base)

        ids = torch.tensor(prompt + text, device=DEV)
        n, x = len(ids), self.embed[ids]
        ang = 2 * math.pi * (torch.arange(n, device=DEV)[:, None].double() * self.turns)
        cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

        def turned(y):
            a, b = y.chunk(2, -1)
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

        for i in range(len(self.qkv)):
            q, k, v = (norm(x) @ dense(self.qkv[i]).T).view(n, -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], 1)
            per = self.heads // self.kv_heads
            s = torch.einsum("ihd,jhd->hij", turned(q), turned(k).repeat_interleave(per, 1)) * self.dim ** -0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -math.inf).softmax(-1)
            x = x + torch.einsum("hij,jhd->ihd", s, v.repeat_interleave(per, 1)).flatten(1) @ dense(self.out[i]).T
            h = norm(x)
            x = x + (torch.nn.functional.silu(h @ dense(self.gate[i]).T) * (h @ dense(self.up[i]).T)) @ dense(self.down[i]).T
        logp = (norm(x) @ dense(self.head).T).log_softmax(-1)
        return float(sum(logp[len(prompt) - 1 + i, t] for i, t in enumerate(text)))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=12)
    ap.add_argument("--prompts", type=int, default=3)
    a = ap.parse_args(argv)
    gb.ensureGpuInit(gb.GpuBackend.gbCuda, 0)
    model = Decoder()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.vocab, (7 + 9 * i,), generator=g).tolist() for i in range(a.prompts)]
    found = model.beam_search(prompts, a.beams, a.tokens)
    for prompt, beams in zip(prompts, found):
        for score, text in beams:
            print(f"{score:9.4f} (again without a cache {model.check(prompt, text):9.4f})  {text}")
        print()
    return model, prompts, found


if __name__ == "__main__":
    main()
