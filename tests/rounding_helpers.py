"""What the roundings of paged attention can do to each element of its output, so that a test sees
a lost or doubled stretch of keys however long the cache is."""
import math

import torch


def exact_and_spread(bt, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=None, drop=None):
    """The definition in 64 bits for a kv_helpers.Batch: the output, sum_j p_j |v_j| and
    sqrt(sum_j p_j^2 v_j^2), each [tokens, heads, dim].  drop = (sequence, first, last): keys that
    are left out, to see what a kernel that lost them would give."""
    scale = bt.dim ** -0.5 if scale is None else scale
    per = bt.heads // bt.kv_heads
    out = [torch.zeros(bt.tokens, bt.heads, bt.dim, dtype=torch.float64) for _ in range(3)]
    q = bt.q.cpu().double()
    for b, (n, kv) in enumerate(bt.lens):
        if not n or kv <= 0:
            continue
        pos, j = torch.arange(kv - n, kv)[:, None], torch.arange(kv)[None]
        seen = j <= pos
        if prefix is not None:
            seen = seen | (j < prefix[b])
        if window:
            seen = seen & (pos - j < window)
        seen = seen & (pos >= 0)
        if drop is not None and drop[0] == b:
            seen = seen & ((j < drop[1]) | (j >= drop[2]))
        keys, values = bt.keys[b].double().repeat_interleave(per, 1), bt.values[b].double().repeat_interleave(per, 1)
        s = torch.einsum("ihd,jhd->hij", q[bt.starts[b]:bt.starts[b + 1]], keys) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.cpu().double()[:, None, None] * (pos - j).abs()
        p = torch.where(seen, torch.softmax(s.masked_fill(~seen, -math.inf), -1), 0.0)
        rows = slice(bt.starts[b], bt.starts[b + 1])
        out[0][rows] = torch.einsum("hij,jhd->ihd", p, values)
        out[1][rows] = torch.einsum("hij,jhd->ihd", p, values.abs())
        out[2][rows] = torch.einsum("hij,jhd->ihd", p.square(), values.square()).sqrt()
    return out


# Scores: an fp32 sum over a head on the tensor core, which truncates at each of its dim / 16 steps,
# is off by (dim / 16 + 2) * 2^-23 of scale * sum |q k|, 1.2e-5 for 128 dimensions of order 1, and in
# proportion to the keys' size; a cap adds 2^-22 of the score.  Twice that is a probability's relative
# error (its own and its sum's); fp32 sums add a few 1e-6.
def scores_off(size):
    return 4e-5 * size


def bf16_bound(want, total, spread, size=1.0):
    """A bf16 output: the output rounds by 2^-8 of itself.  Each probability rounds by up to 2^-8 of
    itself before the product with V: what the errors have in common moves the output by 2^-8 of
    itself, and their independent parts (uniform up to 2^-8, a standard deviation of 2^-8 / sqrt 3)
    add to 2^-8 / sqrt 3 of the spread, of which seven (some 4 of the spread) are beyond any of 10^7
    elements.  Exponentials are good to 7.5e-5 of a probability."""
    return 2 * 2.0 ** -8 * want.abs() + 4 * 2.0 ** -8 * spread + (7.5e-5 + scores_off(size)) * total


def f32_bound(want, total, spread, size=1.0):
    """An fp32 output: the scores, and probabilities of 24 bits."""
    return scores_off(size) * total
