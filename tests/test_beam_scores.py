"""beam_select's scores where a row's logits lie far from zero: masks of large negative finite
values, offsets, and beams whose own score is a sentinel."""
import math

import pytest

torch = pytest.importorskip("torch")

from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402

DEV = "cuda:0"
pytestmark = pytest.mark.gpu


def against64(logits, scores, keep, tol=None):
    """Compares a call with prior + log_softmax in 64 bits, order and scores.  Tolerance: the score
    is prior + ((x - m) - log(sum)): each of the three operations and the inputs of the last rounds
    by 2^-24 of a term that is at most |score| + |prior| + log(vocab); the sum's terms are good to 2^-22 (the
    exponential and its argument), a lane adds at most 16 of them here before some 13 joins, each
    rounding by 2^-24 of the sum, which moves its logarithm by that much."""
    got, beam, token = kv.beam_select(logits, scores, keep)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    groups, beams = scores.shape
    x = logits.cpu().double().view(groups, beams, -1)
    s = scores.cpu().double()[..., None] + torch.log_softmax(x, -1)
    want, at = torch.sort(s.flatten(1), dim=1, descending=True, stable=True)
    want, at = want[:, :keep], at[:, :keep]
    got = got.cpu().double()
    fixed = 2.0 ** -22 + 29 * 2.0 ** -24
    bound = fixed + 2.0 ** -22 * (want.abs() + scores.cpu().abs().max().double() + math.log(x.shape[2]))
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() - bound).max())
    place = beam.cpu().long() * x.shape[2] + token.cpu().long()
    mine = torch.gather(s.flatten(1), 1, place)
    assert ((mine - want).abs() <= bound).all()
    assert all(len(set(p.tolist())) == keep for p in place)
    return got, beam.cpu(), token.cpu(), at


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 4096, 4099, 128256])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -1e20, -1e30, -2.5e38, "least"])
def test_finite_masks(mask, vocab, dtype):
    """Eight free tokens of the vocabulary, the others at a large negative number: most lanes see
    nothing but masked logits."""
    g = torch.Generator().manual_seed(vocab)
    mask = float(torch.finfo(dtype).min) if mask == "least" else mask
    x = torch.full((6, vocab), mask)
    for row in range(6):
        x[row, torch.randperm(vocab, generator=g)[:8]] = 2 * torch.randn(8, generator=g)
    s = -torch.rand(2, 3, generator=g)
    x = x.to(dtype).to(DEV)
    got, beam, token, at = against64(x, s.to(DEV), 8)
    assert (got > -100).all()
    # the masked ones come last, by their own order: two free tokens a row at most stand before them
    y = torch.full((1, vocab), mask)
    y[0, [vocab // 2, 7]] = torch.tensor([1.0, 3.0])
    got, beam, token, at = against64(y.to(dtype).to(DEV), torch.zeros(1, 1, device=DEV), 6)
    assert token[0].tolist() == [7, vocab // 2, 0, 1, 2, 3]


@pytest.mark.parametrize("vocab", [1000, 32768, 128256])
@pytest.mark.parametrize("offset", [0.0, 50.0, -200.0, 200.0, -1000.0, 1000.0, -10000.0, 10000.0])
def test_offsets(offset, vocab):
    """Logits that share an offset have the same log-softmax."""
    g = torch.Generator().manual_seed(int(abs(offset)) + vocab)
    x = (2 * torch.randn(8, vocab, generator=g) + offset).to(DEV)
    s = -4 * torch.rand(2, 4, generator=g)
    against64(x, s.to(DEV), 16)


def test_offset_rows_in_bf16():
    g = torch.Generator().manual_seed(1)
    x = 2 * torch.randn(8, 32768, generator=g) + torch.tensor([0.0, 100, -100, 200, -200, 30, 500, -500])[:, None]
    against64(x.to(torch.bfloat16).to(DEV), (-4 * torch.rand(2, 4, generator=g)).to(DEV), 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("prior", [-1e9, -1e20])
def test_priors_that_swallow_the_logits(prior, dtype):
    """All of a beam's continuations round to its sentinel: they keep the order of their logits,
    equal logits that of their tokens, and a beam's order is the lower beam's first."""
    g = torch.Generator().manual_seed(11)
    x = (torch.randn(3, 5000, generator=g) * 2).to(dtype)
    x[1, 100] = x[1, 4000] = x[1].max() + 1
    s = torch.tensor([[prior, prior, 2 * prior]])
    score, beam, token = kv.beam_select(x.to(DEV), s.to(DEV), 12)
    assert beam.tolist() == [[0] * 12] and (score == prior).all()
    assert token[0].tolist() == torch.sort(x[0].float(), descending=True, stable=True).indices[:12].tolist()
    score, beam, token = kv.beam_select(x[1:].contiguous().to(DEV), torch.tensor([[prior, -1.0]], device=DEV), 64)
    assert (beam == 1).all()
    score, beam, token = kv.beam_select(x[1:2].to(DEV), torch.tensor([[prior]], device=DEV), 5)
    assert token[0].tolist() == torch.sort(x[1].float(), descending=True, stable=True).indices[:5].tolist() and token[0, :2].tolist() == [100, 4000]


def test_beams_whose_scores_round_alike():
    """Two beams with the same logits: at equal scores the lower beam comes first, each with its
    continuations in the order of their logits."""
    x = torch.full((2, 300), -50.0)
    x[:, [250, 17, 40]] = torch.tensor([2.0, 2.0 + 2.0 ** -22, 1.0])
    score, beam, token = kv.beam_select(x.to(DEV), torch.full((1, 2), -1000.0, device=DEV), 6)
    got = list(zip(beam[0].tolist(), token[0].tolist()))
    assert got == [(0, 17), (0, 250), (1, 17), (1, 250), (0, 40), (1, 40)]
