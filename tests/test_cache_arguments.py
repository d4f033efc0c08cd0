"""The page pool's and the page copies' arguments, on the host."""
import pytest

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")

from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402


@pytest.mark.parametrize("pairs", [
    [(1 << 32, 1)], [(0, (1 << 32) + 1)], torch.tensor([[0, (1 << 32) + 1]]), np.array([[0, (1 << 32) + 1]]), np.array([[0, -(1 << 32)]]),
    np.array([[0, 3000000000]], dtype=np.uint32), torch.tensor([[0.0, 1.5]]), np.array([[0.25, 1.0]]), [(0, 1.5)], [1, 2], torch.tensor([[True, False]])])
def test_pairs_that_are_no_page_ids(pairs):
    """Wider integers are not wrapped into the range of the pages, nor fractions cut off."""
    with pytest.raises(_lib.BybyCudaError, match="pairs must be whole numbers"):
        kv._pairs(pairs)


@pytest.mark.parametrize("pairs,want", [
    ([], []), ([(3, 4)], [[3, 4]]), (((3, 4), (5, 6)), [[3, 4], [5, 6]]), (torch.tensor([[3, 4]], dtype=torch.int64), [[3, 4]]),
    (torch.tensor([[3, 4]], dtype=torch.int32), [[3, 4]]), (torch.tensor([[3, 4], [5, 6]], dtype=torch.int16).t().t(), [[3, 4], [5, 6]]),
    (np.array([[3, 4]]), [[3, 4]]), (np.array([[3, 4]], dtype=np.uint32), [[3, 4]]), (np.zeros((0, 2), dtype=np.int32), []),
    (torch.tensor([[3, 5], [4, 6]], dtype=torch.int32).t(), [[3, 4], [5, 6]]), ([(-1, 2)], [[-1, 2]]), ([np.array([3, 4])], [[3, 4]])])
def test_pairs(pairs, want):
    got = kv._pairs(pairs)
    assert got.dtype == torch.int32 and got.is_contiguous() and got.tolist() == want


@pytest.mark.parametrize("pairs", [[(1, 2, 3)], [(1, 2), (3,)], torch.zeros(2, 2, 2, dtype=torch.int32), torch.tensor(3)])
def test_pairs_of_another_shape(pairs):
    with pytest.raises(_lib.BybyCudaError, match="not \\[n, 2\\]"):
        kv._pairs(pairs)


@pytest.mark.parametrize("seqs,parents", [("ab", [0, 2]), ("ab", [0, -1]), ("ab", [1, 0, 7]), ("aa", [0, 1]), ("a?", [0, 0]), ("a?", [0, 1])])
def test_a_refused_reorder_changes_nothing(seqs, parents):
    pool = kv.PagePool(8, 4)
    a, b = pool.new(), pool.new()
    pool.extend(a, 6)
    pool.extend(b, 3)
    ids = [{"a": a, "b": b, "?": 99}[x] for x in seqs]
    before = (list(pool._refs), pool.free_pages, pool.pages(a), pool.pages(b), pool.length(a), pool.length(b), sorted(pool._seqs))
    with pytest.raises(_lib.BybyCudaError):
        pool.reorder(ids, parents)
    assert before == (list(pool._refs), pool.free_pages, pool.pages(a), pool.pages(b), pool.length(a), pool.length(b), sorted(pool._seqs))


def test_reorder_to_more_and_fewer():
    pool = kv.PagePool(8, 4)
    a, b = pool.new(), pool.new()
    pool.extend(a, 6)
    pool.extend(b, 3)
    c, d, e = pool.reorder([a, b], [1, 1, 0])
    assert [pool.length(s) for s in (c, d, e)] == [3, 3, 6] and pool.pages(c) == pool.pages(d)
    f, = pool.reorder([c, d, e], [2])
    assert pool.length(f) == 6 and pool.free_pages == 6


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(max_q=1 << 31), dict(max_kv=1 << 40), dict(window=-(1 << 40)), dict(scale=1e300), dict(softcap=1e300), dict(route=1 << 33),
                                dict(max_q=2.5)], ids=str)
def test_numbers_that_do_not_fit(kw):
    from kv_helpers import Batch
    bt = Batch([(1, 20)], page=16, heads=4, kv_heads=2, dim=64, seed=1)
    with pytest.raises(_lib.BybyCudaError, match="paged_attention"):
        kv.paged_attention(bt.q, *bt.args(), **{**dict(max_q=1, max_kv=20), **kw})
    x = torch.zeros(1, 8, 64, device=bt.q.device)
    with pytest.raises(_lib.BybyCudaError, match="rope_append"):
        kv.rope_append(x[:, :4], x[:, 4:6], x[:, 6:], *bt.args(), kv.rope_frequencies(64), magnitude=1e300)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [-1, 0, 65, 1 << 40])
def test_a_keep_out_of_range(keep):
    with pytest.raises(_lib.BybyCudaError, match="keep="):
        kv.beam_select(torch.zeros(2, 100, device="cuda:0"), torch.zeros(1, 2, device="cuda:0"), keep)
