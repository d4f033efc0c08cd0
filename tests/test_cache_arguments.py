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
