"""What the paged-cache operators refuse on the host, before any device work."""
import pytest

from bybylang_b200 import _lib
from test_kvcache import attention, cache, refused, rope

# (token stride, head stride) of 3 tokens and 8 heads of 64
OVERLAPPING = [(0, 64), (64, 64), (32, 128), (448, 64), (504, 64), (64, 128), (128, 192), (1 << 40, 1 << 39), (64, 184)]
APART = [(512, 64), (520, 64), (1024, 128), (64, 192), (64, 512), (72, 208), (1 << 40, 1 << 36)]


@pytest.mark.parametrize("token,head", OVERLAPPING)
def test_outputs_whose_vectors_overlap(token, head):
    lib = _lib.load()
    refused(lib.bybycu_rope_append(cache(), rope(out_token_stride=token, out_head_stride=head), None), _lib.ERR_ARGS, "overlapping strides")
    refused(lib.bybycu_paged_attention(cache(), attention(out_token_stride=token, out_head_stride=head), None), _lib.ERR_ARGS, "overlap")


@pytest.mark.parametrize("token,head", OVERLAPPING + APART)
def test_the_overlap_rule_against_the_elements(token, head):
    """The table above, element by element where the strides are small."""
    if token > 1 << 20:
        return
    spans = [range(t * token + h * head, t * token + h * head + 64) for t in range(3) for h in range(8)]
    places = {x for s in spans for x in s}
    assert (len(places) < 3 * 8 * 64) == ((token, head) in OVERLAPPING) or (token, head) == (128, 192)   # interleaved: refused all the same


no_device = pytest.mark.skipif("__import__('torch').cuda.is_available()", reason="addresses that must not be followed")


@no_device
@pytest.mark.parametrize("token,head", APART)
def test_outputs_whose_vectors_lie_apart(token, head):
    """Not refused: the call comes as far as the device, and there is none."""
    lib = _lib.load()
    for rc in (lib.bybycu_rope_append(cache(), rope(out_token_stride=token, out_head_stride=head), None),
               lib.bybycu_paged_attention(cache(), attention(out_token_stride=token, out_head_stride=head), None)):
        assert rc not in (_lib.ERR_ARGS, _lib.ERR_SHAPE, 0), _lib.last_error()


def test_strides_of_one_token_and_one_head():
    """The one that steps nowhere may be anything, the other may not be 0."""
    lib = _lib.load()
    refused(lib.bybycu_paged_attention(cache(kv_heads=1), attention(q_heads=1, out_token_stride=0, out_head_stride=0), None), _lib.ERR_ARGS, "overlap")
    refused(lib.bybycu_paged_attention(cache(n_tokens=1), attention(out_token_stride=0, out_head_stride=0), None), _lib.ERR_ARGS, "overlap")
    refused(lib.bybycu_paged_attention(cache(n_tokens=1), attention(out_token_stride=0, q=0), None), _lib.ERR_ARGS, "missing")


@no_device
@pytest.mark.parametrize("pairs", [33, 1 << 30, (1 << 30) + 16, (1 << 31) - 1])
def test_pairs_beyond_the_head(pairs):
    """2 * pairs may not wrap around to a number that fits."""
    refused(_lib.load().bybycu_rope_append(cache(), rope(pairs=pairs), None), _lib.ERR_SHAPE, "pairs")


@no_device
def test_launches_past_32_bits():
    lib, wide = _lib.load(), dict(q_token_stride=1 << 21, out_token_stride=1 << 21)
    one = dict(kv_heads=1, n_tokens=1 << 16)
    refused(lib.bybycu_paged_attention(cache(**one), attention(q_heads=1 << 15, max_q=1 << 16, **wide), None), _lib.ERR_SHAPE, "2^31 rows")


@no_device
@pytest.mark.parametrize("max_pages,page_size", [(524286, 4096), (1, 2 ** 31 - 8192), (2 ** 31 - 1, 1)])
def test_tables_close_to_2_31_positions(max_pages, page_size):
    kw = dict(max_pages=max_pages, page_size=page_size, table_stride=max_pages, head_stride=page_size * 64, page_stride=4 * page_size * 64)
    refused(_lib.load().bybycu_paged_attention(cache(**kw), attention(), None), _lib.ERR_SHAPE, "2^31 - 8193")
    refused(_lib.load().bybycu_rope_append(cache(**kw), rope(), None), _lib.ERR_SHAPE, "2^31 - 8193")
