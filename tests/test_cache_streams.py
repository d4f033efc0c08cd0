"""The streams of the paged-cache operators."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from bybylang_b200 import _lib  # noqa: E402
from bybylang_b200 import kvcache as kv  # noqa: E402

DEV = "cuda:0"


def test_a_stream_of_another_device_is_refused(monkeypatch):
    """On the host: the default stream has the same handle on every device, so the handle alone
    would launch on the current device with another one's addresses."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    own, other = SimpleNamespace(cuda_stream=0, device_index=0), SimpleNamespace(cuda_stream=0, device_index=1)
    assert kv._stream("op", 0, own) == 0
    with pytest.raises(_lib.BybyCudaError, match="the stream is on cuda:1, the tensors are on cuda:0"):
        kv._stream("op", 0, other)
    for stream in (own, other):
        with pytest.raises(_lib.BybyCudaError, match="on cuda:1, the current device is cuda:0"):
            kv._stream("op", 1, stream)


# ---- outputs of calls on another stream ------------------------------------------------------

def freed_block(n_bytes):
    """The address of a block that the current stream has just given back: the allocator's next of
    that size on this stream."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    x = torch.empty(n_bytes, dtype=torch.uint8, device=DEV)
    at = x.data_ptr()
    del x
    return at


def calls():
    """name -> (bytes of the output, a call that allocates it)"""
    from kv_helpers import Batch
    bt = Batch([(20, 700), (12, 12)], page=16, heads=64, kv_heads=4, dim=128, seed=1)
    qkv = torch.randn(32, 64 + 8, 128, generator=torch.Generator().manual_seed(2)).to(DEV)
    q, k, v = qkv.split([64, 4, 4], 1)
    turns = kv.rope_frequencies(128, device=DEV)
    x, s = torch.randn(4, 999, generator=torch.Generator().manual_seed(3)).to(DEV), torch.zeros(2, 2, device=DEV)
    return {"rope_append": (32 * 64 * 128 * 2, lambda st: kv.rope_append(q, k, v, *bt.args(), turns, stream=st)),
            "paged_attention": (32 * 64 * 128 * 2, lambda st: kv.paged_attention(bt.q, *bt.args(), max_q=20, max_kv=700, stream=st)),
            "beam_select": (2 * 8 * 4, lambda st: kv.beam_select(x, s, 8, stream=st)[0])}


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rope_append", "paged_attention", "beam_select"])
def test_outputs_come_from_the_stream_that_writes_them(name):
    """A block that the current stream may still be using is not written by another one."""
    size, call = calls()[name]
    want = call(None).clone()
    at = freed_block(size)
    out = call(None)
    assert out.data_ptr() == at                       # what the other stream must not get
    del out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    at = freed_block(size)
    out = call(s)
    assert out.data_ptr() != at
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    out.record_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def weights(kind):
    from bybylang_b200 import gpubackend as gb
    gb.ensureGpuInit(gb.GpuBackend.gbCuda, 0)
    g = torch.Generator().manual_seed(4)
    wq = torch.randint(0, 256, (512, 128), generator=g, dtype=torch.uint8)
    if kind == "Q4B32":
        return gb.Q4B32Weights(wq, torch.full((512, 8), 0.05).to(torch.float16), device=DEV)
    return gb.Q4AsymWeights(wq, torch.full((512, 8), 0.05), torch.full((512, 8), 7.5), K=256, group_size=32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["Q4B32", "Q4"])
def test_projections_come_from_the_stream_that_writes_them(kind):
    w = weights(kind)
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(5)).to(DEV)
    want = w.matmul(x).clone()
    size = 4 * 512 * 4
    at = freed_block(size)
    out = w.matmul(x)
    assert out.data_ptr() == at
    del out
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    at = freed_block(size)
    out = w.matmul(x, stream=s)
    assert out.data_ptr() != at
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
