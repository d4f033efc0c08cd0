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
