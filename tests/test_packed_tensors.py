"""CPU: which tensors, addresses and formats a packed weight hands on, with a stand-in for the launches."""
import ctypes

import pytest
import torch
import torch.nn as nn

from quantization_amd import packed


class StandIn:
    """libmq.so with launches that only note the weight's addresses; sizes come from the library itself."""

    def __init__(self, real):
        self.real, self.seen = real, []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def _note(self, ref):
        c = ctypes.cast(ref, ctypes.POINTER(packed._W4)).contents
        self.seen.append((c.data, c.params, c.norm))
        return 0

    def mq_linear4(self, ref, *args):
        return self._note(ref)

    def mq_linear4_grad(self, ref, *args):
        return self._note(ref)


@pytest.fixture
def launches(monkeypatch):
    s = StandIn(packed._bind())
    monkeypatch.setattr(packed, "_bound", s)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(packed, "_on_device", lambda call, t, *args: call(t, *args, 0))
    return s


def host_weight(n=32, k=128, group=64, bits=4, fmt="int4", fill=0):
    """A weight whose tensors lie on the host."""
    c = packed._W4(experts=1, n=n, k=k, group=group, kind=packed._kind_of(bits, fmt)[0])
    L = packed._bind()
    data = torch.full((L.mq_w4_data_bytes(1, n, k) // 4,), fill, dtype=torch.int32)
    params = torch.full((L.mq_w4_params_bytes(ctypes.byref(c)) // 2,), fill, dtype=torch.int16)
    return packed.PackedWeight(data, params, torch.ones(1, dtype=torch.int32), None, n, k, group, bits, fmt)


def addresses(w):
    return w.data.data_ptr(), w.params.data_ptr(), w.norm.data_ptr()


def rows(m=3, k=128):
    return torch.zeros(m, k, dtype=torch.float16)


def run(x, w, bias=None, counts=None):
    return packed._on_device(packed._forward, x, w, bias, counts)


def test_a_tensor_with_other_storage_is_taken_up(launches):
    """t.data = other keeps the tensor object and frees its memory."""
    w = host_weight()
    run(rows(), w)
    assert launches.seen[-1] == addresses(w)
    keep = []   # (the old memory must not be given out again at the same address)
    for name in ("data", "params", "norm"):
        t = getattr(w, name)
        keep.append(t.detach())
        t.data = t.data.clone()
        run(rows(), w)
        assert launches.seen[-1] == addresses(w), name
    w.data.data = w.data.data[:-4].clone()
    with pytest.raises(ValueError):
        run(rows(), w)
