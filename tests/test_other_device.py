"""Tensors on another device than the current one: the launch goes to theirs (no second device is needed to see it)."""

import contextlib
import ctypes as ct

import pytest
import torch

from mamformer_amd import _lib, ops


@pytest.fixture
def two_devices(monkeypatch):
    """Two devices with default streams, the first one current; what a call sees of them."""
    seen = []
    current = [0]

    class Library:
        @staticmethod
        def mh_fn(*args):
            seen.append((current[0], int(args[-1])))
            return 0

    @contextlib.contextmanager
    def device(i):
        was, current[0] = current[0], i
        try:
            yield
        finally:
            current[0] = was

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "_lib", Library)
    return seen, current


def test_a_launch_goes_to_its_tensors_device(two_devices):
    seen, current = two_devices
    for i in (0, 1):
        _lib.call("mh_fn", None, ops._stream(torch.device("cuda", i)))
    assert seen == [(0, 0), (1, 0)] and current == [0]
    assert type(ops._stream(torch.device("cuda", 0))) is int     # the usual call costs no object


def test_a_handle_passes_ctypes():
    assert ct.c_void_p.from_param(_lib.StreamElsewhere(0x1230, 1)) is not None
    f = ct.CFUNCTYPE(ct.c_size_t, ct.c_void_p)(lambda p: p or 0)
    assert f(_lib.StreamElsewhere(0x1230, 1)) == 0x1230
