"""LinearInt4's refusals that need a layer but no kernel, on the host."""
import ctypes as C

import numpy as np
import pytest
import torch

from trba_b200.ops import LinearInt4


def test_state_of_a_layer_on_another_device_is_refused(lib):
    """The fields that come first in a layer: in, out, group, groups, device;
    no process has a device 63."""
    lib.trba_clear_error()
    layer = (C.c_int * 64)(8, 4, 32, 1, 63)
    q, s, b = np.full((4, 4), 7, np.uint8), np.full((4, 1), 7, np.float32), np.full(4, 7, np.float32)
    p = lambda a: C.c_void_p(a.ctypes.data)  # noqa: E731
    rc = lib.trba_linear_int4_get(layer, p(q), p(s), p(b))
    assert rc == -1 and b"another device" in lib.trba_last_error_string()
    lib.trba_clear_error()
    assert all((a == 7).all() for a in (q, s, b))


def test_state_is_read_on_the_layers_device(monkeypatch):
    now, used = [0], []

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            now.append(self.index)

        def __exit__(self, *exc):
            now.pop()

    class Lib:
        def trba_linear_int4_get(self, h, codes, scales, bias):
            used.append(now[-1])
            return 0

        def trba_linear_int4_destroy(self, h):
            pass

    lin = LinearInt4.__new__(LinearInt4)
    lin.L, lin.torch, lin.h, lin.device = Lib(), torch, 1, torch.device("cuda", 1)
    lin.in_features, lin.out_features, lin.group = 8, 4, 32
    monkeypatch.setattr(torch.cuda, "device", Device)
    assert lin.state()["codes"].shape == (4, 4) and used == [1] and now == [0]


def test_a_closed_layer_is_refused():
    """Before the library is called, which ends the process on a bad argument
    unless it was told not to."""
    class Lib:
        def trba_linear_int4_destroy(self, h):
            pass

    from trba_b200 import decode
    lin = LinearInt4.__new__(LinearInt4)
    lin.L, lin.torch, lin.decode, lin.h = Lib(), torch, decode, 1
    lin.device, lin.in_features, lin.out_features, lin.group = torch.device("cpu"), 8, 4, 32
    lin.close()
    lin.close()
    for call in (lambda: lin.forward(torch.zeros(2, 8)), lin.state):
        with pytest.raises(RuntimeError, match="closed"):
            call()
