"""CPU: arguments of kernel calls that are no plain tensors or numbers, on the first call of an entry point and on later ones."""
import ctypes

import pytest
import torch

from ferrite_b200._lib import KernelLib
from ferrite_b200.models.glm import View


@pytest.fixture
def probe():
    """(library, arguments that arrived, calls that were converted argument by argument)"""
    seen, slow = [], []
    kind = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p)
    fn = kind(lambda p, i, f, s: (seen.append((p, i, f, s)), 0)[1])

    class Lib:
        def __getitem__(self, name):
            return ctypes.cast(fn, ctypes.CDLL(None)._FuncPtr)

    class Probe(KernelLib):
        def __init__(self):
            self.lib, self._fns, self._fast, self.launches, self.keep = Lib(), {"fb_probe": fn}, {}, 0, fn

        def _call_by_kind(self, *args):
            slow.append(1)
            return super()._call_by_kind(*args)

    return Probe(), seen, slow


def test_views_parameters_and_pointers_take_the_short_way_too(probe):
    k, seen, slow = probe
    t, par = torch.zeros(4, 4), torch.nn.Parameter(torch.zeros(3))
    v = View(t, 2)
    for a in (t, v, par, ctypes.c_void_p(t.data_ptr()), None, t[1]):
        k.call("fb_probe", a, 1, 0.5, stream=9)
    at = t.data_ptr()
    assert [p for p, *_ in seen] == [at, at + 8, par.data_ptr(), at, None, at + 16]
    assert all(rest == [1, 0.5, 9] for _, *rest in seen)
    assert len(slow) == 1 and k.launches == 6


@pytest.mark.parametrize("bad", ["text", b"bytes", [1], object()])
def test_arguments_that_no_kernel_takes_are_refused_every_time(probe, bad):
    k, seen, _ = probe
    for _ in range(2):
        with pytest.raises(TypeError, match="unsupported argument"):
            k.call("fb_probe", bad, 1, 0.5, stream=0)
        k.call("fb_probe", None, 1, 0.5, stream=0)
    assert len(seen) == 2
