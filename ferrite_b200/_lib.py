"""ctypes loader for the sm_100a kernel library (``libferrite_b200_kernels.so``).

The library is built in-tree by :mod:`ferrite_b200.build`.  Loading checks the build id
baked into the binary against the hash of the sources on disk and refuses a stale pair.
On a machine with a GPU the ops fail loudly when the library is missing: there is no eager
fallback behind the CUDA path.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path
from typing import Optional

import torch

_PKG = Path(__file__).resolve().parent
_LIB_PATH = _PKG / "libferrite_b200_kernels.so"


class KernelError(RuntimeError):
    pass


_Tensor = torch.Tensor
_NUMBERS = frozenset((int, float, bool, type(None)))


def _argument(a, name: str):
    """What a call hands to ctypes for an argument that is neither a plain tensor nor a plain number."""
    if hasattr(a, "data_ptr"):      # a View, a Parameter
        return a.data_ptr()
    if isinstance(a, (int, float, ctypes._SimpleCData, ctypes.Array, ctypes._Pointer)):
        return a
    raise TypeError(f"{name}: unsupported argument {type(a)}")


class KernelLib:
    def __init__(self, path: Path = _LIB_PATH, check_build_id: bool = True):
        if not path.exists():
            raise KernelError(f"{path} is missing: run `python -m ferrite_b200.build`")
        self.path = path
        self.lib = ctypes.CDLL(str(path))
        self.lib.fb_build_id.restype = ctypes.c_char_p
        self.build_id = self.lib.fb_build_id().decode()
        if check_build_id and (_PKG.parent / "csrc" / "kernels").exists():
            from .build import kernel_build_id
            want = kernel_build_id()
            if want != self.build_id:
                raise KernelError(f"stale kernel library: built from {self.build_id}, sources are {want}; "
                                  "rebuild with `python -m ferrite_b200.build`")
        self._fns = {}
        self._fast = {}
        self.launches = 0  # kernels launched through this handle (entry points, not replays)

    def fn(self, name: str):
        f = self._fns.get(name)
        if f is None:
            f = getattr(self.lib, name)
            f.restype = ctypes.c_int
            self._fns[name] = f
        return f

    def call(self, name: str, *args, stream: Optional[int] = None):
        if stream is None:
            stream = torch.cuda.current_stream().cuda_stream
        fast = self._fast.get(name)
        rc = None
        if fast is not None:   # argument kinds are known from the first call: ctypes converts plain numbers by itself
            try:
                rc = fast(*[a.data_ptr() if type(a) is _Tensor else a if type(a) in _NUMBERS else _argument(a, name) for a in args], stream)
            except ctypes.ArgumentError:
                rc = None
        if rc is None:
            rc = self._call_by_kind(name, args, stream)
        self.launches += 1
        if rc != 0:
            raise KernelError(f"{name} failed with CUDA error {rc}")

    def _call_by_kind(self, name: str, args, stream: int) -> int:
        cargs = []
        for a in args:
            if isinstance(a, torch.Tensor) or hasattr(a, "data_ptr"):
                cargs.append(ctypes.c_void_p(a.data_ptr()))
            elif a is None:
                cargs.append(ctypes.c_void_p(0))
            elif isinstance(a, bool):
                cargs.append(ctypes.c_int64(int(a)))
            elif isinstance(a, int):
                cargs.append(ctypes.c_int64(a))
            elif isinstance(a, float):
                cargs.append(ctypes.c_float(a))
            elif isinstance(a, (ctypes._SimpleCData, ctypes.Array, ctypes._Pointer)):
                cargs.append(a)
            else:
                raise TypeError(f"{name}: unsupported argument {type(a)}")
        cargs.append(ctypes.c_void_p(stream))
        rc = self.fn(name)(*cargs)
        if name not in self._fast and all(type(c) in (ctypes.c_void_p, ctypes.c_int64, ctypes.c_float) for c in cargs):
            fast = self.lib[name]   # a function object of its own: the other one keeps taking arguments of any kind
            fast.restype = ctypes.c_int
            fast.argtypes = [type(c) for c in cargs]
            self._fast[name] = fast
        return rc


_LIB: Optional[KernelLib] = None


def lib() -> KernelLib:
    global _LIB
    if _LIB is None:
        _LIB = KernelLib()
    return _LIB


def have_lib() -> bool:
    return _LIB_PATH.exists()


def ptr(t: torch.Tensor, offset_elems: int = 0) -> ctypes.c_void_p:
    """Raw pointer into a tensor's storage, offset by elements (for column views)."""
    return ctypes.c_void_p(t.data_ptr() + offset_elems * t.element_size())
