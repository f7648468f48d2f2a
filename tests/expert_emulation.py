"""Runs dimo_amd/experts.py (and mx4.py) on host tensors through the CPU SIMT emulation of the expert kernels.  Test
infrastructure only: the product has no CPU path, this swaps the loaded library for the emulated one."""
import contextlib
import ctypes as C

from dimo_amd import _lib
from tests.simt import build as simt_build

_L = None


def emulated_library():
    global _L
    if _L is None:
        L = C.CDLL(simt_build.build(target="experts"))
        for name, (res, args) in _lib._SIGNATURES.items():
            if hasattr(L, name):
                getattr(L, name).restype, getattr(L, name).argtypes = res, args
        _L = L
    return _L


def use(monkeypatch, *modules):
    """Points the modules' calls at the emulated library and lets them take host tensors."""
    L = emulated_library()
    monkeypatch.setattr(_lib, "lib", lambda: L)
    monkeypatch.setattr(_lib, "current_stream", lambda: None)
    for m in modules:
        monkeypatch.setattr(m, "_gpu", lambda *t: t[0].device)
        monkeypatch.setattr(m, "_on", lambda device: contextlib.nullcontext())
