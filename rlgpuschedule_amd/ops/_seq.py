"""Loader of the sequence operators' torch bindings (librlsched_seq.so, from
csrc/seq_bind.cpp) and of the kernel libraries they are linked with."""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading

from .build import _BINDS, build_lib, verify_loaded

_NAME = "librlsched_seq"
_ext = None
_lock = threading.Lock()


def ext():
    """The binding module; built first if it is missing or stale. Threads that
    ask for it at once get the same one, which one of them loads."""
    return _ext if _ext is not None else _load()


def _load():
    global _ext
    with _lock:
        if _ext is None:
            so = f"{_NAME}.so"
            for lib in _BINDS[so]:
                verify_loaded(ctypes.CDLL(str(build_lib(lib))), lib)
            path = str(build_lib(so))
            spec = importlib.util.spec_from_file_location(
                _NAME, path,
                loader=importlib.machinery.ExtensionFileLoader(_NAME, path))
            mod = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(mod)
            verify_loaded(ctypes.CDLL(path), so)
            _ext = mod
    return _ext
