"""What the sequence operators' bindings share (norm.py, scan.py,
logprob.py): element types, row layouts, argument checks, and the guard
around captured backward passes."""
from __future__ import annotations

import ctypes
import weakref

import torch

from .build import build_lib, verify_loaded

# element type codes of csrc/seq_common.h
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

P, I64, I32, F64 = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int,
                    ctypes.c_double)


def load_lib(name: str, signatures: dict) -> ctypes.CDLL:
    """dlopen one library; signatures: {function: [argument types]}."""
    lib = ctypes.CDLL(str(build_lib(name)))
    verify_loaded(lib, name)
    for fn, args in signatures.items():
        f = getattr(lib, fn)
        f.restype = I64 if fn.endswith(("_parts", "_scratch")) else I32
        f.argtypes = args
    return lib


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed: {rc}")


def type_code(t: torch.Tensor, name: str) -> int:
    code = TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, "
                        f"got {t.dtype}")
    return code


def same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def where(t: torch.Tensor) -> tuple[int, int]:
    """Device ordinal and that device's current stream."""
    i = t.device.index
    return i, torch.cuda.current_stream(i).cuda_stream


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def rows_of(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t [..., D] as rows of unit stride: (tensor, elements from one row to
    the next). Leading dims that no single stride walks, and last dims of
    another stride, are copied."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    t2 = t.reshape(-1, d)
    if d > 1 and t2.stride(1) != 1:
        t2 = t2.contiguous()
    return t2, t2.stride(0)


# ---- captured backward passes ---------------------------------------------
# torch runs a leaf's gradient accumulation on the stream that was current
# when the leaf first entered a live graph. If that was an eager stream, a
# backward pass under capture has to synchronise with it, which ends the
# process. Each graph made by these operators leaves a note of its leaves and
# stream, for as long as it lives; a capture that meets a note of another
# stream is refused while it can still be refused.

class _Note:
    __slots__ = ("stream", "leaves", "__weakref__")

    def __init__(self, stream, leaves):
        self.stream, self.leaves = stream, leaves


_notes: weakref.WeakSet = weakref.WeakSet()


def note_leaves(*tensors) -> _Note | None:
    """To be kept on the autograd context of the operator's call."""
    leaves = [t for t in tensors
              if t is not None and t.requires_grad and t.grad_fn is None]
    if not leaves:
        return None
    stream = torch.cuda.current_stream(leaves[0].device.index).cuda_stream
    if torch.cuda.is_current_stream_capturing():
        for note in list(_notes):
            if note.stream != stream and any(
                    r() is t for r in note.leaves for t in leaves):
                raise RuntimeError(
                    "an eager autograd graph of the same leaves is alive: "
                    "its backward pass cannot be captured. Release that "
                    "graph (its outputs and losses) before the capture, or "
                    "use the operator's _fwd and _bwd functions.")
    note = _Note(stream, [weakref.ref(t) for t in leaves])
    _notes.add(note)
    return note
