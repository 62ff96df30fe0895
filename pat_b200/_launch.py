"""Cheap calls into the library for operators whose kernels take a few microseconds.

An argument check of a tensor costs Python about as much as a small launch costs the GPU.  The operators
that use this module check everything once per *signature* - types, shapes, strides and devices of the
arguments, never their addresses or contents - and keep the part of the argument structure that
follows from it as bytes; a call with a known signature only adds the pointers."""
from __future__ import annotations

import torch

_LIMIT = 1024          # signatures kept per operator


class Signatures(dict):
    """signature -> what the checks of an operator returned for it."""

    def remember(self, sig, value):
        if len(self) >= _LIMIT:
            self.clear()
        self[sig] = value
        return value


def strides_of(t: torch.Tensor):
    """Strides with those of one-element dimensions, which nobody uses and torch leaves arbitrary, set to
    dense ones."""
    out, dense = list(t.stride()), 1
    for i in reversed(range(t.dim())):
        if t.shape[i] <= 1:
            out[i] = dense
        dense = max(dense, out[i] * t.shape[i])
    return out


def struct_tail(args, head_bytes: int) -> bytes:
    """The bytes of a ctypes structure behind its leading pointers."""
    return bytes(args)[head_bytes:]


def launch(fn, args, index: int) -> int:
    """Calls ``fn(args, stream)`` on the current stream of device ``index``, with that device current."""
    if torch._C._cuda_getDevice() == index:
        return fn(args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return fn(args, torch._C._cuda_getCurrentRawStream(index))
