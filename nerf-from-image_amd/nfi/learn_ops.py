"""What the operators of include/nfi_learn.h share on the Python side: type codes, checks, calls."""

from __future__ import annotations

import torch

from . import _lib
from .ops import _stream

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_fns = {}


def call(name, *args):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.load(), name)
    rc = fn(*args)
    if rc:
        _lib.check(rc, name)


def ptr(t):
    return None if t is None else t.data_ptr()


def stream(dev):
    return _stream(dev)


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on(dev):
    """A context with `dev` as the current device (a launch goes to the current device's streams)."""
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def type_code(t, what):
    code = TYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f'{what}: float32, bfloat16 or float16 is wanted, not {t.dtype}')
    return code


def same_device(what, first, **others):
    """Every tensor on `first`'s HIP device."""
    if not first.is_cuda:
        raise RuntimeError(f'{what}: nfi ops run on HIP devices only (got a {first.device.type} tensor)')
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f'{what}: {name} is on {t.device}, the first input on {first.device}')
