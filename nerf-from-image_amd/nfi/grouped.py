"""Products grouped by ragged runs of rows (include/nfi_learn.h): the rows of a batch that mixes several heads,
each run of rows through its own head's weight.

    y[r] = weight[e] @ x[r] + bias[e]        offsets[e] <= r < offsets[e + 1]

The layer is stylegan.py:148-180's linear one (the caller scales the weight by its gain), for `groups` of them in one
launch; the offsets stay on the device.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib, learn_ops as lo

MAX_GROUPS, MAX_WIDTH = 65535, 2097152


def _args(x, weight, offsets):
    a = _lib.NfiGroupedArgs()
    a.x, a.w, a.offsets = x.data_ptr(), weight.data_ptr(), offsets.data_ptr()
    a.rows = x.shape[0]
    a.groups, a.out_width, a.in_width = weight.shape
    a.dtype = lo.TYPES[x.dtype]
    a.offsets64 = offsets.dtype == torch.int64
    return a


def _run(name, a, dev):
    size = getattr(_lib.load(), f'{name}_work_bytes')(ctypes.byref(a))
    work = None
    if size > 0:
        work = torch.empty((size,), device=dev, dtype=torch.uint8)
        a.work, a.work_bytes = work.data_ptr(), size
    with lo.on(dev):
        lo.call(name, ctypes.byref(a), lo.stream(dev))


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, bias):
        y = torch.empty((x.shape[0], weight.shape[1]), device=x.device, dtype=x.dtype)
        if y.numel():
            a = _args(x, weight, offsets)
            a.bias, a.y = lo.ptr(bias), y.data_ptr()
            _run('nfi_grouped_forward', a, x.device)
        ctx.save_for_backward(x, weight, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, offsets = ctx.saved_tensors
        need = ctx.needs_input_grad
        gx = torch.empty_like(x) if need[0] else None
        gw = torch.empty_like(weight) if need[1] else None
        gb = torch.empty(weight.shape[:2], device=x.device, dtype=x.dtype) if need[3] else None
        if x.shape[0] == 0:
            return gx, None if gw is None else gw.zero_(), None, None if gb is None else gb.zero_()
        gy = gy.contiguous()
        a = _args(x, weight, offsets)
        a.gy, a.gx, a.gw, a.gb = gy.data_ptr(), lo.ptr(gx), lo.ptr(gw), lo.ptr(gb)
        _run('nfi_grouped_backward', a, x.device)
        return gx, gw, None, gb


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None):
    """y [rows, N] of x [rows, K], weight [groups, N, K] and bias [groups, N] (or None), all float32, bfloat16 or
    float16 alike: row r of group e, offsets[e] <= r < offsets[e + 1], gives weight[e] @ x[r] + bias[e]; rows that no
    group holds give zeros.  offsets [groups + 1] int32 or int64 on the device, not decreasing (it is not read on the host:
    values outside [0, rows] count as the nearest end, and decreasing ones give wrong rows, never a wrong access).

    Sums are held in 32 bits and rounded once.  Gradients reach x, weight and bias, summed in a fixed order (no double
    backward); an empty group's weight and bias get zeros."""
    what = 'grouped_linear'
    lo.same_device(what, x, weight=weight, offsets=offsets, bias=bias)
    lo.type_code(x, what)
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1]:
        raise ValueError(f'{what}: x [rows, K] and weight [groups, N, K] are wanted, not {tuple(x.shape)} and {tuple(weight.shape)}')
    e, n, k = weight.shape
    if not 1 <= e <= MAX_GROUPS or not 1 <= n <= MAX_WIDTH or not 1 <= k <= MAX_WIDTH:
        raise ValueError(f'{what}: 1 to {MAX_GROUPS} groups and widths of 1 to {MAX_WIDTH} are wanted, not {tuple(weight.shape)}')
    if offsets.shape != (e + 1,) or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f'{what}: offsets [{e + 1}] int32 or int64 are wanted, not {tuple(offsets.shape)} {offsets.dtype}')
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise RuntimeError(f'{what}: x, weight and bias are of one type, not {x.dtype}, {weight.dtype}'
                           + ('' if bias is None else f', {bias.dtype}'))
    if bias is not None and bias.shape != (e, n):
        raise ValueError(f'{what}: bias [{e}, {n}] is wanted, not {tuple(bias.shape)}')
    return _GroupedLinear.apply(x.contiguous(), weight.contiguous(), offsets.contiguous(), None if bias is None else bias.contiguous())
