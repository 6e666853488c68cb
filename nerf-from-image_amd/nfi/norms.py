"""The norm of a block's output fused with what a residual trunk does around it (include/nfi_learn.h):

    x = scale * (residual + gate * leaky_relu(norm(h) * weight + bias, slope))
    y = next_norm(x) * next_weight + next_bias

One pass over memory each way.  The mapper trunks of the reference (generator.py:132-253) are made of it:
LayerNorm, LeakyReLU(0.2), shortcut, sqrt(2) / 2; the gate is a width's, an image's or a row's own factor, and
the next block's norm reads the new residual before it is rounded.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib, learn_ops as lo

KINDS = {None: 0, 'layer': 1, 'rms': 2}
MAX_WIDTH = 8192


def _args(h, residual, gate, weight, bias, next_weight, next_bias, conf):
    norm, next_norm, slope, scale, eps = conf
    a = _lib.NfiResnormArgs()
    a.h, a.residual, a.gate, a.weight, a.bias = map(lo.ptr, (h, residual, gate, weight, bias))
    a.next_weight, a.next_bias = lo.ptr(next_weight), lo.ptr(next_bias)
    a.rows, a.width = h.shape
    p = next((t for t in (weight, bias, next_weight, next_bias) if t is not None), h)
    a.affine_groups = p is not h and p.dim() == 2
    a.groups = gate.shape[0] if gate is not None else p.shape[0] if a.affine_groups else 0
    a.dtype = lo.TYPES[h.dtype]
    a.gate_dtype = a.dtype if gate is None else lo.TYPES[gate.dtype]
    a.param_dtype = lo.TYPES[p.dtype]
    a.norm, a.next_norm, a.slope, a.scale, a.eps = norm, next_norm, slope, scale, eps
    return a


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, residual, gate, weight, bias, next_weight, next_bias, conf):
        a = _args(h, residual, gate, weight, bias, next_weight, next_bias, conf)
        x = torch.empty_like(h)
        y = torch.empty_like(h) if conf[1] else None
        train = any(ctx.needs_input_grad[:7])
        stats = torch.empty((h.shape[0], 4), device=h.device, dtype=torch.float32) if train else None
        a.x, a.y, a.stats = lo.ptr(x), lo.ptr(y), lo.ptr(stats)
        if h.shape[0]:
            with lo.on(h.device):
                lo.call('nfi_resnorm_forward', ctypes.byref(a), lo.stream(h.device))
        ctx.conf = conf
        ctx.set_materialize_grads(False)
        if train:
            ctx.save_for_backward(h, residual, gate, weight, bias, next_weight, next_bias, stats)
        return x if y is None else (x, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, gx, gy=None):
        *ins, stats = ctx.saved_tensors
        if gx is None and gy is None:
            return (None,) * 8
        h, residual = ins[0], ins[1]
        gx, gy = (None if g is None else g.contiguous() for g in (gx, gy))
        out = [torch.empty_like(t) if t is not None and need else None for t, need in zip(ins, ctx.needs_input_grad)]
        if h.shape[0] == 0:
            return tuple(None if o is None else o.zero_() for o in out) + (None,)
        if gy is None:                       # nothing reached the second norm
            for k in (5, 6):
                if out[k] is not None:
                    out[k].zero_()
        a = _args(*ins, ctx.conf)
        a.stats, a.gx, a.gy = lo.ptr(stats), lo.ptr(gx), lo.ptr(gy)
        a.dh, a.dresidual, a.dgate, a.dweight, a.dbias = map(lo.ptr, out[:5])
        a.dnext_weight, a.dnext_bias = (lo.ptr(out[k]) if gy is not None else None for k in (5, 6))
        size = _lib.load().nfi_resnorm_work_bytes(a.rows, a.groups, a.affine_groups, a.width)
        work = torch.empty((size,), device=h.device, dtype=torch.uint8)
        a.work = lo.ptr(work)
        with lo.on(h.device):
            lo.call('nfi_resnorm_backward', ctypes.byref(a), lo.stream(h.device))
        return tuple(out) + (None,)


def residual_norm(h: torch.Tensor, residual: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, norm: Optional[str] = 'layer',
                  slope: float = 1.0, scale: float = 1.0, next_weight: Optional[torch.Tensor] = None,
                  next_bias: Optional[torch.Tensor] = None, next_norm: Optional[str] = None, eps: float = 1e-5):
    """x, or (x, y) with `next_norm`, of h [..., D] (float32, bfloat16 or float16; D up to 8192):

        x = scale * (residual + gate * leaky_relu(norm(h) * weight + bias, slope)),  y = next_norm(x) * next_weight + next_bias

    `norm` and `next_norm`: 'layer', 'rms' or None.  residual: h's shape and type.  gate: [D], or [G, D] where G divides
    the number of rows and row r takes gate r // (rows / G) (an image's rows side by side: one gate for each image; G = rows:
    a gate for each row).  weight, bias, next_weight, next_bias: all [D], or all [G, D] with the gate's G (a conditional
    norm: each image's own), all of one type.  Statistics and sums are held in 32 bits and every output is rounded once; y is taken from x before its rounding.
    Gradients reach every tensor argument, in a fixed order of summation (no double backward)."""
    what = 'residual_norm'
    lo.same_device(what, h, residual=residual, gate=gate, weight=weight, bias=bias, next_weight=next_weight,
                   next_bias=next_bias)
    lo.type_code(h, what)
    if norm not in KINDS or next_norm not in KINDS:
        raise ValueError(f"{what}: norms are 'layer', 'rms' or None, not {norm!r}, {next_norm!r}")
    if h.dim() < 1 or not 1 <= h.shape[-1] <= MAX_WIDTH:
        raise ValueError(f'{what}: rows of 1 to {MAX_WIDTH} values are wanted, not {tuple(h.shape)}')
    d = h.shape[-1]
    if residual is not None and (residual.shape != h.shape or residual.dtype != h.dtype):
        raise ValueError(f'{what}: residual is {tuple(residual.shape)} {residual.dtype}, h {tuple(h.shape)} {h.dtype}')
    if next_norm is None and (next_weight is not None or next_bias is not None):
        raise ValueError(f'{what}: next_weight and next_bias need next_norm')
    rows = h.numel() // d
    first = None
    for name, t in (('weight', weight), ('bias', bias), ('next_weight', next_weight), ('next_bias', next_bias)):
        if t is None:
            continue
        lo.type_code(t, f'{what}: {name}')
        fits = t.shape == (d,) or (t.dim() == 2 and t.shape[1] == d and t.shape[0] >= 1 and rows % t.shape[0] == 0)
        if not fits or (first is not None and (t.dtype != first.dtype or t.shape != first.shape)):
            raise ValueError(f'{what}: {name} is {tuple(t.shape)} {t.dtype}; [{d}], or [G, {d}] with G a divisor of {rows} '
                             'rows is wanted, all of one shape and type')
        first = t
    if eps < 0:
        raise ValueError(f'{what}: eps {eps}')
    shape = h.shape
    affine = first is not None and first.dim() == 2
    if gate is not None:
        lo.type_code(gate, f'{what}: gate')
        if gate.dim() == 1:
            gate = gate[None]
        if gate.dim() != 2 or gate.shape[1] != d or gate.shape[0] < 1 or rows % gate.shape[0]:
            raise ValueError(f'{what}: gate is {tuple(gate.shape)}; [{d}] or [G, {d}] with G a divisor of {rows} rows is wanted')
        if affine and gate.shape[0] != first.shape[0]:
            if gate.shape[0] != 1:
                raise ValueError(f'{what}: {gate.shape[0]} gates and {first.shape[0]} groups of parameters')
            gate = gate.expand(first.shape[0], d)
        gate = gate.contiguous()
    conf = (KINDS[norm], KINDS[next_norm], float(slope), float(scale), float(eps))
    flat = [None if t is None else t.reshape(rows, d).contiguous() for t in (h, residual)]
    params = [None if t is None else t.contiguous() for t in (weight, bias, next_weight, next_bias)]
    out = _ResidualNorm.apply(*flat, gate, *params, conf)
    return tuple(o.view(shape) for o in out) if next_norm else out.view(shape)
