"""The norm of a block's output fused with what a residual trunk does around it (include/nfi_learn.h):

    x = scale * (residual + gate * leaky_relu(norm(h) * weight + bias, slope))
    y = next_norm(x) * next_weight + next_bias

One pass over memory each way.  The mapper trunks of the reference (generator.py:132-253) are made of it:
LayerNorm, LeakyReLU(0.2), shortcut, sqrt(2) / 2; the gate is a width's, an image's or a row's own factor, and
the next block's norm reads the new residual before it is rounded.  Checks and autograd: csrc/nfi_torch_learn.cpp.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import torch_ops

KINDS = {None: 0, 'layer': 1, 'rms': 2}
MAX_WIDTH = 8192
_op = None


def residual_norm(h: torch.Tensor, residual: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, norm: Optional[str] = 'layer',
                  slope: float = 1.0, scale: float = 1.0, next_weight: Optional[torch.Tensor] = None,
                  next_bias: Optional[torch.Tensor] = None, next_norm: Optional[str] = None, eps: float = 1e-5):
    """x, or (x, y) with `next_norm`, of h [..., D] (float32, bfloat16 or float16; D up to 8192):

        x = scale * (residual + gate * leaky_relu(norm(h) * weight + bias, slope)),  y = next_norm(x) * next_weight + next_bias

    `norm` and `next_norm`: 'layer', 'rms' or None.  residual: h's shape and type.  gate: [D], or [G, D] where G divides
    the number of rows and row r takes gate r // (rows / G) (an image's rows side by side: one gate for each image; G = rows:
    a gate for each row).  weight, bias, next_weight, next_bias: all [D], or all [G, D] with the gate's G (a conditional
    norm: each image's own), all of one type.  Statistics and sums are held in 32 bits and every output is rounded once; y
    is taken from x before its rounding.  Gradients reach every tensor argument, in a fixed order of summation (no double
    backward)."""
    global _op
    if _op is None:
        _op = torch_ops.op('residual_norm')
    try:
        kinds = KINDS[norm], KINDS[next_norm]
    except KeyError:
        raise ValueError(f"residual_norm: norms are 'layer', 'rms' or None, not {norm!r}, {next_norm!r}") from None
    out = _op(h, residual, gate, weight, bias, next_weight, next_bias, *kinds, slope, scale, eps)
    return tuple(out) if kinds[1] else out[0]
