"""Products grouped by ragged runs of rows (include/nfi_learn.h): the rows of a batch that mixes several heads,
each run of rows through its own head's weight.

    y[r] = weight[e] @ x[r] + bias[e]        offsets[e] <= r < offsets[e + 1]

The layer is stylegan.py:148-180's linear one (the caller scales the weight by its gain), for `groups` of them in one
launch; the offsets stay on the device.  Checks and autograd: csrc/nfi_torch_learn.cpp.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import torch_ops

MAX_GROUPS, MAX_WIDTH = 65535, 2097152
_op = None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None):
    """y [rows, N] of x [rows, K], weight [groups, N, K] and bias [groups, N] (or None), all float32, bfloat16 or
    float16 alike: row r of group e, offsets[e] <= r < offsets[e + 1], gives weight[e] @ x[r] + bias[e]; rows that no
    group holds give zeros.  offsets [groups + 1] int32 or int64 on the device, not decreasing (it is not read on the host:
    values outside [0, rows] count as the nearest end, and decreasing ones give wrong rows, never a wrong access).

    Sums are held in 32 bits and rounded once (32-bit values to 2^-24 of themselves, and 2^-133); what is not finite gives what such a sum gives, in its own rows and columns.  Gradients reach x, weight and bias, summed in a fixed order (no double
    backward); an empty group's weight and bias get zeros."""
    global _op
    if _op is None:
        _op = torch_ops.op('grouped_linear')
    return _op(x, weight, offsets, bias)
