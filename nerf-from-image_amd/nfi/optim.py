"""Orthogonalised updates (include/nfi_learn.h): an update's singular values are brought near 1 by Newton-Schulz
products, so that every direction of a weight (or of an image's block of latents) moves by about the same length.

    orthogonalize(u)    the update alone, over any leading dimensions
    Muon                the optimiser: momentum, orthogonalised update, decoupled decay, one call for all matrices

Beside torch.optim.Adam in the inversion loop (nfi.inversion, InversionConfig.latent_update) and for the matrices of the
generator and its mapper heads (linear and convolution weights; a convolution's is taken as [out, in * kh * kw]).
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, Sequence

import torch

from . import _lib, learn_ops as lo

QUINTIC = (3.4445, -4.7750, 2.0315)
MAX_SIDE = 262144


def _launch(items, dev, g_type, w_type, update, nesterov, steps, momentum, step, decay, coefficients, eps):
    arr = (_lib.NfiOrthoItem * len(items))(*items)
    a = _lib.NfiOrthoArgs()
    a.items, a.n_items = arr, len(items)
    a.g_type, a.w_type, a.update, a.nesterov, a.steps = g_type, w_type, update, nesterov, steps
    a.momentum, a.step, a.decay, a.eps = momentum, step, decay, eps
    a.a, a.b, a.c = coefficients
    size = _lib.load().nfi_ortho_work_bytes(arr, len(items))
    work = None
    if size:
        work = torch.empty((size,), device=dev, dtype=torch.uint8)
        a.work, a.work_bytes = work.data_ptr(), size
    with lo.on(dev):
        lo.call('nfi_ortho', ctypes.byref(a), lo.stream(dev))


def _check(what, steps, coefficients, eps):
    if not 1 <= int(steps) <= 64:
        raise ValueError(f'{what}: 1 to 64 steps are wanted, not {steps}')
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f'{what}: three finite coefficients are wanted, not {coefficients!r}')
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f'{what}: eps {eps}')


def _check_sides(what, rows, cols, count):
    if not (1 <= rows <= MAX_SIDE and 1 <= cols <= MAX_SIDE):
        raise ValueError(f'{what}: sides of 1 to {MAX_SIDE} are wanted, not {rows} x {cols}')
    if 4 * (-(-rows // 128)) * (-(-cols // 128)) * count >= 1 << 26:
        raise ValueError(f'{what}: {count} matrices of {rows} x {cols} are too much for one call')


@torch.no_grad()
def orthogonalize(u: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = QUINTIC, eps: float = 1e-7) -> torch.Tensor:
    """u [..., m, n] (float32, bfloat16 or float16) with each matrix's singular values brought near 1: X = u / max(|u|_F,
    eps), then `steps` times X <- (a + b X X^T + c (X X^T)^2) X, (a, b, c) = `coefficients`.  Products are held to 32-bit
    accuracy whatever u's type; the result is rounded once.  Not differentiable."""
    what = 'orthogonalize'
    lo.same_device(what, u)
    code = lo.type_code(u, what)
    _check(what, steps, coefficients, eps)
    if u.dim() < 2:
        raise ValueError(f'{what}: matrices are wanted, not {tuple(u.shape)}')
    rows, cols = u.shape[-2:]
    src = u.contiguous()
    out = torch.empty_like(src)
    count = 1
    for n in u.shape[:-2]:
        count *= n
    if out.numel() == 0:
        return out
    _check_sides(what, rows, cols, count)
    item = _lib.NfiOrthoItem(src.data_ptr(), None, out.data_ptr(), rows, cols, count, 1.0)
    _launch([item], u.device, code, code, 0, 0, int(steps), 0.0, 0.0, 0.0, coefficients, eps)
    return out


class Muon(torch.optim.Optimizer):
    """For parameters of two or more dimensions, [rows, ...] taken as a matrix [rows, cols] (`batched`: [..., rows, cols]
    as one matrix for each leading index, as a batch of images' latents [b, 15, 512]):

        M <- momentum M + G;  U = G + momentum M (nesterov) or M;  O = orthogonalize(U)
        W <- W (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) O

    M (state 'momentum_buffer') is 32-bit for every type of parameter; gradients and parameters are float32, bfloat16 or
    float16, contiguous.  All matrices of a group of equal types go through one call; lr and the other numbers are read
    when step() is called (a captured graph keeps those of its capture)."""

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
                 steps: int = 5, coefficients: Sequence[float] = QUINTIC, eps: float = 1e-7, batched: bool = False):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f'Muon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}')
        _check('Muon', steps, coefficients, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, batched=batched))
        for group in self.param_groups:
            for p in group['params']:
                if p.dim() < 2:
                    raise ValueError(f'Muon: parameters of two or more dimensions are wanted, not {tuple(p.shape)} '
                                     '(biases and gains belong to another optimiser)')

    @staticmethod
    def _sides(p, batched):
        if batched:
            rows, cols = p.shape[-2:]
            return rows, cols, p.numel() // (rows * cols)
        return p.shape[0], p.numel() // p.shape[0], 1

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            lots = {}
            for p in group['params']:
                g = p.grad
                if g is None or p.numel() == 0:
                    continue
                if g.is_sparse or not p.is_contiguous():
                    raise RuntimeError('Muon: dense gradients and contiguous parameters are wanted')
                key = (p.device, p.dtype, g.dtype)
                lot = lots.get(key)
                if lot is None:
                    lo.same_device('Muon', p)
                    lot = lots[key] = (lo.type_code(g, 'Muon'), lo.type_code(p, 'Muon'), [], [], [])
                state = self.state[p]
                m = state.get('momentum_buffer')
                if m is None:
                    m = state['momentum_buffer'] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                if not g.is_contiguous():
                    g = g.contiguous()
                    lot[3].append(g)                # kept until the call is made
                rows, cols, count = self._sides(p, group['batched'])
                lot[2].append((g.data_ptr(), m.data_ptr(), p.data_ptr(), rows, cols, count, math.sqrt(max(1.0, rows / cols))))
                lot[4].extend((p, m))
            for (dev, _, _), (gt, wt, items, _, written) in lots.items():
                _launch(items, dev, gt, wt, 1, int(group['nesterov']), group['steps'], group['momentum'], group['lr'],
                        group['lr'] * group['weight_decay'], group['coefficients'], group['eps'])
                for t in written:                   # what is cached by a tensor's version is out of date
                    torch.autograd.graph.increment_version(t)
        return loss

    def load_state_dict(self, state_dict):
        """The momentum comes back in 32 bits (the base class would bring it to the parameter's type)."""
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict['param_groups'] for i in g['params']]
        params = [p for g in self.param_groups for p in g['params']]
        for p, i in zip(params, ids):
            m = state_dict['state'].get(i, {}).get('momentum_buffer')
            if m is not None:
                self.state[p]['momentum_buffer'] = m.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()
