"""Orthogonalised updates (include/nfi_learn.h): an update's singular values are brought near 1 by Newton-Schulz
products, so that every direction of a weight (or of an image's block of latents) moves by about the same length.

    orthogonalize(u)    the update alone, over any leading dimensions
    Muon                the optimiser: momentum, orthogonalised update, decoupled decay, one call for all matrices

Beside torch.optim.Adam in the inversion loop (nfi.inversion, InversionConfig.latent_update) and for the matrices of the
generator and its mapper heads (linear and convolution weights; a convolution's is taken as [out, in * kh * kw]).
"""

from __future__ import annotations

import math
from typing import Iterable, Sequence

import torch

from . import torch_ops

QUINTIC = (3.4445, -4.7750, 2.0315)
_ops: dict = {}


def _op(name):
    op = _ops.get(name)
    if op is None:
        op = _ops[name] = torch_ops.op(name)
    return op


def _capturing():
    return torch.cuda.device_count() > 0 and torch.cuda.is_current_stream_capturing()


def _check(what, steps, coefficients, eps):
    if not 1 <= int(steps) <= 64:
        raise ValueError(f'{what}: 1 to 64 steps are wanted, not {steps}')
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f'{what}: three finite coefficients are wanted, not {coefficients!r}')
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f'{what}: eps {eps}')


@torch.no_grad()
def orthogonalize(u: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = QUINTIC, eps: float = 1e-7) -> torch.Tensor:
    """u [..., m, n] (float32, bfloat16 or float16) with each matrix's singular values brought near 1: X = u / max(|u|_F,
    eps), then `steps` times X <- (a + b X X^T + c (X X^T)^2) X, (a, b, c) = `coefficients`.  Products keep 22 bits or
    more of their operands whatever u's type (fewer of values below 2^-17: |u|_F far below eps), sums 32; the result is rounded
    once.  Not differentiable."""
    _check('orthogonalize', steps, coefficients, eps)
    return _op('orthogonalize')(u, int(steps), *coefficients, eps)


class Muon(torch.optim.Optimizer):
    """For parameters of two or more dimensions, [rows, ...] taken as a matrix [rows, cols] (`batched`: [..., rows, cols]
    as one matrix for each leading index, as a batch of images' latents [b, 15, 512]):

        M <- momentum M + G;  U = G + momentum M (nesterov) or M;  O = orthogonalize(U)
        W <- W (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) O

    M (state 'momentum_buffer') is 32-bit for every type of parameter; gradients and parameters are float32, bfloat16 or
    float16, contiguous.  All matrices of a group of equal types go through one call; lr and the other numbers are read
    when step() is called (a captured graph keeps those of its capture).  The first step of a parameter makes its momentum, and
    is refused in a capture, where every replay would make it anew: take one step before."""

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
                 steps: int = 5, coefficients: Sequence[float] = QUINTIC, eps: float = 1e-7, batched: bool = False):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f'Muon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}')
        _check('Muon', steps, coefficients, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, batched=batched))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        params = self.param_groups[-1]['params']
        bad = next((p for p in params if p.dim() < 2), None)
        twice = len({id(p) for p in params}) < len(params)
        if bad is None and not twice:
            return
        self.param_groups.pop()
        if bad is not None:
            raise ValueError(f'Muon: parameters of two or more dimensions are wanted, not {tuple(bad.shape)} '
                             '(biases and gains belong to another optimiser)')
        raise ValueError('Muon: a parameter twice in a group (all steps of a group are taken at a time)')

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = []
        for group in self.param_groups:
            params, grads, momenta = [], [], []
            for p in group['params']:
                g = p.grad
                if g is None or p.numel() == 0:
                    continue
                state = self.state[p]
                m = state.get('momentum_buffer')
                if m is None:
                    if _capturing():
                        raise RuntimeError('Muon: the first step of a parameter makes its momentum, and in a graph every replay would '
                                           'clear it again: take one step before the capture')
                    m = state['momentum_buffer'] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                params.append(p)
                grads.append(g)
                momenta.append(m)
            if params:
                calls.append((group, params, grads, momenta))
        op = _op('muon_step')
        for group, params, grads, momenta in calls:
            op(params, grads, momenta, group['batched'], group['lr'], group['momentum'], group['weight_decay'], group['nesterov'],
               group['steps'], *group['coefficients'], group['eps'])
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
