"""The view-direction mapper of the reference's field (--use_viewdir; models/generator.py:189-252).

Its per-ray trunk — ViewDirectionMapper.forward up to `x` (generator.py:223-238): EqualizedLinear
3->64, two residual pairs of (EqualizedLinear 64->64 without bias, LayerNorm, LeakyReLU 0.2) scaled
by sqrt(2)/2, EqualizedLinear 64->64 + LeakyReLU, EqualizedLinear 64->32 — runs here on the
caller's module (the reference's own `Generator.viewdir_mapper`, or any module with the same
sub-module names), once per ray: B*H*W rows of a small MLP.  The per-sample part of its closure
(generator.py:242-250: output(leaky_relu(x + features))) runs inside the HIP render kernels
(NFI_HEAD_VIEWDIR), which also return dL/d x so autograd reaches the ray directions through
this trunk.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .grouped import grouped_linear
from .norms import residual_norm


def viewdir_trunk(mapper, viewdir: torch.Tensor) -> torch.Tensor:
    """generator.py:223-238 on `mapper`'s layers: viewdir [..., 1, 3] -> x [..., 1, 32]."""
    scale = math.sqrt(2) / 2
    relu = mapper.relu
    x = relu(mapper.fc0(viewdir))
    shortcut = x
    x = relu(mapper.norm1(mapper.fc1(x)))
    x = relu(mapper.norm2(mapper.fc2(x)))
    x = (x + shortcut).mul_(scale)
    shortcut = x
    x = relu(mapper.norm3(mapper.fc3(x)))
    x = relu(mapper.norm4(mapper.fc4(x)))
    x = (x + shortcut).mul_(scale)
    x = relu(mapper.fc5(x))
    x = mapper.fc6(x)
    assert x.shape[-2] == 1, x.shape
    return x


class ViewDirectionMapper(torch.nn.Module):
    """The reference module's structure and state_dict keys (generator.py:189-221): a reference
    checkpoint's `viewdir_mapper.*` entries load into it strictly.  Its trunk runs through
    viewdir_trunk; `output` is read by the renderer (ops.pack_viewdir_head)."""

    def __init__(self, output_size: int, num_features: int = 32):
        super().__init__()
        from .producer import EqualizedLinear
        h = 64
        self.hidden_size = h
        self.fc0 = EqualizedLinear(3, h)
        for i in range(1, 5):
            setattr(self, f'fc{i}', EqualizedLinear(h, h, bias=False))
            setattr(self, f'norm{i}', torch.nn.LayerNorm(h, elementwise_affine=True))
        self.fc5 = EqualizedLinear(h, h)
        self.fc6 = EqualizedLinear(h, num_features)
        self.output = EqualizedLinear(num_features, output_size)
        with torch.no_grad():
            self.output.weight.zero_()
            self.output.bias.zero_()
        self.relu = torch.nn.LeakyReLU(0.2)

    def forward(self, viewdir):
        return viewdir_trunk(self, viewdir)


class ViewDirectionMapperBank(torch.nn.Module):
    """Several mappers' trunks over one batch of rays: image b's rays go through mapper `mapper_of_image[b]` (a batch that
    mixes categories, each with a mapper of its own).  The layers are viewdir_trunk's, all mappers in each launch: grouped
    products (nfi.grouped) and one fused norm, activation and shortcut for each (nfi.norms), the norms' weights taken image
    by image.  Gradients reach the mappers' own parameters and viewdir.  The mappers are alike but for their parameters' values:
    others are refused."""

    def __init__(self, mappers):
        super().__init__()
        self.mappers = torch.nn.ModuleList(mappers)
        if len(self.mappers) == 0:
            raise ValueError('ViewDirectionMapperBank: no mappers')
        self.register_buffer('ends', torch.arange(len(self.mappers) + 1, device=self.mappers[0].fc0.weight.device), persistent=False)
        first = self._form(self.mappers[0])
        for i, m in enumerate(self.mappers):
            if self._form(m) != first:
                a, b = next((x, y) for x, y in zip(self._form(m), first) if x != y)
                raise ValueError(f'ViewDirectionMapperBank: mapper {i} differs from the first, {a} from {b}')

    @staticmethod
    def _form(mapper):
        """What all mappers of a bank share: shapes, gains, and the norms' and the activation's constants."""
        form = [('relu', type(mapper.relu).__name__, getattr(mapper.relu, 'negative_slope', None))]
        for name in (f'fc{i}' for i in range(7)):
            m = getattr(mapper, name)
            form.append((name, tuple(m.weight.shape), m.weight_gain, None if m.bias is None else m.bias_gain))
        for name in (f'norm{i}' for i in range(1, 5)):
            m = getattr(mapper, name)
            if m.weight is None or m.bias is None:
                raise ValueError(f'ViewDirectionMapperBank: {name} has no weight or no bias')
            form.append((name, tuple(m.weight.shape), m.eps))
        if form[0] != ('relu', 'LeakyReLU', 0.2):
            raise ValueError(f'ViewDirectionMapperBank: LeakyReLU(0.2) is wanted, not {mapper.relu}')
        return form

    def _linear(self, name, x, offsets):
        layers = [getattr(m, name) for m in self.mappers]
        w = torch.stack([m.weight for m in layers]) * layers[0].weight_gain
        b = None if layers[0].bias is None else torch.stack([m.bias for m in layers]) * layers[0].bias_gain
        return grouped_linear(x, w, offsets, b)

    def _norm(self, name, h, image, shortcut=None):
        layers = [getattr(m, name) for m in self.mappers]
        w, b = torch.stack([getattr(n, k) for k in ('weight', 'bias') for n in layers]).view(2, len(layers), -1)[:, image].unbind()
        return residual_norm(h, shortcut, None, w, b, slope=0.2, scale=1.0 if shortcut is None else math.sqrt(2) / 2,
                             eps=layers[0].eps)

    def forward(self, viewdir: torch.Tensor, mapper_of_image: torch.Tensor) -> torch.Tensor:
        """viewdir [images, rays, 3], mapper_of_image [images] int64 on the device, in any order -> [images, rays, 32]; zeros,
        and no gradients, for an image whose number is none of a mapper (it is not read on the host)."""
        images, rays = viewdir.shape[:2]
        if mapper_of_image.shape != (images,) or mapper_of_image.dtype != torch.int64:
            raise ValueError(f'mapper_of_image [{images}] int64 is wanted, not {tuple(mapper_of_image.shape)} {mapper_of_image.dtype}')
        if images * rays == 0:   # (an empty result with its graph: rows of groups are at least one)
            return viewdir_trunk(self.mappers[0], viewdir.unsqueeze(-2)).squeeze(-2)
        # the products want a mapper's rows side by side: the images are brought into their mappers' order, and back
        image, order = torch.sort(mapper_of_image, stable=True)
        offsets = torch.searchsorted(image, self.ends.to(image.device)) * rays
        image = image.clamp(0, len(self.mappers) - 1)   # (the products leave such images' rows out)
        x = F.leaky_relu(self._linear('fc0', viewdir.index_select(0, order).reshape(images * rays, 3), offsets), 0.2)
        for a, b in ((1, 2), (3, 4)):
            h = self._norm(f'norm{a}', self._linear(f'fc{a}', x, offsets), image)
            x = self._norm(f'norm{b}', self._linear(f'fc{b}', h, offsets), image, shortcut=x)
        x = F.leaky_relu(self._linear('fc5', x, offsets), 0.2)
        x = self._linear('fc6', x, offsets).view(images, rays, -1)
        return torch.empty_like(x).index_copy_(0, order, x)
