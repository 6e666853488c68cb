"""nfi.norms.residual_norm on the device against the formula in 64 bits: every type, widths that fill a piece,
end inside one or are smaller than one, rows held by part of a wave, a wave and a workgroup, gates of every
kind, absent parameters, and the gradients (against the formula's by autograd in 64 bits, and differences).

Tolerances.  u = 2^-24 (32-bit rounding), e = eps(type) / 2 (the one rounding of an output).  A value is a
handful of 32-bit operations on statistics whose sums have chains of at most 16 serial terms and 9 joining
steps: 64 u of the largest magnitude that enters it is allowed for, beside e of itself.  A sum over rows
adds a chain of at most rows / 1 + 64 + 16 terms: that many u of the sum of its terms' magnitudes."""

import math

import pytest
import torch

from nfi import norms

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
U = 2.0 ** -24
NAMES = ('h', 'residual', 'gate', 'weight', 'bias', 'next_weight', 'next_bias')


def normed(v, kind, eps):
    if kind is None:
        return v
    if kind == 'layer':
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)


def formula(p, norm, next_norm, slope, scale, eps=1e-5):
    """(x, y or None, the largest magnitudes that enter x and y) in the inputs' type."""
    n = normed(p['h'], norm, eps)
    u = n if p['weight'] is None else n * p['weight']
    u = u if p['bias'] is None else u + p['bias']
    v = torch.where(u > 0, u, u * slope)
    if p['gate'] is not None:
        rows = p['h'].shape[0]
        v = v * p['gate'].repeat_interleave(rows // p['gate'].shape[0], 0)
    x = scale * (v if p['residual'] is None else v + p['residual'])
    if next_norm is None:
        return x, None
    m = normed(x, next_norm, eps)
    y = m if p['next_weight'] is None else m * p['next_weight']
    return x, (y if p['next_bias'] is None else y + p['next_bias'])


def inputs(rows, width, dtype, seed, residual=True, gates=0, affine=True, next_affine=True, param=None):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape, dt=dtype, scale=1.0, shift=0.0):
        return (torch.randn(shape, device=DEV, generator=g) * scale + shift).to(dt)

    param = param or dtype
    return {'h': rnd(rows, width, scale=1.5, shift=0.3), 'residual': rnd(rows, width) if residual else None,
            'gate': rnd(gates, width, dt=param, scale=0.5) if gates else None,
            'weight': rnd(width, dt=param, scale=0.1, shift=1) if affine else None,
            'bias': rnd(width, dt=param, scale=0.1) if affine else None,
            'next_weight': rnd(width, dt=param, scale=0.1, shift=1) if next_affine else None,
            'next_bias': rnd(width, dt=param, scale=0.1) if next_affine else None}


def run(p, norm, next_norm, slope, scale):
    q = dict(p)
    if next_norm is None:
        q['next_weight'] = q['next_bias'] = None
    out = norms.residual_norm(q['h'], q['residual'], q['gate'], q['weight'], q['bias'], norm=norm, slope=slope, scale=scale,
                              next_weight=q['next_weight'], next_bias=q['next_bias'], next_norm=next_norm)
    return out if next_norm else (out, None)


def near(got, ref, dtype, terms, chain=64):
    """|got - ref| <= e |ref| + chain u terms, at every place; terms: magnitudes that enter (broadcast)."""
    e = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    err = (got.double() - ref).abs()
    tol = e * ref.abs() * (1 + 2 ** -8) + chain * U * terms + torch.finfo(dtype).smallest_normal
    worst = float((err / tol).max()) if err.numel() else 0.0
    assert worst <= 1, (tuple(got.shape), worst)


CASES = [  # rows, width, residual, gates, norm, next_norm, slope, affine
    (37, 64, True, 0, 'layer', None, 0.2, True),
    (1, 1, True, 0, 'rms', 'rms', 1.0, True),
    (5, 3, True, 5, 'layer', 'layer', 0.2, True),
    (64, 7, False, 2, 'rms', None, 1.0, True),
    (130, 8, True, 1, 'layer', 'rms', 0.2, False),
    (33, 65, True, 3, 'layer', 'layer', 0.2, True),
    (48, 100, True, 4, 'rms', 'layer', 1.0, True),
    (9, 250, False, 9, None, 'layer', 0.2, True),
    (20, 512, True, 5, 'layer', 'layer', 0.2, True),
    (7, 513, True, 1, 'rms', 'rms', 1.0, True),
    (6, 1001, True, 2, 'layer', 'layer', 0.2, True),
    (5, 1024, True, 5, 'rms', 'rms', 1.0, True),
    (4, 2048, True, 2, 'layer', 'rms', 0.2, True),
    (3, 2999, True, 3, 'layer', 'layer', 1.0, False),
    (4, 4096, False, 0, 'rms', 'layer', 1.0, True),
    (2, 8192, True, 1, 'layer', 'layer', 0.2, True),
    (3, 8191, True, 3, 'layer', 'rms', 0.2, True),
    (3000, 64, True, 1500, 'layer', 'layer', 0.2, True),
    (4097, 128, True, 17, 'rms', None, 1.0, True),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{c[0]}x{c[1]}')
def test_values_and_gradients(case, dtype):
    rows, width, residual, gates, norm, next_norm, slope, affine = case
    p = inputs(rows, width, dtype, rows * 31 + width, residual, gates, affine, affine and next_norm is not None)
    scale = math.sqrt(0.5)
    p = {k: None if v is None else v.requires_grad_() for k, v in p.items()}
    p64 = {k: None if v is None else v.detach().double().requires_grad_() for k, v in p.items()}
    x, y = run(p, norm, next_norm, slope, scale)
    rx, ry = formula(p64, norm, next_norm, slope, scale)
    big = 4 + float(rx.detach().abs().max())
    near(x.detach(), rx.detach(), dtype, big)
    g = torch.Generator(device=DEV).manual_seed(5)
    outs, gs = [x], [torch.randn((rows, width), device=DEV, generator=g).to(dtype)]
    routs = [rx]
    if next_norm:
        # (the second norm divides x's own 32-bit error by its deviation)
        gain = float((1 / torch.sqrt(rx.detach().var(-1, unbiased=False) + 1e-5)).max()) if next_norm == 'layer' else \
            float((1 / torch.sqrt(rx.detach().square().mean(-1) + 1e-5)).max())
        near(y.detach(), ry.detach(), dtype, big * max(1.0, gain) * 4)
        outs.append(y)
        routs.append(ry)
        gs.append(torch.randn((rows, width), device=DEV, generator=g).to(dtype))
    leaves = [v for v in p.values() if v is not None]
    got = torch.autograd.grad(outs, leaves, gs)
    ref = torch.autograd.grad(routs, [v for v in p64.values() if v is not None], [v.double() for v in gs])
    names = [k for k in NAMES if p[k] is not None]
    e = torch.finfo(dtype).eps / 2
    for name, a, b in zip(names, got, ref):
        assert a.dtype == dtype and a.shape == p[name].shape
        # by norm: one rounding, and 32-bit sums whose terms are gradients of the gradients' own size; rows with a
        # small deviation amplify both
        dev = normed(p64['h'].detach(), norm, 1e-5)
        amp = 1.0
        if norm is not None and width > 1:
            amp = max(1.0, float((dev.abs().amax(-1) / p64['h'].detach().abs().amax(-1).clamp_min(1e-30)).max()))
        if next_norm is not None:
            amp *= max(1.0, gain)
        total = float(torch.cat([r.flatten() for r in ref]).norm()) if width < 8 else float(b.norm())
        err = float((a.double() - b).norm())
        assert err <= e * float(b.norm()) * (dtype != torch.float32) + (64 + rows / 16) * U * amp * max(total, float(b.norm())) + 1e-30, (name, err, float(b.norm()))


MANY = [  # more rows than workgroups, so that each takes several; no kink, whose side the last bit decides
    (1700, 320, True, 17, 'layer', 'layer', 1.0, True),
    (1600, 520, True, 1600, 'rms', 'layer', 1.0, True),
    (2100, 1000, True, 7, 'layer', 'rms', 1.0, True),
    (1601, 1024, True, 1, 'rms', 'rms', 1.0, True),
    (1500, 1024, False, 750, 'layer', None, 1.0, True),
    (1100, 2000, True, 2, 'layer', 'layer', 1.0, True),
    (600, 4096, True, 4, 'rms', 'rms', 1.0, True),
    (555, 4100, True, 5, 'layer', 'layer', 1.0, True),
    (530, 8192, True, 1, 'rms', 'layer', 1.0, True),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('case', MANY, ids=lambda c: f'{c[0]}x{c[1]}')
def test_many_rows_of_a_workgroup(case, dtype):
    test_values_and_gradients(case, dtype)


def test_gradient_against_differences():
    """Central differences of the 32-bit outputs' scalar product: step 2^-6, truncation ~ step^2, rounding ~ u / step."""
    p = inputs(6, 40, torch.float32, 3, True, 3)
    p = {k: v.requires_grad_() for k, v in p.items()}
    g = torch.Generator(device=DEV).manual_seed(1)
    gx, gy = (torch.randn((6, 40), device=DEV, generator=g) for _ in range(2))

    def value(q):
        x, y = run(q, 'layer', 'layer', 1.0, 0.7)
        return (x.double() * gx.double()).sum() + (y.double() * gy.double()).sum()

    grads = torch.autograd.grad(value(p), list(p.values()))
    for (name, v), d in zip(p.items(), grads):
        way = torch.randn(v.shape, device=DEV, generator=g)
        step = 2.0 ** -6
        hi, lo = (float(value({**p, name: (v + s * way).detach()}).detach()) for s in (step, -step))
        want = float((d.double() * way.double()).sum())
        scale = float(d.norm() * way.norm()) + 1
        assert abs((hi - lo) / (2 * step) - want) <= 30 * step ** 2 * scale, (name, (hi - lo) / (2 * step), want)


def test_mixed_parameter_types_and_broadcast_gate():
    """32-bit parameters and gate beside bf16 rows; a [D] gate is every row's."""
    p = inputs(50, 96, torch.bfloat16, 9, True, 1, param=torch.float32)
    q = {k: v.requires_grad_() for k, v in p.items()}
    q64 = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    x, y = norms.residual_norm(q['h'], q['residual'], q['gate'][0], q['weight'], q['bias'], next_weight=q['next_weight'],
                               next_bias=q['next_bias'], next_norm='rms')
    rx, ry = formula(q64, 'layer', 'rms', 1.0, 1.0)
    near(x.detach(), rx.detach(), torch.bfloat16, 12)
    near(y.detach(), ry.detach(), torch.bfloat16, 24)
    got = torch.autograd.grad([x, y], list(q.values()), [torch.ones_like(x), torch.ones_like(y)])
    ref = torch.autograd.grad([rx, ry], list(q64.values()), [torch.ones_like(rx), torch.ones_like(ry)])
    for name, a, b in zip(NAMES, got, ref):
        e = torch.finfo(a.dtype).eps / 2
        # (ones under a layer norm cancel: the sums' own magnitude is that of the terms, sqrt(rows) at most of the norm)
        assert float((a.double() - b).norm()) <= e * float(b.norm()) + 128 * U * 50 * (1 + float(b.norm())), name


@pytest.mark.parametrize('rows,groups,width,gate', [(4, 4, 512, True), (12, 3, 40, False), (600, 2, 64, True), (1, 1, 9, True),
                                                    (2048, 1024, 72, True), (4096, 4, 130, False)])
def test_parameters_of_groups(rows, groups, width, gate):
    """Each group of rows with its own weight, bias and next norm (a conditional norm), some gradients left out."""
    g = torch.Generator(device=DEV).manual_seed(rows)

    def rnd(*shape, shift=0.0):
        return (torch.randn(shape, device=DEV, generator=g) * 0.3 + shift).requires_grad_()
    p = {'h': rnd(rows, width), 'residual': rnd(rows, width), 'gate': rnd(groups, width, shift=1) if gate else None,
         'weight': rnd(groups, width, shift=1), 'bias': rnd(groups, width), 'next_weight': rnd(groups, width, shift=1),
         'next_bias': rnd(groups, width)}
    p64 = {k: None if v is None else v.detach().double().requires_grad_() for k, v in p.items()}
    spread = {k: (v if v is None or k in ('h', 'residual', 'gate') else v.repeat_interleave(rows // groups, 0)) for k, v in p64.items()}
    x, y = run(p, 'layer', 'rms', 1.0, 0.7)
    rx, ry = formula(spread, 'layer', 'rms', 1.0, 0.7)
    near(x.detach(), rx.detach(), torch.float32, 8)
    near(y.detach(), ry.detach(), torch.float32, 32)
    gx, gy = torch.randn((rows, width), device=DEV, generator=g), torch.randn((rows, width), device=DEV, generator=g)
    keys = [k for k in NAMES if p[k] is not None]
    got = torch.autograd.grad([x, y], [p[k] for k in keys], [gx, gy], retain_graph=True)
    ref = torch.autograd.grad([rx, ry], [p64[k] for k in keys], [gx.double(), gy.double()])
    for k, a, b in zip(keys, got, ref):
        assert float((a.double() - b).norm()) <= (64 + rows / 16) * U * 16 * float(b.norm()), k
    some = torch.autograd.grad([x, y], [p['bias'], p['next_weight']], [gx, gy])
    assert torch.equal(some[0], got[keys.index('bias')]) and torch.equal(some[1], got[keys.index('next_weight')])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,groups,width', [(1600, 800, 1000), (800, 2, 1024), (6, 3, 4096), (260, 260, 5000), (520, 4, 8192), (1600, 4, 320)])
def test_parameters_of_groups_of_wide_rows(rows, groups, width, dtype):
    """The same where a row takes a workgroup, beside 16-bit rows too (the parameters 32-bit, their gradients unrounded)."""
    g = torch.Generator(device=DEV).manual_seed(rows + width)

    def rnd(*shape, shift=0.0, dt=torch.float32):
        return (torch.randn(shape, device=DEV, generator=g) * 0.3 + shift).to(dt).requires_grad_()
    p = {'h': rnd(rows, width, dt=dtype), 'residual': rnd(rows, width, dt=dtype), 'gate': rnd(groups, width, shift=1),
         'weight': rnd(groups, width, shift=1), 'bias': rnd(groups, width), 'next_weight': rnd(groups, width, shift=1),
         'next_bias': rnd(groups, width)}
    p64 = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    spread = {k: (v if k in ('h', 'residual', 'gate') else v.repeat_interleave(rows // groups, 0)) for k, v in p64.items()}
    x, y = run(p, 'layer', 'rms', 1.0, 0.7)
    rx, ry = formula(spread, 'layer', 'rms', 1.0, 0.7)
    near(x.detach(), rx.detach(), dtype, 8)
    near(y.detach(), ry.detach(), dtype, 32)
    gx, gy = (torch.randn((rows, width), device=DEV, generator=g).to(dtype) for _ in range(2))
    got = torch.autograd.grad([x, y], list(p.values()), [gx, gy])
    ref = torch.autograd.grad([rx, ry], list(p64.values()), [gx.double(), gy.double()])
    for k, a, b in zip(p, got, ref):
        e = torch.finfo(a.dtype).eps / 2 if a.dtype != torch.float32 else 0.0
        assert float((a.double() - b).norm()) <= (e + (64 + rows / 16) * U * 16) * float(b.norm()), k


def test_refusals():
    h = torch.zeros((6, 8), device=DEV)
    w = torch.ones((8,), device=DEV)
    for kw, word in ((dict(norm='batch'), 'norms are'), (dict(residual=h[:3]), 'residual'), (dict(residual=h.half()), 'residual'),
                     (dict(weight=w[:7]), 'weight'), (dict(weight=w, bias=w.half()), 'bias'), (dict(next_weight=w), 'next_norm'),
                     (dict(gate=torch.ones((4, 8), device=DEV)), 'gate'), (dict(weight=torch.ones((4, 8), device=DEV)), 'weight'),
                     (dict(weight=torch.ones((2, 8), device=DEV), gate=torch.ones((3, 8), device=DEV)), 'gates'),
                     (dict(eps=-1.0), 'eps'), (dict(weight=w.double()), 'float32'), (dict(weight=w.cpu()), 'cpu')):
        with pytest.raises((RuntimeError, ValueError), match=word):
            norms.residual_norm(h, **kw)
    with pytest.raises(RuntimeError, match='float32'):
        norms.residual_norm(h.double())
    with pytest.raises(ValueError, match='rows of 1'):
        norms.residual_norm(torch.zeros((1, 8193), device=DEV))


def test_partial_gradients_and_one_output():
    """A gradient for one output, or for one argument, gives what the whole gives in that place."""
    p = {k: v.requires_grad_() for k, v in inputs(24, 72, torch.float32, 4, True, 4).items()}
    x, y = run(p, 'layer', 'layer', 0.2, 0.5)
    only_x = torch.autograd.grad(x.sum(), [p['h'], p['gate'], p['next_weight']], retain_graph=True, allow_unused=True)
    p64 = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    rx, ry = formula(p64, 'layer', 'layer', 0.2, 0.5)
    ref = torch.autograd.grad(rx.sum(), [p64['h'], p64['gate']], retain_graph=True)
    for a, b in zip(only_x, ref):
        assert float((a.double() - b).abs().max()) <= 512 * U * (1 + float(b.abs().max()))
    assert only_x[2] is None or float(only_x[2].abs().max()) == 0
    gw, = torch.autograd.grad(y.sum(), [p['weight']])
    rw, = torch.autograd.grad(ry.sum(), [p64['weight']])
    assert float((gw.double() - rw).abs().max()) <= 512 * U * (1 + float(rw.abs().max())) * 24


def test_strided_views_streams_and_empty():
    p = inputs(32, 64, torch.float32, 6)
    base = torch.randn((32, 2, 64), device=DEV)
    view = base[:, 1]                                     # rows of stride 128
    x, _ = run({**p, 'h': view}, 'layer', None, 1.0, 1.0)
    ref, _ = formula({k: None if v is None else v.double() for k, v in {**p, 'h': view}.items()}, 'layer', None, 1.0, 1.0)
    near(x, ref, torch.float32, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x2, _ = run({**p, 'h': view}, 'layer', None, 1.0, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(x, x2)
    h = torch.empty((0, 16), device=DEV, requires_grad=True)
    w = torch.ones((16,), device=DEV, requires_grad=True)
    out = norms.residual_norm(h, weight=w)
    gh, gw = torch.autograd.grad(out.sum(), [h, w])
    assert out.shape == (0, 16) and gh.shape == (0, 16) and float(gw.abs().sum()) == 0


def test_rows_do_not_reach_each_other():
    """NaN and infinity in one row leave the others' values and gradients as they were."""
    p = inputs(16, 100, torch.float32, 8)
    bad = p['h'].clone()
    bad[5, 3], bad[9, 0] = math.nan, math.inf
    a, ya = run(p, 'layer', 'layer', 0.2, 1.0)
    b, yb = run({**p, 'h': bad}, 'layer', 'layer', 0.2, 1.0)
    rest = [i for i in range(16) if i not in (5, 9)]
    assert torch.equal(a[rest], b[rest]) and torch.equal(ya[rest], yb[rest])
    assert bool(torch.isnan(b[5]).all()) and bool(torch.isnan(b[9]).any())


def test_captured_and_replayed():
    """Forward and backward in one captured graph, replayed with new inputs between eager calls."""
    p = {k: v.requires_grad_() for k, v in inputs(200, 64, torch.float32, 2, True, 4).items()}
    leaves = list(p.values())
    gx, gy = torch.randn((200, 64), device=DEV), torch.randn((200, 64), device=DEV)

    def step():
        x, y = run(p, 'layer', 'layer', 0.2, 0.7)
        return [x.detach(), y.detach()] + list(torch.autograd.grad([x, y], leaves, [gx, gy]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            p['h'].copy_(torch.randn((200, 64), device=DEV) + k)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_one_gate_beside_groups_of_parameters(dtype):
    """A [D] or [1, D] gate for rows whose norms have parameters of groups: its gradient is summed over all of them in 32 bits
    and rounded once, where gradients of opposite signs cancel too."""
    g = torch.Generator(device=DEV).manual_seed(12)
    rows, groups, width = 512, 64, 40

    def rnd(*shape, shift=0.0, scale=0.5):
        return (torch.randn(shape, device=DEV, generator=g) * scale + shift).to(dtype)
    h, gate, weight, bias = rnd(rows, width), rnd(width, shift=1).requires_grad_(), rnd(groups, width, scale=0.1), rnd(groups, width, shift=2)
    gx = rnd(rows, width, shift=1, scale=0.1)
    gx[rows // groups * (groups // 2):] *= -1      # (half of the groups against the other half)
    p64 = {'h': h.double(), 'residual': None, 'gate': gate.detach().double().expand(groups, width),
           'weight': weight.double().repeat_interleave(rows // groups, 0), 'bias': bias.double().repeat_interleave(rows // groups, 0),
           'next_weight': None, 'next_bias': None}
    v, _ = formula({**p64, 'gate': None}, 'layer', None, 0.2, 1.0)
    rx, _ = formula(p64, 'layer', None, 0.2, 1.0)
    terms = gx.double() * v
    e = torch.finfo(dtype).eps / 2
    # each v is off by 64 u of the largest value that enters it (below 8), and sums of rows / groups, 16 and groups terms follow
    tol = 64 * U * 8 * gx.double().abs().sum(0) + (rows // groups + 16 + groups) * U * terms.abs().sum(0) + e * (1 + 2 ** -8) * terms.sum(0).abs()
    for shape in ((width,), (1, width)):
        x = norms.residual_norm(h, None, gate.view(shape), weight, bias, slope=0.2)
        near(x.detach(), rx, dtype, 8)
        got, = torch.autograd.grad(x, [gate], gx)
        assert float(((got.double() - terms.sum(0)).abs() / tol).max()) <= 1
