"""nfi.optim on the device against the formula in 64 bits: matrices of every shape and both kernels (whole in a workgroup,
128 x 128 tiles), types, momentum, decay, empty and degenerate matrices, capture.

Tolerance.  One step X -> a X + (b A + c A^2) X is a function of X whose derivative is at most L = 4 for singular values
up to 1.2 (the quintic's own is 3.4 at 0 and below 4 at 1.2).  Every product is held to 8 x 2^-22 of its factors' norms
(a pair of halves keeps 2^-22 of a value, the dropped product is of the same size, sums add 2^-24 for each of their
steps of 32), so k steps are off by at most (1 + L + ... + L^(k-1)) 8 x 2^-22 |X|_F = 341 x 8 x 2^-22 |X|_F after five.  That is
the worst case; beside it the error has to be at most 4 times that of the same formula in torch's 32-bit products, plus 2^-21."""

import copy
import math

import pytest
import torch

from nfi import optim
from nfi.producer import EqualizedLinear

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def formula(u, steps=5, abc=optim.QUINTIC, eps=1e-7):
    a, b, c = abc
    turned = u.shape[-2] > u.shape[-1]
    x = u.transpose(-2, -1) if turned else u
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    for _ in range(steps):
        g = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.transpose(-2, -1) if turned else x


def near(got, u, dtype, steps=5, abc=optim.QUINTIC):
    ref = formula(u.double(), steps, abc)
    plain = formula(u.float(), steps, abc)
    size = float(ref.norm())
    e = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    err = float((got.double() - ref).norm())
    own = float((plain.double() - ref).norm())
    assert err <= e * size + 341 * 8 * 2.0 ** -22 * max(size, 1.0), (tuple(u.shape), err, size)
    if dtype == torch.float32:
        assert err <= 4 * own + 2.0 ** -21 * max(size, 1e-30), (tuple(u.shape), err, own, size)


SHAPES = [(1, 1), (1, 7), (9, 1), (3, 3), (2, 15, 512), (16, 16), (17, 40), (40, 17), (3, 33, 33), (64, 64), (64, 448), (448, 64), (64, 449), (64, 384), (384, 60), (50, 390), (48, 500), (20, 900), (31, 33), (16, 1900), (15, 2049), (4, 128), (130, 16), (2048, 9),
          (65, 70), (33, 1100), (128, 128), (129, 257), (300, 200), (2, 3, 96, 512), (513, 700), (11, 64), (5, 3000), (1, 70000),
          (640, 1300)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', SHAPES, ids=lambda s: 'x'.join(map(str, s)))
def test_orthogonalize(shape, dtype):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    u = (torch.randn(shape, device=DEV, generator=g) * torch.exp2(-2 * torch.rand(shape[-1], device=DEV, generator=g))).to(dtype)
    out = optim.orthogonalize(u)
    assert out.shape == u.shape and out.dtype == dtype
    near(out, u, dtype)
    assert torch.equal(out, optim.orthogonalize(u))      # the same bits again


@pytest.mark.parametrize('steps,abc', [(1, optim.QUINTIC), (3, optim.QUINTIC), (12, (1.5, -0.5, 0.0)), (5, (2.0, -1.5, 0.5)), (10, (1.875, -1.25, 0.375))])
@pytest.mark.parametrize('shape', [(20, 50), (200, 150)])
def test_other_polynomials(shape, steps, abc):
    g = torch.Generator(device=DEV).manual_seed(3)
    u = torch.randn(shape, device=DEV, generator=g)
    near(optim.orthogonalize(u, steps, abc), u, torch.float32, steps, abc)


@pytest.mark.parametrize('shape', [(12, 30), (150, 260)])
def test_degenerate_matrices(shape):
    """Zeros stay zeros, a matrix of rank one gets one singular value, magnitudes do not matter, what is not finite stays
    in its matrix."""
    g = torch.Generator(device=DEV).manual_seed(1)
    u = torch.randn((4,) + shape, device=DEV, generator=g)
    z = u.clone()
    z[1] = 0
    z[2] = torch.outer(u[2, :, 0], u[2, 0])
    out = optim.orthogonalize(z)
    assert float(out[1].abs().max()) == 0
    near(out[2], z[2], torch.float32)
    s = torch.linalg.svdvals(out[2].double().cpu())
    assert 0.6 < float(s[0]) < 1.3 and float(s[1]) < 1e-3
    assert torch.equal(out[0], optim.orthogonalize(u)[0])
    near(optim.orthogonalize(u[0] * 1e-3, eps=1e-30), u[0], torch.float32)
    near(optim.orthogonalize(u[0] * 2.0 ** -60, eps=1e-30), u[0], torch.float32)
    near(optim.orthogonalize(u[0] * 2.0 ** 100), u[0], torch.float32)
    big = (u[0] * 2.0 ** 120).bfloat16()
    assert torch.equal(optim.orthogonalize(big), optim.orthogonalize((u[0] * 2.0 ** 20).bfloat16()))   # (a power of two)
    # below eps the update shrinks instead of being raised from noise: X0 = u 1e-12 / 1e-3, and as far from 1 the
    # polynomial is a X, five times.  Entries of 1e-9 x 2^15 are kept to half a subnormal step of a half, 2^-25: 2^-10 of them
    small = optim.orthogonalize(u[0] * 1e-12, eps=1e-3)
    want = optim.QUINTIC[0] ** 5 * 1e-9 * float(u[0].double().norm())
    assert abs(float(small.double().norm()) - want) <= 2.0 ** -8 * want
    for bad in (math.nan, math.inf):
        w = u.clone()
        w[3, 1, 1] = bad
        o = optim.orthogonalize(w)
        assert torch.equal(o[:3], optim.orthogonalize(u)[:3]) and not bool(torch.isfinite(o[3]).all())


def test_orthogonalize_views_streams_and_empty():
    u = torch.randn((60, 200), device=DEV)
    want = optim.orthogonalize(u)
    assert torch.equal(optim.orthogonalize(u.t().contiguous().t()), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = optim.orthogonalize(u)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert optim.orthogonalize(torch.zeros((0, 3, 4), device=DEV)).shape == (0, 3, 4)
    assert optim.orthogonalize(torch.zeros((2, 0, 4), device=DEV)).shape == (2, 0, 4)
    for bad, word in (((u[0],), 'matrices'), ((u.double(),), 'float32'), ((u, 0), 'steps'), ((u, 5, (1.0, 2.0)), 'coefficients'),
                      ((u, 5, optim.QUINTIC, 0.0), 'eps')):
        with pytest.raises((RuntimeError, ValueError), match=word):
            optim.orthogonalize(*bad)
    with pytest.raises(RuntimeError, match='polynomial'):
        optim.orthogonalize(u, 5, (9.0, 9.0, 9.0))


def reference_step(w, g, m, lr, beta, decay, nesterov, batched=False):
    w, g, m = w.double(), g.double(), m.double()
    m = beta * m + g
    u = g + beta * m if nesterov else m
    mat = u if batched else u.reshape(u.shape[0], -1)
    o = formula(mat)
    return w * (1 - lr * decay) - lr * math.sqrt(max(1.0, mat.shape[-2] / mat.shape[-1])) * o.reshape(w.shape), m


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('nesterov', [True, False])
def test_muon_steps(dtype, nesterov):
    """Several steps over small, tiled, tall, convolution and odd weights, more than a launch's 32 matrices."""
    g = torch.Generator(device=DEV).manual_seed(11)
    shapes = [(64, 3), (64, 64), (32, 64), (128, 64, 3, 3), (200, 130), (700, 300), (5, 5), (1, 40), (40, 1), (96, 512, 1, 1)] + [(24, 31)] * 34
    params = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g).to(dtype)) for s in shapes]
    opt = optim.Muon(params, lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
    ref = [(p.detach().double(), torch.zeros_like(p, dtype=torch.float64)) for p in params]
    for k in range(3):
        for p in params:
            p.grad = (torch.randn(p.shape, device=DEV, generator=g) * 1e-2).to(dtype)
        before = [p.detach().clone() for p in params]
        opt.step()
        for i, p in enumerate(params):
            w, m = reference_step(before[i], p.grad, ref[i][1], 0.05, 0.9, 0.1, nesterov)
            ref[i] = (w, m)
            e = torch.finfo(dtype).eps / 2
            # the update's own error (see above) times lr, the rounding of W, and 4 roundings of 32 bits
            tall = math.sqrt(max(1.0, p.shape[0] / (p.numel() // p.shape[0])))
            tol = e * float(w.norm()) + 0.05 * tall * 341 * 8 * 2.0 ** -22 * 1.2 * math.sqrt(min(p.shape[0], p.numel() // p.shape[0])) + 4 * 2.0 ** -24 * float(w.norm())
            assert float((p.detach().double() - w).norm()) <= tol, (shapes[i], k)
            buf = opt.state[p]['momentum_buffer']
            assert buf.dtype == torch.float32
            assert float((buf.double() - m).norm()) <= (k + 1) * 2 * 2.0 ** -24 * float(m.norm()) * 2


def test_muon_batched_absent_gradients_and_state():
    g = torch.Generator(device=DEV).manual_seed(2)
    z = torch.nn.Parameter(torch.randn((4, 15, 512), device=DEV, generator=g))
    rest = torch.nn.Parameter(torch.randn((30, 20), device=DEV, generator=g))
    opt = optim.Muon([z, rest], lr=0.1, momentum=0.5, batched=True)
    z.grad = torch.randn(z.shape, device=DEV, generator=g)
    w, _ = reference_step(z.detach(), z.grad, torch.zeros_like(z), 0.1, 0.5, 0.0, True, batched=True)
    kept = rest.detach().clone()
    opt.step()
    assert torch.equal(rest.detach(), kept) and 'momentum_buffer' not in opt.state[rest]
    assert float((z.detach().double() - w).norm()) <= 2.0 ** -20 * float(w.norm())
    # a state that is saved and loaded goes on as the first one does, also where the parameters are of 16 bits
    for dtype in (torch.float32, torch.bfloat16):
        p = torch.nn.Parameter(torch.randn((40, 50), device=DEV, generator=g).to(dtype))
        a = optim.Muon([p], lr=0.1)
        p.grad = torch.randn((40, 50), device=DEV, generator=g).to(dtype)
        a.step()
        q = torch.nn.Parameter(p.detach().clone())
        b = optim.Muon([q], lr=0.1)
        b.load_state_dict(copy.deepcopy(a.state_dict()))
        q.grad = p.grad = torch.randn((40, 50), device=DEV, generator=g).to(dtype)
        a.step()
        b.step()
        assert torch.equal(p, q) and torch.equal(a.state[p]['momentum_buffer'], b.state[q]['momentum_buffer'])


def test_muon_refusals_and_groups():
    with pytest.raises(ValueError, match='two or more'):
        optim.Muon([torch.nn.Parameter(torch.zeros(3, device=DEV))])
    with pytest.raises(ValueError, match='momentum'):
        optim.Muon([torch.nn.Parameter(torch.zeros((3, 3), device=DEV))], momentum=1.0)
    p = torch.nn.Parameter(torch.zeros((3, 3)))
    p.grad = torch.ones((3, 3))
    with pytest.raises(RuntimeError, match='HIP devices only'):
        optim.Muon([p]).step()
    t = torch.nn.Parameter(torch.zeros((4, 3), device=DEV).t())
    t.grad = torch.ones((3, 4), device=DEV)
    with pytest.raises(RuntimeError, match='contiguous'):
        optim.Muon([t]).step()
    a, b = (torch.nn.Parameter(torch.ones((8, 8), device=DEV)) for _ in range(2))
    opt = optim.Muon([{'params': [a], 'lr': 0.0}, {'params': [b], 'lr': 1.0}])
    a.grad = b.grad = torch.eye(8, device=DEV)
    opt.step()
    assert torch.equal(a.detach(), torch.ones((8, 8), device=DEV)) and not torch.equal(a, b)


def test_a_step_reaches_what_is_cached_by_version():
    """EqualizedLinear keeps its scaled weight by the parameter's version: an evaluation after a step uses the new one."""
    lin = EqualizedLinear(64, 64, bias=False).to(DEV)
    x = torch.randn((5, 64), device=DEV)
    with torch.no_grad():
        before = lin(x)
    opt = optim.Muon([lin.weight], lr=0.5)
    lin(x).square().sum().backward()
    opt.step()
    lin.requires_grad_(False)
    with torch.no_grad():
        after = lin(x)
        assert float((after - x @ (lin.weight * lin.weight_gain).t()).abs().max()) < 1e-4
    assert float((after - before).abs().max()) > 1e-2


def test_captured_step():
    """Steps replayed from a graph equal eager ones on the same gradients, both kernels, between eager work."""
    g = torch.Generator(device=DEV).manual_seed(4)
    shapes = [(64, 64), (200, 300), (30, 512)]
    p = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g)) for s in shapes]
    q = [torch.nn.Parameter(v.detach().clone()) for v in p]
    grads = [torch.randn(s, device=DEV, generator=g) for s in shapes]
    oa, ob = optim.Muon(p, lr=0.1), optim.Muon(q, lr=0.1)
    for v, w, d in zip(p, q, grads):
        v.grad, w.grad = d, d
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        oa.step()
    torch.cuda.current_stream().wait_stream(side)
    ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for k in range(4):
        for d in grads:
            d.copy_(torch.randn(d.shape, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        ob.step()
        assert all(torch.equal(a, b) for a, b in zip(p, q)), k
        assert all(torch.equal(oa.state[a]['momentum_buffer'], ob.state[b]['momentum_buffer']) for a, b in zip(p, q))


def test_two_wide_bf16_matrices_repeat_and_stay_as_near_as_32_bit_products():
    """The largest tiles' case, 272 of them for 256 compute units: the same bits whatever its workspace held before and
    whatever else runs; and before its one rounding it is as near to 64 bits as the formula in 32-bit products (2.4e-6 of the
    norm, those 3.8e-6), so that the 0.4 % of values where the two fall on different sides of a bf16 border are not its errors."""
    g = torch.Generator(device=DEV).manual_seed(7)
    u = (torch.randn((2, 2048, 2048), device=DEV, generator=g) * torch.exp2(-2 * torch.randn((2048,), device=DEV, generator=g).abs()) * 1e-3).bfloat16()
    first = optim.orthogonalize(u)
    side, other = torch.cuda.Stream(), torch.randn((4096, 4096), device=DEV)
    for k in range(4):
        junk = torch.full((1 << 26,), math.nan, device=DEV)
        del junk
        with torch.cuda.stream(side):
            other @ other
        assert torch.equal(optim.orthogonalize(u), first), k
    torch.cuda.synchronize()
    v = u.float()
    own = optim.orthogonalize(v)
    assert torch.equal(own.bfloat16(), first)
    near(own, v, torch.float32)


def step_op(params, grads, momenta, batched=False, lr=0.1):
    from nfi import torch_ops
    torch_ops.op('muon_step')(params, grads, momenta, batched, lr, 0.9, 0.0, True, 5, *optim.QUINTIC, 1e-7)


def test_the_step_operator_leaves_empty_parameters_alone():
    """torch.ops.nfi.muon_step, as a C++ or TorchScript caller reaches it: a parameter without values divides nothing, and
    the others of its call are stepped."""
    for batched, shapes in ((False, [(0, 3), (3, 0), (0, 0), (4, 0, 3)]), (True, [(2, 0, 4), (0, 3, 4), (2, 3, 0)])):
        empty = [torch.zeros(s, device=DEV) for s in shapes]
        step_op(empty, [torch.zeros_like(t) for t in empty], [torch.zeros_like(t) for t in empty], batched)
        w, g = torch.ones((6, 8), device=DEV), torch.randn((6, 8), device=DEV)
        m = torch.zeros_like(w)
        want, want_m = reference_step(w, g, m, 0.1, 0.9, 0.0, True)
        params = empty[:1] + [w] + empty[1:]
        step_op(params, [torch.zeros_like(t) if t is not w else g for t in params], [torch.zeros_like(t) if t is not w else m for t in params], batched)
        # (the update's own error times lr, see above, and W's roundings; M is G itself)
        assert float((w.double() - want).norm()) <= 0.1 * 341 * 8 * 2.0 ** -22 * 6 ** 0.5 + 4 * 2.0 ** -24 * float(want.norm())
        assert torch.equal(m, g) and float((m.double() - want_m).abs().max()) == 0


def test_a_refused_matrix_stops_the_step_before_anything_changes():
    """One call steps the 32-bit parameters, another the 16-bit ones: a matrix that the second refuses leaves the first's
    weights, momenta and versions as they were, and so does a polynomial."""
    def tensors(dtype, *shape):
        return torch.ones(shape, device=DEV, dtype=dtype), torch.ones(shape, device=DEV, dtype=dtype), torch.zeros(shape, device=DEV)
    w, g, m = tensors(torch.float32, 6, 8)
    # 2^24 matrices of one value: too many for a call
    many, many_g, many_m = tensors(torch.bfloat16, 1 << 24, 1, 1)
    bw, bg, bm = w[None], g[None], m[None]
    versions = w._version, m._version
    with pytest.raises(RuntimeError, match='too large'):
        step_op([bw, many], [bg, many_g], [bm, many_m], batched=True)
    from nfi import torch_ops
    with pytest.raises(RuntimeError, match='polynomial'):
        torch_ops.op('muon_step')([w, many[:3, 0]], [g, many_g[:3, 0]], [m, many_m[:3, 0]], False, 0.1, 0.9, 0.0, True, 5, 9.0, 9.0, 9.0, 1e-7)
    assert torch.equal(w, torch.ones_like(w)) and float(m.abs().max()) == 0 and (w._version, m._version) == versions
    assert float((many - 1).abs().max()) == 0 and float(many_m.abs().max()) == 0


def test_the_first_step_is_refused_in_a_capture():
    """And taken eagerly behind it, from where the parameter was; then the capture works."""
    p = torch.nn.Parameter(torch.ones((20, 30), device=DEV))
    p.grad = torch.randn((20, 30), device=DEV)
    opt = optim.Muon([p], lr=0.1)
    optim.orthogonalize(p.grad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='before the capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), torch.ones_like(p)) and 'momentum_buffer' not in opt.state.get(p, {})
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = p.grad
    other = optim.Muon([q], lr=0.1)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        other.step()
        assert torch.equal(p, q)


def test_more_small_matrices_than_a_launch_takes():
    """4,300,000 of 2 x 3 (a launch has fewer than 2^32 threads, 2^22 workgroups of 1024): each as in a call of its own."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n = 4300000
    u = torch.randn((n, 2, 3), device=DEV, generator=g)
    out = optim.orthogonalize(u)
    for at in (0, (1 << 21) - 3, (1 << 21), (1 << 22) - 5, (1 << 22), n - 9):
        assert torch.equal(out[at:at + 9], optim.orthogonalize(u[at:at + 9].clone())), at
    ref = formula(u.double())
    # (each matrix's own bound, see above: |X|_F is at most sqrt(2))
    assert float((out.double() - ref).norm(dim=(1, 2)).max()) <= 341 * 8 * 2.0 ** -22 * 2 ** 0.5
    p = torch.nn.Parameter(torch.ones((n, 2, 3), device=DEV, dtype=torch.bfloat16))
    p.grad = u.bfloat16()
    opt = optim.Muon([p], lr=0.5, momentum=0.0, batched=True)
    opt.step()
    o = optim.orthogonalize(p.grad)
    assert float((p.detach().float() - (1 - 0.5 * o.float())).abs().max()) <= 2.0 ** -7 * 2
    assert torch.equal(opt.state[p]['momentum_buffer'], p.grad.float())


@pytest.mark.parametrize('count', [9, 32, 33, 70])
def test_many_tiled_matrices(count):
    """More matrices that run as tiles than one, eight or thirty-two of a launch: each launch has the work buffer to itself, and the
    next begins behind it."""
    g = torch.Generator(device=DEV).manual_seed(count)
    shapes = [(65 + 7 * (i % 11), 66 + 31 * (i % 7)) if i % 3 else (260 - 3 * (i % 5), 70 + i) for i in range(count)]
    params = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g)) for s in shapes]
    for p in params:
        p.grad = torch.randn(p.shape, device=DEV, generator=g)
    before = [p.detach().clone() for p in params]
    opt = optim.Muon(params, lr=0.05, momentum=0.9, weight_decay=0.1)
    opt.step()
    for p, old in zip(params, before):
        w, m = reference_step(old, p.grad, torch.zeros_like(old), 0.05, 0.9, 0.1, True)
        tall = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        tol = 0.05 * tall * 341 * 8 * 2.0 ** -22 * 1.2 * math.sqrt(min(p.shape)) + 4 * 2.0 ** -24 * float(w.norm())
        assert float((p.detach().double() - w).norm()) <= tol, tuple(p.shape)
        # each alone, in a call of its own, is the same update within 32 bits (its products may be divided otherwise)
        alone = torch.nn.Parameter(old.clone())
        alone.grad = p.grad
        optim.Muon([alone], lr=0.05, momentum=0.9, weight_decay=0.1).step()
        assert float((alone.detach().double() - p.detach().double()).norm()) <= 2 * tol


def test_parameters_that_share_memory_are_refused():
    """The same tensor twice, a view beside its base, a momentum that two share: their steps would run at a time."""
    w, g = torch.ones((12, 8), device=DEV), torch.randn((12, 8), device=DEV)
    m, m2 = torch.zeros_like(w), torch.zeros_like(w)
    for params, grads, momenta in (([w, w], [g, g], [m, m2]), ([w, w[4:9]], [g, g[4:9]], [m, m2[4:9]]), ([w, w[:1]], [g, g[:1]], [m, m2[:1]]),
                                   ([w, w.clone()], [g, g], [m, m]), ([w], [g], [w])):
        with pytest.raises(ValueError, match='share memory'):
            step_op(params, grads, momenta)
    a = torch.nn.Parameter(w)
    b = torch.nn.Parameter(w[2:5])
    a.grad, b.grad = g, g[2:5]
    with pytest.raises(ValueError, match='share memory'):
        optim.Muon([a, b]).step()
    assert torch.equal(w, torch.ones_like(w)) and float(m.abs().max()) == 0 and float(m2.abs().max()) == 0
    # neighbours in one buffer, and one gradient for two, are separate parameters
    step_op([w[:6], w[6:]], [g[:6], g[:6]], [m[:6], m[6:]])
    assert torch.equal(w[:6], w[6:]) and torch.equal(m[:6], g[:6])
