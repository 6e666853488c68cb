"""The operators that train the field's heads, used together: a bank of view-direction mappers over a batch that mixes
categories, against each mapper's own trunk (viewdir_trunk in 64 bits), its gradients, steps of its weights by Muon, and
the inversion loop with orthogonalised latent updates."""

import copy

import pytest
import torch

import nfi
from nfi import inversion, optim
from nfi.viewdir import ViewDirectionMapper, ViewDirectionMapperBank, viewdir_trunk
from test_producer import inversion_setup

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
U = 2.0 ** -24


def bank(count, seed=0):
    torch.manual_seed(seed)
    mappers = [ViewDirectionMapper(10).to(DEV) for _ in range(count)]
    for m in mappers:
        for k in range(1, 5):
            with torch.no_grad():
                getattr(m, f'norm{k}').weight.add_(torch.randn(64, device=DEV) * 0.1)
                getattr(m, f'norm{k}').bias.add_(torch.randn(64, device=DEV) * 0.1)
    return ViewDirectionMapperBank(mappers)


@pytest.mark.parametrize('which', [[0, 0, 1, 2], [0], [1, 1, 3], [2, 2, 2]])
def test_bank_against_each_trunk(which):
    """Depth: 7 products (longest sum 64) and 4 norms, each amplifying what it gets by at most its row's 1 / deviation (about
    1 to 4 here): 2^9 u of the largest value is 7 layers' own errors times that, with room."""
    b = bank(4)
    rays = 133
    v = torch.nn.functional.normalize(torch.randn((len(which), rays, 3), device=DEV), dim=-1).requires_grad_()
    image = torch.tensor(which, device=DEV)
    x = b(v, image)
    g = torch.randn_like(x)
    params = dict(b.named_parameters())
    used = [k for k in params if 'output' not in k]
    got = torch.autograd.grad(x, [v] + [params[k] for k in used], g)
    b64 = copy.deepcopy(b).double()
    v64 = v.detach().double().requires_grad_()
    ref = torch.stack([viewdir_trunk(b64.mappers[m], v64[i].unsqueeze(-2)).squeeze(-2) for i, m in enumerate(which)])
    params64 = dict(b64.named_parameters())
    want = torch.autograd.grad(ref, [v64] + [params64[k] for k in used], g.double(), allow_unused=True)
    assert float((x.double() - ref).abs().max()) <= 2 ** 9 * U * max(1.0, float(ref.abs().max()))
    for k, a, w in zip(['viewdir'] + used, got, want):
        if w is None:
            assert float(a.abs().max()) == 0, k     # a mapper that no image went through
        else:
            # (by norm; sums over up to 400 rows, and the slope's steps at zero are the same on both sides for these seeds)
            assert float((a.double() - w).norm()) <= 2 ** 11 * U * float(w.norm()) + 1e-12, k


def test_training_steps_of_a_bank():
    """Two steps by Muon on the mappers' matrices: each weight moves as the formula says for its gradient."""
    b = bank(3, 1)
    image = torch.tensor([0, 1, 1, 2], device=DEV)
    v = torch.nn.functional.normalize(torch.randn((4, 200, 3), device=DEV), dim=-1)
    target = torch.randn((4, 200, 32), device=DEV)
    weights = [p for k, p in b.named_parameters() if p.dim() == 2 and 'output' not in k]
    opt = optim.Muon(weights, lr=0.02)
    for _ in range(2):
        opt.zero_grad()
        (b(v, image) - target).square().mean().backward()
        before = [w.detach().clone() for w in weights]
        state = [opt.state[w]['momentum_buffer'].clone() if w in opt.state else torch.zeros_like(w) for w in weights]
        opt.step()
        for w, old, m in zip(weights, before, state):
            m = 0.95 * m + w.grad
            o = optim.orthogonalize(w.grad + 0.95 * m)
            tall = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
            assert float((w.detach() - (old - 0.02 * tall * o)).abs().max()) <= 1e-5


def test_no_double_backward():
    """A graph of the gradients is refused, not built without them."""
    from nfi.grouped import grouped_linear
    from nfi.norms import residual_norm
    x = torch.randn((6, 8), device=DEV, requires_grad=True)
    w = torch.randn((1, 5, 8), device=DEV, requires_grad=True)
    for y in (residual_norm(x), grouped_linear(x, w, torch.tensor([0, 6], device=DEV))):
        with pytest.raises(RuntimeError, match='double backward'):
            torch.autograd.grad(y.sum(), [x], create_graph=True)


def test_bank_refuses():
    b = bank(2)
    with pytest.raises(ValueError, match='mapper_of_image'):
        b(torch.zeros((2, 5, 3), device=DEV), torch.zeros((3,), device=DEV, dtype=torch.int64))
    with pytest.raises(ValueError, match='mapper_of_image'):
        b(torch.zeros((2, 5, 3), device=DEV), torch.zeros((2,), device=DEV, dtype=torch.int32))


@pytest.mark.parametrize('graph', [False, True])
def test_inversion_with_orthogonalised_latent_steps(graph):
    """InversionConfig.latent_update = 'muon': each image's latent moves by an orthogonalised step of the given length, the
    pose as with Adam; eager and replayed, twice over the same graph."""
    gen, d, meta, cfg = inversion_setup(DEV)
    nfi.configure(scene_range=float(meta['scene_range']), white_background=False, fine_sampling=True, use_sdf=True,
                  attention_values=10, use_viewdir=False)
    cfg.latent_update, cfg.latent_lr, cfg.steps, cfg.graph = 'muon', 0.05, 4, graph
    for _ in range(2):
        seen = [d['w_init'].to(DEV).expand(d['target'].shape[0], -1, -1).clone()]
        res = inversion.invert(gen, d['target'], d['cam0'], d['focal0'], d['w_init'], cfg, checkpoints=(1, 2, 3, 4),
                               on_checkpoint=lambda it, v: seen.append(v[0].detach().clone() * cfg.gain_z))
        assert len(res.losses) == 4 and all(torch.isfinite(torch.tensor(res.losses)))
        for a, c in zip(seen, seen[1:]):
            step = (c - a) / cfg.gain_z / 0.05                      # 15 x 512: singular values near 1 where the gradient has any
            s = torch.linalg.svdvals(step.double().cpu())
            assert float(s.max()) < 1.3 and float(s[:, 0].min()) > 0.6
    cfg.latent_update = 'sgd'
    with pytest.raises(ValueError, match='latent_update'):
        inversion.invert(gen, d['target'], d['cam0'], d['focal0'], d['w_init'], cfg)


def test_two_graphs_and_eager_calls_take_turns():
    """Two captured runs of all three operators (products whose rows are split, a norm with its gradients, an update in
    tiles), replayed in turn on two streams and between eager calls: each leaves what it left alone."""
    from nfi import grouped, norms

    def setup(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)

        def rnd(*shape):
            return torch.randn(shape, device=DEV, generator=g)
        x, w, gy = rnd(3001, 200).requires_grad_(), (rnd(3, 136, 200) * 0.1).requires_grad_(), rnd(3001, 136)
        gate, weight, bias = (rnd(136).requires_grad_() for _ in range(3))
        offsets = torch.tensor([0, 1200 + seed, 1200 + seed, 2990], device=DEV, dtype=torch.int32)

        def step():
            h = grouped.grouped_linear(x, w, offsets)
            y = norms.residual_norm(h, None, gate, weight, bias, slope=0.2)
            grads = torch.autograd.grad(y, [x, w, gate, weight, bias], gy)
            return [y.detach(), *grads, optim.orthogonalize(grads[1])]
        return x, step

    runs = [setup(1), setup(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _, step in runs:
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, held = [], []
    for _, step in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step())
        graphs.append(graph)
    for turn in range(4):
        with torch.no_grad():
            for x, _ in runs:
                x.mul_(0.9)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        for (_, step), h in zip(runs, held):
            assert all(torch.equal(a, b) for a, b in zip(h, step()))
        torch.cuda.synchronize()


@pytest.mark.parametrize('which', [[1, 0, 1], [3, 0, 2, 0, 1]])
def test_bank_takes_images_in_any_order(which):
    """Each image's rows and gradients are those of the same images in their mappers' order, bit for bit (a row's sums
    do not depend on its place; the weights' gradients are summed over the same rows in the same order)."""
    b = bank(4)
    v = torch.nn.functional.normalize(torch.randn((len(which), 70, 3), device=DEV), dim=-1)
    g = torch.randn((len(which), 70, 32), device=DEV)
    image = torch.tensor(which, device=DEV)
    order = torch.tensor(sorted(range(len(which)), key=lambda i: which[i]), device=DEV)
    params = [p for k, p in b.named_parameters() if 'output' not in k]
    results = []
    for pick in (slice(None), order):
        leaf = v[pick].clone().requires_grad_()
        x = b(leaf, image[pick])
        results.append([x.detach(), *torch.autograd.grad(x, [leaf] + params, g[pick])])
    (x, gv, *gp), (xs, gvs, *gps) = results
    assert torch.equal(x[order], xs) and torch.equal(gv[order], gvs)
    assert all(torch.equal(p, q) for p, q in zip(gp, gps))
    for i, m in enumerate(which):
        ref = viewdir_trunk(copy.deepcopy(b.mappers[m]).double(), v[i].double().unsqueeze(-2)).squeeze(-2)
        assert float((x[i].double() - ref).abs().max()) <= 2 ** 9 * U * max(1.0, float(ref.abs().max())), i


def test_bank_leaves_out_images_of_no_mapper():
    """They give zeros and no gradients; the others, and every parameter's gradient, are what they are without them."""
    b = bank(3)
    v = torch.nn.functional.normalize(torch.randn((5, 40, 3), device=DEV), dim=-1)
    g = torch.randn((5, 40, 32), device=DEV)
    which = torch.tensor([2, -1, 0, 3, 2], device=DEV)
    keep = torch.tensor([0, 2, 4], device=DEV)
    params = [p for k, p in b.named_parameters() if 'output' not in k]
    leaf, alone = v.clone().requires_grad_(), v[keep].clone().requires_grad_()
    x, y = b(leaf, which), b(alone, which[keep])
    gv, *gp = torch.autograd.grad(x, [leaf] + params, g)
    gw, *gq = torch.autograd.grad(y, [alone] + params, g[keep])
    assert torch.equal(x[keep], y) and torch.equal(gv[keep], gw)
    assert float(x[[1, 3]].detach().abs().max()) == 0 and float(gv[[1, 3]].abs().max()) == 0
    # (sums over the same rows; zeros of the rows left out may stand between them)
    assert all(float((p - q).abs().max()) <= 2 ** 8 * U * float(q.abs().max()) + 1e-12 for p, q in zip(gp, gq))


@pytest.mark.parametrize('images,rays', [(0, 5), (3, 0)])
def test_bank_of_an_empty_batch(images, rays):
    b = bank(2)
    v = torch.zeros((images, rays, 3), device=DEV, requires_grad=True)
    x = b(v, torch.zeros((images,), device=DEV, dtype=torch.int64))
    assert x.shape == (images, rays, 32)
    gv, gw = torch.autograd.grad(x.sum(), [v, b.mappers[0].fc1.weight])
    assert gv.shape == v.shape and float(gw.abs().max()) == 0


def test_traced_and_scripted_calls():
    """Fake tensors of the device give shapes, forward and backward, without a launch; under a mode that looks on, and
    from TorchScript, the values and gradients are the call's own, bit for bit."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.utils._python_dispatch import TorchDispatchMode
    from test_learn_host import shapes_of_calls
    from nfi import grouped, norms, torch_ops
    with FakeTensorMode():
        shapes_of_calls('cuda', True)

    seen = []

    class Looks(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    g = torch.Generator(device=DEV).manual_seed(9)

    def rnd(*shape):
        return torch.randn(shape, device=DEV, generator=g)
    h, gate, weight, gx = rnd(12, 40), rnd(3, 40), rnd(40), rnd(12, 40)
    x, w, b, gy = rnd(30, 24), rnd(2, 16, 24), rnd(2, 16), rnd(30, 16)
    off = torch.tensor([0, 13, 28], device=DEV)
    leaves = [t.requires_grad_() for t in (h, gate, weight, x, w, b)]

    def all_of_it():
        n = norms.residual_norm(h, None, gate, weight, slope=0.2, next_norm='rms')
        y = grouped.grouped_linear(x, w, off, b)
        return [*(t.detach() for t in (*n, y)), *torch.autograd.grad([*n, y], leaves, [gx, gx, gy]), optim.orthogonalize(w)]
    want = all_of_it()
    with Looks():
        got = all_of_it()
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    for name in ('residual_norm_fwd', 'residual_norm_bwd', 'grouped_linear_fwd', 'grouped_linear_bwd', 'orthogonalize'):
        assert any(name in s for s in seen), name

    torch_ops.load()
    unit = torch.jit.CompilationUnit('''
def run(h: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, x: torch.Tensor, w: torch.Tensor, off: torch.Tensor, b: torch.Tensor):
    n = torch.ops.nfi.residual_norm(h, None, gate, weight, None, None, None, 1, 2, 0.2, 1.0, 1e-5)
    y = torch.ops.nfi.grouped_linear(x, w, off, b)
    return n[0], n[1], y, torch.ops.nfi.orthogonalize(w.detach(), 5, 3.4445, -4.7750, 2.0315, 1e-7)
''')
    for _ in range(3):
        n0, n1, y, o = unit.run(h, gate, weight, x, w, off, b)
        got = [n0.detach(), n1.detach(), y.detach(), *torch.autograd.grad([n0, n1, y], leaves, [gx, gx, gy]), o]
        assert all(torch.equal(a, c) for a, c in zip(want, got))


def test_halves_refuse_what_they_cannot_take():
    """The plain operators behind the two autograd functions check their own arguments."""
    from nfi import torch_ops
    torch_ops.load()
    ops = torch.ops.nfi
    z = torch.zeros
    h, st = z((4, 8), device=DEV), z((4, 4), device=DEV)
    conf = (1, 0, 1.0, 1.0, 1e-5)
    none6 = (None,) * 6
    needs = [True] + [False] * 6
    assert ops.residual_norm_fwd(h, *none6, *conf, True)[2].shape == (4, 4)
    assert ops.residual_norm_bwd(h, None, h, *none6, st, *conf, needs)[0].shape == (4, 8)
    x, w, off = z((5, 8), device=DEV), z((2, 3, 8), device=DEV), z((3,), device=DEV, dtype=torch.int64)
    gy = z((5, 3), device=DEV)
    for f, word in ((lambda: ops.residual_norm_fwd(z((2, 2, 8), device=DEV), *none6, *conf, True), 'rows, width'),
                    (lambda: ops.residual_norm_fwd(h.t(), *none6, *conf, True), 'contiguous'),
                    (lambda: ops.residual_norm_fwd(h, None, z((8,), device=DEV), *none6[2:], *conf, True), 'gate'),
                    (lambda: ops.residual_norm_bwd(None, None, h, *none6, st, *conf, needs), 'no gradient'),
                    (lambda: ops.residual_norm_bwd(h, None, h, *none6, None, *conf, needs), 'stats'),
                    (lambda: ops.residual_norm_bwd(h, None, h, *none6, st[:3], *conf, needs), 'stats'),
                    (lambda: ops.residual_norm_bwd(h[:3], None, h, *none6, st, *conf, needs), 'gradients like h'),
                    (lambda: ops.residual_norm_bwd(h, h, h, *none6, st, *conf, needs), 'next norm'),
                    (lambda: ops.residual_norm_bwd(h, None, h, *none6, st, *conf, [True] * 7), 'absent'),
                    (lambda: ops.grouped_linear_fwd(x, w.transpose(1, 2).contiguous().transpose(1, 2), off), 'contiguous'),
                    (lambda: ops.grouped_linear_bwd(gy[:4], x, w, off, [True] * 3), 'gy'),
                    (lambda: ops.grouped_linear_bwd(gy.half(), x, w, off, [True] * 3), 'gy'),
                    (lambda: ops.grouped_linear_bwd(gy, x, w, off[:2], [True] * 3), 'offsets')):
        with pytest.raises((RuntimeError, ValueError), match=word):
            f()


def behind(need, held=0xa5):
    """A work buffer of `need` bytes at the head of a longer one, and a function that says whether what follows is untouched."""
    buf = torch.full((max(need, 0) + (1 << 20),), 0xa5, device=DEV, dtype=torch.uint8)
    buf[:max(need, 0)] = held
    return buf.data_ptr(), lambda: bool((buf[max(need, 0):] == 0xa5).all())


@pytest.mark.parametrize('width', [24, 64, 512, 513, 1000, 1024, 1025, 2048, 2049, 4100, 8192])
@pytest.mark.parametrize('groups,affine', [(0, 0), (7, 0), (7, 1), (400, 1), (800, 0), (1600, 1)])
def test_norm_workspace_is_enough(width, groups, affine):
    """Every layout's backward through the C interface, its work buffer of the size that it is told: nothing behind it is
    written, and the parameters' gradients do not depend on what it held."""
    import ctypes
    from nfi import _lib
    lib = _lib.load()
    rows = 2800 if groups == 7 else 1600
    t = {k: torch.randn((rows, width), device=DEV) for k in ('h', 'residual', 'gx', 'gy')}
    t.update(stats=torch.rand((rows, 4), device=DEV) + 0.5, dh=torch.empty((rows, width), device=DEV), dresidual=torch.empty((rows, width), device=DEV))
    per = (groups, width) if affine else (width,)
    for k in ('weight', 'bias', 'next_weight', 'next_bias'):
        t[k], t['d' + k] = torch.randn(per, device=DEV), torch.empty(per, device=DEV)
    if groups:
        t['gate'], t['dgate'] = torch.randn((groups, width), device=DEV), torch.empty((groups, width), device=DEV)
    a = _lib.NfiResnormArgs()
    for k, v in t.items():
        setattr(a, k, v.data_ptr())
    a.rows, a.groups, a.width, a.norm, a.next_norm, a.affine_groups = rows, groups, width, 1, 2, affine
    a.slope, a.scale, a.eps = 0.2, 0.7, 1e-5
    need = lib.nfi_resnorm_work_bytes(rows, groups, affine, width)
    kept = []
    for held in (0, 0xff):
        a.work, untouched = behind(need, held)
        assert lib.nfi_resnorm_backward(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0, lib.nfi_last_error()
        torch.cuda.synchronize()
        assert untouched()
        kept.append([t[k].clone() for k in t if k[0] == 'd'])
    assert all(torch.equal(p, q) for p, q in zip(*kept))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,groups,k,n,need', [(700, 3, 33, 65, 'xwb'), (5000, 1, 64, 64, 'xwb'), (5000, 2, 129, 40, 'xw'), (40000, 1, 7, 130, 'b'),
                                                  (3000, 2, 200, 136, 'wb'), (90, 20, 31, 33, 'x')])
def test_grouped_workspace_is_enough(rows, groups, k, n, need, dtype):
    import ctypes
    from nfi import _lib
    lib = _lib.load()
    x, w, gy = (torch.randn(s, device=DEV).to(dtype) for s in ((rows, k), (groups, n, k), (rows, n)))
    bias = torch.randn((groups, n), device=DEV).to(dtype)
    off = torch.linspace(0, rows, groups + 1, device=DEV).to(torch.int32)
    y, gx, gw, gb = (torch.empty_like(v) for v in (gy, x, w, bias))
    a = _lib.NfiGroupedArgs()
    a.x, a.w, a.bias, a.offsets, a.y = (v.data_ptr() for v in (x, w, bias, off, y))
    a.rows, a.groups, a.in_width, a.out_width, a.dtype = rows, groups, k, n, 0 if dtype == torch.float32 else 1
    stream = torch.cuda.current_stream().cuda_stream
    for size, call in ((lib.nfi_grouped_forward_work_bytes, lib.nfi_grouped_forward), (lib.nfi_grouped_backward_work_bytes, lib.nfi_grouped_backward)):
        if call is lib.nfi_grouped_backward:
            a.gy = gy.data_ptr()
            a.gx, a.gw, a.gb = (v.data_ptr() if c in need else None for c, v in zip('xwb', (gx, gw, gb)))
        a.work_bytes = size(ctypes.byref(a))
        a.work, untouched = behind(a.work_bytes)
        assert call(ctypes.byref(a), stream) == 0, lib.nfi_last_error()
        torch.cuda.synchronize()
        assert untouched()


def test_ortho_workspace_is_enough():
    import ctypes
    from nfi import _lib
    lib = _lib.load()
    shapes = [(200, 300, 1), (65, 1300, 3), (640, 70, 2), (15, 2049, 1), (64, 64, 5)] + [(70 + i, 90, 1) for i in range(40)] + [(300, 300, 2)]
    held = [torch.randn((c, r, n), device=DEV) for r, n, c in shapes]
    out = [torch.empty_like(v) for v in held]
    items = (_lib.NfiOrthoItem * len(shapes))(*[_lib.NfiOrthoItem(v.data_ptr(), None, o.data_ptr(), r, n, c, 1.0)
                                                for v, o, (r, n, c) in zip(held, out, shapes)])
    a = _lib.NfiOrthoArgs()
    a.items, a.n_items, a.steps, a.eps = ctypes.cast(items, ctypes.POINTER(_lib.NfiOrthoItem)), len(shapes), 5, 1e-7
    a.a, a.b, a.c = optim.QUINTIC
    a.work_bytes = lib.nfi_ortho_work_bytes(items, len(shapes))
    results = []
    for fill in (0, 0xff):
        a.work, untouched = behind(a.work_bytes, fill)
        assert lib.nfi_ortho(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0, lib.nfi_last_error()
        torch.cuda.synchronize()
        assert untouched()
        results.append([o.clone() for o in out])
    assert all(torch.equal(p, q) for p, q in zip(*results))
    for v, o in zip(held, out):
        alone = optim.orthogonalize(v)
        assert float((alone.double() - o.double()).norm()) <= 2 * 341 * 8 * 2.0 ** -22 * float(alone.double().norm())


def test_a_captured_bank():
    """Forward and backward captured, replayed with other rays and other images' mappers between eager calls."""
    b = bank(3)
    v = torch.nn.functional.normalize(torch.randn((4, 50, 3), device=DEV), dim=-1).requires_grad_()
    image, g = torch.tensor([1, 0, 2, 1], device=DEV), torch.randn((4, 50, 32), device=DEV)
    params = [p for k, p in b.named_parameters() if 'output' not in k]

    def step():
        x = b(v, image)
        return [x.detach(), *torch.autograd.grad(x, [v] + params, g)]

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
    for which in ([1, 0, 2, 1], [2, 2, 0, 0], [0, 0, 0, 0], [5, 1, -1, 2], [0, 1, 2, 2]):
        with torch.no_grad():
            v.copy_(torch.nn.functional.normalize(torch.randn_like(v), dim=-1))
            image.copy_(torch.tensor(which))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step())), which
        torch.cuda.synchronize()
