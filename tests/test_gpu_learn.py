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
