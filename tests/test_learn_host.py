"""CPU: what the operators of include/nfi_learn.h refuse before anything is launched, and the layout of their
argument structs."""

import ctypes
import os
import subprocess

import pytest
import torch

from nfi import _lib, grouped, norms, optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize('name,struct', [('nfi_resnorm_args', 'NfiResnormArgs'), ('nfi_grouped_args', 'NfiGroupedArgs'),
                                         ('nfi_ortho_item', 'NfiOrthoItem'), ('nfi_ortho_args', 'NfiOrthoArgs')])
def test_struct_layout(tmp_path, name, struct):
    py = getattr(_lib, struct)
    fields = [f[0] for f in py._fields_]
    header = os.path.join(ROOT, 'include', 'nfi_learn.h')
    src = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{header}"', 'int main(void){',
           f'printf("%zu\\n", sizeof({name}));'] + [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ['return 0;}']
    (tmp_path / 'p.c').write_text('\n'.join(src))
    subprocess.run(['gcc', '-o', str(tmp_path / 'p'), str(tmp_path / 'p.c')], check=True)
    vals = [int(v) for v in subprocess.run([str(tmp_path / 'p')], check=True, capture_output=True, text=True).stdout.split()]
    assert vals == [ctypes.sizeof(py)] + [getattr(py, f).offset for f in fields]


def test_residual_norm_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match='HIP devices only'):
        norms.residual_norm(torch.zeros(2, 4))


def test_resnorm_entry_refuses_bad_arguments():
    lib = _lib.load()
    one = ctypes.c_void_p(16)

    def args(**kw):
        a = _lib.NfiResnormArgs()
        a.h = a.x = one
        a.rows, a.width, a.norm, a.eps = 4, 8, 1, 1e-5
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, word in (({'h': None}, b'null input'), ({'rows': 0}, b'rows'), ({'width': 8193}, b'width'),
                     ({'dtype': 7}, b'type'), ({'norm': 3}, b'norm'), ({'next_norm': -1}, b'norm'),
                     ({'gate': one, 'groups': 3}, b'groups'), ({'gate': one}, b'groups'), ({'affine_groups': 1}, b'groups'), ({'eps': -1.0}, b'eps'),
                     ({'x': None}, b'null output'), ({'next_norm': 1}, b'null output')):
        assert lib.nfi_resnorm_forward(ctypes.byref(args(**kw)), None) == -1, kw
        assert word in lib.nfi_last_error(), (kw, lib.nfi_last_error())
    for kw, word in (({}, b'statistics'), ({'stats': one, 'work': one}, b'no gradient'),
                     ({'stats': one, 'work': one, 'gy': one}, b'next norm')):
        assert lib.nfi_resnorm_backward(ctypes.byref(args(**kw)), None) == -1, kw
        assert word in lib.nfi_last_error(), kw


@pytest.mark.parametrize('affine', [0, 1])
@pytest.mark.parametrize('rows,groups', [(1, 0), (1, 1), (7, 7), (10 ** 6, 0), (10 ** 6, 2), (4096, 512), (4096, 2048), (511 * 3, 511)])
def test_resnorm_work_holds_every_workgroup(rows, groups, affine):
    """The plan's workgroups (restated) fit the work buffer for every number of rows a workgroup may hold."""
    lib = _lib.load()
    for slots in (1, 4, 8, 16, 32):
        g = groups if groups and (groups < rows or affine) else 1
        per_group = rows // g
        splits = min(max(1, 512 // g), -(-per_group // slots))
        segments = g * splits
        per = 1 if splits > 1 else -(-segments // 512)
        blocks = -(-segments // per)
        assert lib.nfi_resnorm_work_bytes(rows, groups, affine, 24) >= blocks * 5 * 24 * 4


def test_grouped_linear_refuses():
    with pytest.raises(RuntimeError, match='HIP devices only'):
        grouped.grouped_linear(torch.zeros(2, 4), torch.zeros(1, 3, 4), torch.tensor([0, 2]))
    lib = _lib.load()
    one = ctypes.c_void_p(16)

    def args(**kw):
        a = _lib.NfiGroupedArgs()
        a.x = a.w = a.y = a.offsets = one
        a.rows, a.groups, a.in_width, a.out_width = 4, 2, 8, 8
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, word in (({'offsets': None}, b'null input'), ({'rows': 0}, b'rows'), ({'rows': 1 << 31}, b'rows'), ({'groups': 0}, b'groups'),
                     ({'groups': 65536}, b'groups'), ({'in_width': 0}, b'widths'), ({'out_width': 1 << 22}, b'widths'),
                     ({'dtype': 3}, b'type'), ({'x': None}, b'null tensor'), ({'y': None}, b'null tensor'),
                     ({'in_width': 9}, b'work'), ({'rows': (1 << 31) - 1, 'out_width': 1 << 21}, b'tiles')):
        assert lib.nfi_grouped_forward(ctypes.byref(args(**kw)), None) == -1, kw
        assert word in lib.nfi_last_error(), (kw, lib.nfi_last_error())
    for kw, word in (({}, b'null tensor'), ({'gy': one, 'gx': one, 'w': None}, b'null tensor'),
                     ({'gy': one, 'gw': one, 'x': None}, b'null tensor'), ({'gy': one, 'gx': one, 'out_width': 7}, b'work')):
        assert lib.nfi_grouped_backward(ctypes.byref(args(**kw)), None) == -1, kw
        assert word in lib.nfi_last_error(), kw


@pytest.mark.parametrize('sizes,before,behind', [([1], 0, 0), ([0, 0, 5], 3, 0), ([128, 129, 0, 1], 0, 7), ([1] * 200, 1, 1),
                                                 ([300, 0, 4000, 127], 0, 128), ([0, 0], 2, 1)])
def test_row_tiles_cover_every_run(sizes, before, behind):
    """The launch's bound on row tiles (restated) is enough for every run of 128-row tiles, the rows of no group too."""
    rows = before + sum(sizes) + behind
    runs = sizes + [before, behind]
    assert sum(-(-r // 128) for r in runs) <= -(-rows // 128) + min(len(sizes) + 2, rows)


def test_ortho_refuses():
    with pytest.raises(RuntimeError, match='HIP devices only'):
        optim.orthogonalize(torch.zeros(2, 4))
    lib = _lib.load()
    one = ctypes.c_void_p(16)

    def args(item=None, **kw):
        it = _lib.NfiOrthoItem(one, None, one, 4, 5, 1, 1.0)
        for k, v in (item or {}).items():
            setattr(it, k, v)
        a = _lib.NfiOrthoArgs()
        a.items, a.n_items, a.steps, a.eps = ctypes.pointer(it), 1, 5, 1e-7
        a.a, a.b, a.c = optim.QUINTIC
        for k, v in kw.items():
            setattr(a, k, v)
        a.keep = it
        return a

    for item, kw, word in (({}, {'n_items': 0}, b'no matrices'), ({}, {'g_type': 5}, b'type'), ({}, {'steps': 0}, b'steps'),
                           ({}, {'steps': 65}, b'steps'), ({}, {'eps': 0.0}, b'eps'), ({'rows': 0}, {}, b'sides'),
                           ({'cols': 262145}, {}, b'sides'), ({'count': 0}, {}, b'sides'), ({'count': 1 << 25}, {}, b'too large'),
                           ({'g': None}, {}, b'null'), ({'w': None}, {}, b'null'), ({}, {'a': 50.0}, b'polynomial'),
                           ({}, {'a': float('nan')}, b'polynomial'), ({}, {'a': 0.0, 'b': 0.0, 'c': 0.0}, b'polynomial'),
                           ({'rows': 100, 'cols': 100}, {}, b'work')):
        assert lib.nfi_ortho(ctypes.byref(args(item, **kw)), None) == -1, (item, kw)
        assert word in lib.nfi_last_error(), (item, kw, lib.nfi_last_error())


def test_ortho_work_is_that_of_the_largest_launch():
    lib = _lib.load()

    def bytes_of(shapes):
        arr = (_lib.NfiOrthoItem * len(shapes))(*[_lib.NfiOrthoItem(16, None, 16, r, c, n, 1.0) for r, c, n in shapes])
        return lib.nfi_ortho_work_bytes(arr, len(shapes))

    assert bytes_of([(64, 64, 5), (15, 512, 32), (512, 15, 1)]) == 0
    # X twice, A and Q in pairs of halves of 256 x 384 and 256 x 256, and at most 8 partial tiles of 128 x 128 for each of 3
    one = bytes_of([(200, 300, 1)])
    plain = 2 * 256 * 384 * 4 + 2 * 256 * 256 * 4
    assert plain <= one <= plain + 8 * 3 * 128 * 128 * 4 + 4096
    assert bytes_of([(300, 200, 1)]) == one and bytes_of([(64, 64, 1), (200, 300, 1)]) == one
    # a launch holds 32: the largest of them counts
    assert bytes_of([(200, 300, 1)] * 32) >= 32 * plain
    assert bytes_of([(200, 300, 1)] * 33) == bytes_of([(200, 300, 1)] * 32)
    assert bytes_of([(128, 128, 1)] * 32 + [(2000, 3000, 1)]) == bytes_of([(2000, 3000, 1)])


def test_muon_refuses_vectors_and_repeated_parameters():
    """In the constructor and for groups that come later; a refused group is not kept."""
    from nfi import optim
    a, b = (torch.nn.Parameter(torch.zeros(3, 4)) for _ in range(2))
    vector = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match='two or more dimensions'):
        optim.Muon([a, vector])
    with pytest.raises(ValueError, match='twice'), pytest.warns(UserWarning):
        optim.Muon([a, a])
    o = optim.Muon([a])
    with pytest.raises(ValueError, match='two or more dimensions'):
        o.add_param_group({'params': [vector]})
    with pytest.raises(ValueError, match='twice'), pytest.warns(UserWarning):
        o.add_param_group({'params': [b, b]})
    with pytest.raises(ValueError):
        o.add_param_group({'params': [a]})
    assert len(o.param_groups) == 1
    o.add_param_group({'params': [b], 'lr': 0.5})
    assert len(o.param_groups) == 2 and o.param_groups[1]['lr'] == 0.5


def test_ortho_work_refuses_what_the_call_refuses():
    """A caller of several calls in a row can size them all, and hears of a refused matrix, before the first one runs."""
    lib = _lib.load()
    for shape, word in (((0, 4, 1), b'sides'), ((4, 262145, 1), b'sides'), ((4, 4, 0), b'sides'), ((4, 4, 1 << 24), b'too large'),
                        ((262144, 262144, 4), b'too large')):
        arr = (_lib.NfiOrthoItem * 2)(_lib.NfiOrthoItem(16, None, 16, 200, 300, 1, 1.0), _lib.NfiOrthoItem(16, None, 16, *shape, 1.0))
        assert lib.nfi_ortho_work_bytes(arr, 2) == -1 and word in lib.nfi_last_error(), shape
    assert lib.nfi_ortho_work_bytes(arr, 1) > 0


def test_muon_refuses_a_first_step_in_a_capture(monkeypatch):
    """Before any parameter is stepped, those of earlier groups too, and without leaving a momentum behind."""
    a, b = (torch.nn.Parameter(torch.ones(3, 4)) for _ in range(2))
    o = optim.Muon([{'params': [a]}, {'params': [b]}])
    o.state[a]['momentum_buffer'] = torch.zeros(3, 4)
    a.grad, b.grad = torch.ones(3, 4), torch.ones(3, 4)
    stepped = []
    monkeypatch.setattr(optim, '_op', lambda name: lambda params, *rest: stepped.extend(params))
    monkeypatch.setattr(optim, '_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='before the capture'):
        o.step()
    assert not stepped and 'momentum_buffer' not in o.state.get(b, {})
    b.grad = None
    o.step()                     # (a parameter without a gradient has no part in it)
    assert stepped == [a]
    b.grad = torch.ones(3, 4)
    monkeypatch.setattr(optim, '_capturing', lambda: False)
    o.step()
    assert stepped == [a, a, b] and float(o.state[b]['momentum_buffer'].abs().max()) == 0


@pytest.fixture
def plain_bank(monkeypatch):
    """A bank of three mappers on the CPU, its two operators in torch."""
    from nfi import viewdir

    def linear(x, weight, offsets, bias=None):
        y = x.new_zeros((x.shape[0], weight.shape[1]))
        for e in range(weight.shape[0]):
            r = slice(int(offsets[e]), int(offsets[e + 1]))
            y[r] = x[r] @ weight[e].t() + (0 if bias is None else bias[e])
        return y

    def norm(h, residual, gate, weight, bias, *, slope, scale, eps):
        assert weight.shape[0] >= 1
        n = torch.nn.functional.layer_norm(h, h.shape[-1:], eps=eps).view(weight.shape[0], -1, h.shape[-1])
        u = torch.nn.functional.leaky_relu(n * weight[:, None] + bias[:, None], slope).view(h.shape)
        return scale * (u + (0 if residual is None else residual))

    monkeypatch.setattr(viewdir, 'grouped_linear', linear)
    monkeypatch.setattr(viewdir, 'residual_norm', norm)
    torch.manual_seed(0)
    mappers = [viewdir.ViewDirectionMapper(10) for _ in range(3)]
    for m in mappers:
        for k in range(1, 5):
            with torch.no_grad():
                getattr(m, f'norm{k}').weight.add_(torch.randn(64) * 0.1)
                getattr(m, f'norm{k}').bias.add_(torch.randn(64) * 0.1)
    return viewdir.ViewDirectionMapperBank(mappers)


@pytest.mark.parametrize('which', [[0, 1, 2], [1, 0, 1], [2, 2, 0, 1], [1]])
def test_bank_gives_each_image_its_own_mapper(plain_bank, which):
    from nfi.viewdir import viewdir_trunk
    v = torch.nn.functional.normalize(torch.randn((len(which), 5, 3)), dim=-1)
    x = plain_bank(v, torch.tensor(which))
    for i, m in enumerate(which):
        torch.testing.assert_close(x[i], viewdir_trunk(plain_bank.mappers[m], v[i].unsqueeze(-2)).squeeze(-2), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('which', [[3, 1, 0], [-1, 2, -5], [7]])
def test_bank_leaves_out_images_of_no_mapper(plain_bank, which):
    from nfi.viewdir import viewdir_trunk
    v = torch.nn.functional.normalize(torch.randn((len(which), 5, 3)), dim=-1)
    x = plain_bank(v, torch.tensor(which))
    for i, m in enumerate(which):
        want = viewdir_trunk(plain_bank.mappers[m], v[i].unsqueeze(-2)).squeeze(-2) if 0 <= m < 3 else torch.zeros(5, 32)
        torch.testing.assert_close(x[i], want, rtol=1e-5, atol=1e-5)


def test_bank_refuses_mappers_that_differ():
    """In a gain, a bias, a norm's eps, a slope or a width: one launch takes the first mapper's for all."""
    from nfi.viewdir import ViewDirectionMapper, ViewDirectionMapperBank

    def change(f):
        m = ViewDirectionMapper(10)
        f(m)
        return m

    for f, word in ((lambda m: setattr(m.fc2, 'weight_gain', 0.5), 'fc2'), (lambda m: setattr(m.fc5, 'bias_gain', 0.5), 'fc5'),
                    (lambda m: setattr(m.fc0, 'bias', None), 'fc0'), (lambda m: setattr(m.norm3, 'eps', 1e-6), 'norm3'),
                    (lambda m: setattr(m.relu, 'negative_slope', 0.1), 'LeakyReLU'),
                    (lambda m: setattr(m, 'relu', torch.nn.ReLU()), 'LeakyReLU'), (lambda m: setattr(m.norm1, 'bias', None), 'norm1'),
                    (lambda m: setattr(m, 'fc6', type(m.fc6)(64, 16)), 'fc6')):
        with pytest.raises(ValueError, match=word):
            ViewDirectionMapperBank([ViewDirectionMapper(10), change(f)])
    with pytest.raises(ValueError, match='no mappers'):
        ViewDirectionMapperBank([])
    ViewDirectionMapperBank([ViewDirectionMapper(10), ViewDirectionMapper(4)])   # (the output layers are not the bank's)


@pytest.mark.parametrize('images,rays', [(0, 5), (3, 0), (0, 0)])
def test_bank_of_an_empty_batch(plain_bank, images, rays):
    v = torch.zeros((images, rays, 3), requires_grad=True)
    x = plain_bank(v, torch.zeros((images,), dtype=torch.int64))
    assert x.shape == (images, rays, 32)
    gv, gw = torch.autograd.grad(x.sum(), [v, plain_bank.mappers[0].fc1.weight])
    assert gv.shape == v.shape and float(gw.abs().max()) == 0


@pytest.fixture
def fake():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        yield mode


def shapes_of_calls(device, backward):
    """Every operator on tensors of `device` without memory: shapes, types and devices of what it gives."""
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, device=device, dtype=dtype, requires_grad=dtype != torch.int64)

    def like(got, want):
        for a, b in zip(got, want):
            assert (a.shape, a.dtype, a.device) == (b.shape, b.dtype, b.device)

    def grads(out, leaves, given):
        if backward:
            like(torch.autograd.grad(out, leaves, given), leaves)
    h, res, gate, w, b, w2, b2 = empty(2, 3, 40), empty(2, 3, 40), empty(2, 40, dtype=torch.float32), *(empty(40) for _ in range(4))
    x, y = norms.residual_norm(h, res, gate, w, b, next_weight=w2, next_bias=b2, next_norm='rms')
    like([x, y], [h, h])
    grads([x, y], [h, res, gate, w, b, w2, b2], [h, h])
    x, y = norms.residual_norm(h, None, None, w, next_norm='layer')
    grads([x], [h, w], [h])
    x = norms.residual_norm(h, res)
    like([x], [h])
    grads([x], [res], [h])
    empties = norms.residual_norm(empty(0, 40), weight=w)
    like([empties], [empty(0, 40)])
    grads([empties], [w], [empty(0, 40)])
    with torch.no_grad():
        like([norms.residual_norm(h)], [h])

    x, w, bias, off = empty(50, 24), empty(3, 16, 24), empty(3, 16), empty(4, dtype=torch.int64)
    y = grouped.grouped_linear(x, w, off, bias)
    like([y], [empty(50, 16)])
    grads([y], [x, w, bias], [y])
    grads([grouped.grouped_linear(x, w, off)], [w], [empty(50, 16)])

    u = empty(2, 30, 20)
    like([optim.orthogonalize(u), optim.orthogonalize(u.transpose(1, 2))], [u, u.transpose(1, 2)])


def test_traced_calls_give_shapes(fake):
    """Through the Meta kernels, with no launch (here there is no device that could take one)."""
    shapes_of_calls('cuda', False)


def test_meta_tensors_give_shapes_and_gradients():
    shapes_of_calls('meta', True)


def test_traced_calls_are_checked(fake):
    """What a call refuses it refuses in a trace too."""
    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, device='cuda', dtype=dtype)
    for f, word in ((lambda: norms.residual_norm(empty(4, 8), empty(4, 9)), 'residual'),
                    (lambda: norms.residual_norm(empty(4, 8), gate=empty(3, 8)), 'gate'),
                    (lambda: norms.residual_norm(empty(4, 8), weight=empty(2, 8), gate=empty(4, 8)), 'groups of parameters'),
                    (lambda: grouped.grouped_linear(empty(4, 8), empty(2, 5, 8), empty(2, dtype=torch.int32)), 'offsets'),
                    (lambda: optim.orthogonalize(empty(8)), 'matrices')):
        with pytest.raises((RuntimeError, ValueError), match=word):
            f()


def test_traced_steps(fake):
    """Muon's step over tensors without memory: its state's shapes, the checks of every parameter, and empty parameters, which
    divide nothing."""
    def param(*shape, dtype=torch.float32):
        p = torch.nn.Parameter(torch.empty(shape, device='cuda', dtype=dtype))
        p.grad = torch.empty_like(p)
        return p
    ps = [param(6, 4, 3, 3), param(0, 3), param(8, 8, dtype=torch.bfloat16)]
    o = optim.Muon(ps)
    o.step()
    assert o.state[ps[2]]['momentum_buffer'].dtype == torch.float32 and o.state[ps[0]]['momentum_buffer'].shape == ps[0].shape
    from nfi import torch_ops

    def step(shapes, batched):
        ts = [torch.empty(s, device='cuda') for s in shapes]
        torch_ops.op('muon_step')(ts, [torch.empty_like(t) for t in ts], [torch.empty_like(t) for t in ts], batched, 0.1, 0.9, 0.0, True, 5,
                                  *optim.QUINTIC, 1e-7)
    step([(0, 3), (3, 0), (0, 0), (4, 0, 3), (5, 6)], False)
    step([(2, 0, 4), (0, 3, 4), (2, 3, 0), (2, 3, 4)], True)
    with pytest.raises(ValueError, match='sides'):
        step([(5, 6), (2, 300000)], False)
    with pytest.raises(RuntimeError, match='dense gradients'):
        torch_ops.op('muon_step')([torch.empty(8, device='cuda')], [torch.empty(8, device='cuda')], [torch.empty(8, device='cuda')], False, 0.1,
                                  0.9, 0.0, True, 5, *optim.QUINTIC, 1e-7)


def test_no_tensors_are_no_step():
    from nfi import torch_ops
    torch_ops.op('muon_step')([], [], [], False, 0.1, 0.9, 0.0, True, 5, *optim.QUINTIC, 1e-7)


@pytest.mark.parametrize('affine', [0, 1])
@pytest.mark.parametrize('width,workgroups', [(24, 512), (512, 512), (513, 768), (1024, 768), (1025, 512), (2048, 512), (2049, 256), (8192, 256)])
def test_resnorm_work_holds_every_workgroup_of_each_width(width, workgroups, affine):
    """The plan (restated) with the workgroups that a width takes, for every number of rows one may hold."""
    lib = _lib.load()
    for rows, groups in [(1, 0), (1, 1), (7, 7), (10 ** 6, 0), (10 ** 6, 2), (4096, 512), (4096, 2048), (511 * 3, 511), (769 * 5, 769), (255 * 9, 255),
                         (257 * 2, 257), (768, 768), (3 * 10 ** 5, 300)]:
        for slots in (1, 4, 8, 16, 32):
            g = groups if groups and (groups < rows or affine) else 1
            splits = min(max(1, workgroups // g), -(-(rows // g) // slots))
            segments = g * splits
            per = 1 if splits > 1 else -(-segments // workgroups)
            assert lib.nfi_resnorm_work_bytes(rows, groups, affine, width) >= -(-segments // per) * 5 * width * 4, (rows, groups, slots)


@pytest.mark.parametrize('groups', [0, 2, 4])
def test_resnorm_backward_refuses_a_gradient_of_no_gate(groups):
    lib = _lib.load()
    one = ctypes.c_void_p(16)
    a = _lib.NfiResnormArgs()
    a.h = a.x = a.stats = a.work = a.gx = a.dh = a.dgate = one
    a.rows, a.width, a.groups, a.norm, a.eps = 4, 8, groups, 1, 1e-5
    assert lib.nfi_resnorm_backward(ctypes.byref(a), None) == -1 and b'without a gate' in lib.nfi_last_error()
