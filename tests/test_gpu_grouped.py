"""nfi.grouped.grouped_linear on the device against the products of each group in 64 bits: every type, ragged and empty
groups, rows of no group, widths that are no multiple of anything, a single row to many, and the gradients.

Tolerances.  u = 2^-24, e = eps(type) / 2 (the one rounding of an output).  A 32-bit sum of L products p is off by at
most (L + 1) u sum |p| (any order); products of 16-bit values are exact in 32 bits, and those of 32-bit values round once.  The
test allows e |ref| + (L + 2) u sum |p|, with sum |p| from the operands' magnitudes in 64 bits."""

import pytest
import torch

from nfi import grouped

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(sizes, k, n, dtype, seed, bias=True, before=0, behind=0, idx=torch.int32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = before + sum(sizes) + behind
    off = [before]
    for s in sizes:
        off.append(off[-1] + s)

    def rnd(*shape):
        return torch.randn(shape, device=DEV, generator=g).to(dtype)
    return (rnd(rows, k).requires_grad_(), rnd(len(sizes), n, k).requires_grad_(),
            torch.tensor(off, device=DEV, dtype=idx), rnd(len(sizes), n).requires_grad_() if bias else None, rnd(rows, n), off)


def reference(x, w, off, b, gy):
    """Outputs and gradients in 64 bits, each with the sum of magnitudes and length of its sums."""
    x, w, gy = x.detach().double(), w.detach().double(), gy.double()
    y, ym = torch.zeros_like(gy), torch.zeros_like(gy)
    gx, gxm = torch.zeros_like(x), torch.zeros_like(x)
    gw, gwm = torch.zeros_like(w), torch.zeros_like(w)
    gb, gbm = (torch.zeros(w.shape[:2], device=DEV, dtype=torch.float64) for _ in range(2))
    for e in range(w.shape[0]):
        r = slice(off[e], off[e + 1])
        y[r], ym[r] = x[r] @ w[e].T, x[r].abs() @ w[e].abs().T
        if b is not None:
            y[r] += b[e].detach().double()
            ym[r] += b[e].detach().double().abs()
        gx[r], gxm[r] = gy[r] @ w[e], gy[r].abs() @ w[e].abs()
        gw[e], gwm[e] = gy[r].T @ x[r], gy[r].abs().T @ x[r].abs()
        gb[e], gbm[e] = gy[r].sum(0), gy[r].abs().sum(0)
    longest = max(off[e + 1] - off[e] for e in range(w.shape[0]))
    return [(y, ym, x.shape[1] + 1), (gx, gxm, w.shape[1]), (gw, gwm, longest), (gb, gbm, longest)]


def near(got, ref, dtype):
    value, mags, length = ref
    e = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tol = e * value.abs() * (1 + 2 ** -7) + (length + 2) * U * mags + torch.finfo(dtype).smallest_normal
    worst = float(((got.double() - value).abs() / tol).max())
    assert worst <= 1, (tuple(got.shape), worst)


CASES = [  # sizes, k, n, before, behind
    ([1], 1, 1, 0, 0),
    ([3, 0, 2], 5, 7, 1, 2),
    ([64, 0, 65, 1], 64, 64, 0, 0),
    ([130, 127, 128], 32, 96, 0, 5),
    ([500, 13, 0, 260], 200, 130, 3, 0),
    ([1, 2, 0, 1] * 20, 48, 72, 0, 0),
    ([2000, 700], 100, 33, 0, 129),
    ([700], 64, 260, 140, 0),
    ([300, 301], 513, 257, 0, 0),
    ([0, 0, 0], 16, 24, 4, 4),
    ([40] * 70, 24, 8, 0, 0),
    ([5000, 3000], 64, 64, 0, 0),
]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{len(c[0])}g{sum(c[0])}r{c[1]}to{c[2]}')
def test_values_and_gradients(case, dtype):
    sizes, k, n, before, behind = case
    x, w, offsets, b, gy, off = make(sizes, k, n, dtype, k * 7 + n, True, before, behind)
    y = grouped.grouped_linear(x, w, offsets, b)
    got = [y.detach()] + list(torch.autograd.grad(y, [x, w, b], gy))
    for a, ref in zip(got, reference(x, w, off, b, gy)):
        near(a, ref, dtype)
    for a in got[:2]:
        assert float(a[:before].abs().sum()) == 0 and float(a[a.shape[0] - behind:].abs().sum()) == 0
    for e, s in enumerate(sizes):
        if s == 0:
            assert float(got[2][e].abs().sum()) == 0 and float(got[3][e].abs().sum()) == 0
    # in place of a sum whose order changes, the same bits again
    y2 = grouped.grouped_linear(x, w, offsets.long(), b)
    again = [y2.detach()] + list(torch.autograd.grad(y2, [x, w, b], gy))
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize('dtype', TYPES)
def test_unaligned_and_strided_operands(dtype):
    """Views whose first element is not at 16 bytes, transposed and sliced tensors, no bias."""
    x, w, offsets, _, gy, off = make([50, 60], 40, 24, dtype, 1, False)
    flat = torch.zeros((x.numel() + 1,), device=DEV, dtype=dtype)
    flat[1:] = x.detach().flatten()
    xs = flat[1:].view(x.shape)
    wt = w.detach().transpose(1, 2).contiguous().transpose(1, 2)
    y = grouped.grouped_linear(xs, wt, offsets)
    assert torch.equal(y, grouped.grouped_linear(x, w, offsets))
    wide = torch.zeros((110, 80), device=DEV, dtype=dtype)
    wide[:, 8:48] = x.detach()
    assert torch.equal(y, grouped.grouped_linear(wide[:, 8:48], w, offsets).detach())
    gs = torch.zeros((110, 48), device=DEV, dtype=dtype)
    gs[:, ::2] = gy
    yy = grouped.grouped_linear(x, w, offsets)
    a = torch.autograd.grad(yy, [x, w], gs[:, ::2], retain_graph=True)
    b = torch.autograd.grad(yy, [x, w], gy)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradient_against_differences():
    """The product is linear in each argument: a difference of any step is the gradient, up to 32-bit rounding."""
    x, w, offsets, b, gy, off = make([9, 0, 14], 20, 12, torch.float32, 2)

    def value(x, w, b):
        return float((grouped.grouped_linear(x, w, offsets, b).detach().double() * gy.double()).sum())
    y = grouped.grouped_linear(x, w, offsets, b)
    grads = torch.autograd.grad(y, [x, w, b], gy)
    for i, d in enumerate(grads):
        way = torch.randn_like(d)
        args = [v.detach() for v in (x, w, b)]
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + way, args[i] - way
        want = float((d.double() * way.double()).sum())
        mags = 2 * float(y.abs().sum() * gy.abs().max()) + abs(want) + float(d.abs().sum() * way.abs().max())
        assert abs((value(*hi) - value(*lo)) / 2 - want) <= 64 * U * mags


def test_infinities_stay_in_their_rows():
    x, w, offsets, b, gy, off = make([40, 30], 64, 32, torch.float32, 3)
    bad = x.detach().clone()
    bad[7, 5], bad[50, 0] = float('nan'), float('inf')
    y, z = grouped.grouped_linear(x, w, offsets, b).detach(), grouped.grouped_linear(bad, w, offsets, b).detach()
    rest = [i for i in range(70) if i not in (7, 50)]
    assert torch.equal(y[rest], z[rest]) and bool(torch.isnan(z[7]).all()) and not bool(torch.isfinite(z[50]).any())
    # a head that no row goes through may hold anything
    x, w, offsets, b, gy, off = make([40, 0, 30], 64, 32, torch.bfloat16, 4)
    w2 = w.detach().clone()
    w2[1] = float('nan')
    assert torch.equal(grouped.grouped_linear(x, w, offsets, b), grouped.grouped_linear(x, w2, offsets, b))


def test_offsets_out_of_range_count_as_the_ends():
    x, w, _, b, _, _ = make([40, 30], 32, 32, torch.float32, 5)
    a = grouped.grouped_linear(x, w, torch.tensor([-9, 40, 999], device=DEV), b)
    want = grouped.grouped_linear(x, w, torch.tensor([0, 40, 70], device=DEV), b)
    assert torch.equal(a, want)


def test_streams_empty_and_refusals():
    x, w, offsets, b, gy, off = make([40, 30], 32, 32, torch.float32, 6)
    y = grouped.grouped_linear(x, w, offsets, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = grouped.grouped_linear(x, w, offsets, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)
    e = torch.zeros((0, 32), device=DEV, requires_grad=True)
    out = grouped.grouped_linear(e, w, torch.zeros((3,), device=DEV, dtype=torch.int32), b)
    gx, gw, gb = torch.autograd.grad(out.sum(), [e, w, b])
    assert out.shape == (0, 32) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0
    for bad, word in (((x, w, offsets[:2], b), 'offsets'), ((x, w, offsets.float(), b), 'offsets'), ((x, w[:, :, :31], offsets, b), 'wanted'),
                      ((x, w, offsets, b[:, :5]), 'bias'), ((x, w.half(), offsets, b), 'one type'), ((x.double(), w.double(), offsets, None), 'float32'),
                      ((x[0], w, offsets, b), 'wanted'), ((x, w, offsets.cpu(), b), 'cpu')):
        with pytest.raises((RuntimeError, ValueError), match=word):
            grouped.grouped_linear(*bad)


def test_captured_and_replayed():
    """Forward and backward captured, replayed with other rows and other offsets, between eager calls."""
    x, w, offsets, b, gy, off = make([400, 100, 12], 64, 96, torch.float32, 7)

    def step():
        y = grouped.grouped_linear(x, w, offsets, b)
        return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], gy))

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
    for at in ([0, 10, 20, 512], [0, 0, 512, 512], [5, 6, 300, 310]):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            offsets.copy_(torch.tensor(at, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step()))


def alike(got, ref, dtype):
    """The same infinities and the same places without a number as the formula in 64 bits; the rest within the tolerance."""
    value, mags, length = ref
    got64 = got.double()
    assert torch.equal(torch.isnan(got64), torch.isnan(value))
    inf = torch.isinf(value)
    assert torch.equal(torch.isinf(got64), inf) and torch.equal(got64[inf], value[inf])
    keep = torch.isfinite(value)
    near(got[keep], (value[keep], mags[keep], length), dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('k,n', [(40, 24), (64, 64), (200, 130), (513, 257)])
def test_infinities_and_large_values_are_those_of_the_formula(k, n, dtype):
    """An infinity in a row, a weight or a gradient gives the sums that hold it (infinities of its sign; no number where it
    meets its opposite or a zero), and values next to the type's largest, which 16 bits of their leading part may not hold, give their
    products.  What holds none of them keeps its bits."""
    x, w, offsets, b, gy, off = make([300, 0, 150], k, n, dtype, k + n)
    clean_y = grouped.grouped_linear(x, w, offsets, b)
    clean = [clean_y.detach()] + list(torch.autograd.grad(clean_y, [x, w, b], gy))
    big = torch.finfo(dtype).max
    with torch.no_grad():
        x[7, 5], x[9, 0], x[9, 1], x[40, 3] = float('inf'), float('inf'), float('-inf'), float('-inf')
        x[301, 2] = big * 2.0 ** -6      # (times a weight and added: far from the end, but for rounding up of its leading part)
        x[302, :] = 0
        x[302, 4] = big
        w[2, :, 4] *= 2.0 ** -8
        w[2, 3, 6] = float('inf')        # (row 302 holds a zero there)
        gy[11, 1], gy[350, 2] = float('-inf'), big * 2.0 ** -6
    y = grouped.grouped_linear(x, w, offsets, b)
    got = [y.detach()] + list(torch.autograd.grad(y, [x, w, b], gy))
    refs = reference(x, w, off, b, gy)
    # a value past the type's range is an infinity in it; next to the range's end it may be either, and is not looked at
    for a, (value, mags, length) in zip(got, refs):
        over = value.abs() >= big * (1 + 2.0 ** -6)
        either = torch.isfinite(value) & ~over & (value.abs() + 2.0 ** -7 * mags >= big)
        value = torch.where(over, value.sign() * float('inf'), value).masked_fill(either, 0.0)
        alike(a.masked_fill(either, 0.0), (value, mags, length), dtype)
    rest = [i for i in range(300) if i not in (7, 9, 40)]
    assert torch.equal(got[0][rest], clean[0][rest])
    rest = [i for i in range(300) if i != 11]
    assert torch.equal(got[1][rest], clean[1][rest])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes,before,behind', [([1] * 200, 1, 1), ([129] * 9, 129, 1), ([1, 127, 128, 129, 0, 1], 1, 127), ([2] * 62, 0, 3),
                                                 ([0] * 70 + [1], 0, 0), ([0] * 63 + [5] + [0] * 64 + [200], 257, 129)])
def test_every_row_of_any_division_is_written(sizes, before, behind, dtype):
    """As many row tiles as a division can need, each with few rows: no row of y or gx keeps what its memory held."""
    x, w, offsets, b, gy, off = make(sizes, 40, 72, dtype, len(sizes), True, before, behind)
    for shape in (gy.shape, x.shape):
        junk = [torch.full(shape, float('nan'), device=DEV, dtype=dtype) for _ in range(3)]
        del junk
    y = grouped.grouped_linear(x, w, offsets, b)
    got = [y.detach()] + list(torch.autograd.grad(y, [x, w, b], gy))
    for a, ref in zip(got, reference(x, w, off, b, gy)):
        near(a, ref, dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('sizes,k,n', [([3, 0, 2], 16, 24), ([700, 1300], 48, 40), ([40000], 8, 130), ([5000, 0, 3000, 100], 64, 64), ([300] * 30, 33, 257)])
def test_each_gradient_alone(sizes, k, n, dtype):
    """The gradient of one argument without the others' (the bias has a kernel of its own then, its rows split where they are
    many): those of x and the weight are the same bits as together, the bias's within its sum's rounding."""
    x, w, offsets, b, gy, off = make(sizes, k, n, dtype, k + n, True, 2, 5)
    y = grouped.grouped_linear(x, w, offsets, b)
    refs = reference(x, w, off, b, gy)[1:]
    together = torch.autograd.grad(y, [x, w, b], gy, retain_graph=True)
    for i, leaf in enumerate((x, w, b)):
        alone, = torch.autograd.grad(y, [leaf], gy, retain_graph=True)
        near(alone, refs[i], dtype)
        again, = torch.autograd.grad(y, [leaf], gy, retain_graph=True)
        assert torch.equal(alone, again) and (leaf is b or torch.equal(alone, together[i]))
    pair = torch.autograd.grad(y, [x, b], gy)
    near(pair[1], refs[2], dtype)
    assert torch.equal(pair[0], together[0])
    # without a gradient of x and the weight there is none to make
    with torch.no_grad():
        xd, wd = x.clone(), w.clone()
    alone, = torch.autograd.grad(grouped.grouped_linear(xd, wd, offsets, b), [b], gy)
    near(alone, refs[2], dtype)


@pytest.mark.parametrize('ex,ew', [(-100, 90), (-110, 100), (-120, 100), (-126, 110), (90, -126)])
def test_values_next_to_the_smallest(ex, ew):
    """32-bit values are three 16-bit parts with bf16's range, whose smallest step is 2^-133: below 2^-110 that is what a value is
    held to, beside its own 24 bits (half a step of each operand, with the other's magnitude)."""
    x, w, offsets, b, gy, off = make([70, 30], 96, 40, torch.float32, 9, False)
    with torch.no_grad():
        x.mul_(2.0 ** (ex / 2)).mul_(2.0 ** (ex / 2))
        w.mul_(2.0 ** (ew / 2)).mul_(2.0 ** (ew / 2))
    y = grouped.grouped_linear(x, w, offsets)
    got = [y.detach()] + list(torch.autograd.grad(y, [x, w], gy))
    step = 2.0 ** -133
    ones = lambda t: torch.full_like(t.detach(), step, dtype=torch.float64)
    for i, (a, ref) in enumerate(zip(got, reference(x, w, off, None, gy))):
        value, mags, length = ref
        held = {'x': reference(ones(x), w, off, None, gy), 'w': reference(x, ones(w), off, None, gy), 'gy': reference(x, w, off, None, ones(gy))}
        lost = sum(held[k][i][1] for k in (('x', 'w'), ('gy', 'w'), ('gy', 'x'))[i])   # (its two factors)
        tol = (length + 2) * U * mags + lost + torch.finfo(torch.float32).smallest_normal
        assert float(((a.double() - value).abs() / tol).max()) <= 1, i
