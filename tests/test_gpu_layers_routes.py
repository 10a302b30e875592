"""Layers large enough for the tensor cores' tiles: arrays that TMA reads, arrays that become parts, and rows that are gathered,
each at odd sizes, layouts, types of parameters and values, against 64-bit forms (layer_oracle)."""
import ctypes

import pytest

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from test_gpu_layers import ACTIVATIONS, BF16, F16, F32, KINDS, check_gradient, check_linear, close, made, same_bits, update, within  # noqa: E402

pytestmark = pytest.mark.gpu
CODES = {F32: 0, BF16: 1, F16: 2}


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def workspace(engine, x, weight):
    """Bytes of the forward's workspace for arrays as they are: parts take some, arrays that are read in place none."""
    size = ctypes.c_size_t()
    assert engine.lib.cpde_linear_workspace(CODES[x.dtype], x.data_ptr(), x.stride(-2), x.numel() // x.shape[-1], x.shape[-1],
                                            weight.shape[0], weight.data_ptr(), weight.stride(0), ctypes.byref(size)) == native.OK
    return size.value


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('activation', ACTIVATIONS)
@pytest.mark.parametrize('points,inputs,outputs', [(1500, 200, 600), (1501, 264, 603), (1029, 1030, 130)])
def test_ragged_tiles(engine, kind, activation, points, inputs, outputs):
    """Tiles whose warps have lanes behind the last row and columns behind the last one, and functions with branches."""
    x, weight = made(1, points, inputs, dtype=kind), made(2, outputs, inputs, dtype=kind, scale=2 * inputs ** -0.5)
    bias, residual = made(3, outputs, dtype=kind), made(4, points, outputs, dtype=kind)
    _, z = check_linear(engine, x, weight, bias, activation, residual)
    check_gradient(engine, made(5, points, outputs, dtype=kind), x, weight, bias, activation, None if activation == 'linear' else z)


def around(t, left, right, above=0):
    """The same rows inside of a larger array, `left` and `right` further elements beside them."""
    whole = torch.full((*t.shape[:-2], t.shape[-2] + above, t.shape[-1] + left + right), float('nan'), dtype=t.dtype, device='cuda')
    inside = whole[..., above:, left:left + t.shape[-1]]
    inside.copy_(t)
    return inside


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('left,right', [(8, 8), (16, 32), (0, 8), (3, 5), (4, 0), (1, 0), (2, 0)])
def test_layouts_of_tiles(engine, kind, left, right):
    """Rows with strides between NaNs: whole 16 bytes, which TMA reads where they are, and others, which become parts."""
    points, inputs, outputs = 1500, 208, 600
    x, weight = around(made(6, points, inputs, dtype=kind), left, right, 1), around(made(7, outputs, inputs, dtype=kind, scale=0.1), left, right)
    in_place = kind != F32 and left % 8 == 0 and (left + right) % 8 == 0
    assert (workspace(engine, x, weight) < 2 * weight.numel()) == in_place
    residual, grad = around(made(8, points, outputs, dtype=kind), left, right), around(made(9, points, outputs, dtype=kind), right, left)
    bias = made(10, outputs, dtype=kind)
    _, z = check_linear(engine, x, weight, bias, 'tanh', residual)
    check_gradient(engine, grad, x, weight, bias, 'tanh', around(z, left, right))
    check_gradient(engine, grad, x, weight, bias, 'linear', None)


@pytest.mark.parametrize('kind', KINDS)
def test_other_layouts_of_tiles(engine, kind):
    """Transposed, broadcast and skipped rows, further leading dimensions."""
    x, weight, grad = made(11, 1500, 208, dtype=kind), made(12, 600, 208, dtype=kind, scale=0.1), made(13, 1500, 600, dtype=kind)
    for a, w, g in ((x.t().contiguous().t(), weight.t().contiguous().t(), grad), (x, weight, grad.t().contiguous().t()),
                    (x[:1].expand(1500, 208), weight, grad[:1].expand(1500, 600)),
                    (made(14, 3000, 208, dtype=kind)[::2], weight, made(15, 3000, 600, dtype=kind)[1::2]),
                    (made(16, 15, 200, 208, dtype=kind)[:, ::2], weight, made(17, 15, 200, 600, dtype=kind)[:, 1::2])):
        _, z = check_linear(engine, a, w, None, 'silu', g)
        check_gradient(engine, g, a, w, None, 'silu', z)


# Every width of the loads, one and two slabs, a last tile of few rows, outputs between 65 and 128.
GATHERED = [(40001, 100, 77), (40001, 77, 100), (30000, 48, 128), (30016, 128, 65), (25000, 65, 128), (20099, 126, 100), (40000, 20, 96)]


@pytest.mark.parametrize('points,inputs,outputs', GATHERED)
@pytest.mark.parametrize('gap', [0, 1, 2, 4])
def test_gathered_rows(engine, points, inputs, outputs, gap):
    """FP32 layers whose rows go to the tiles without parts in memory, forward and, without a slope, for the gradient of x."""
    x, weight = around(made(20, points, inputs), gap, 0), around(made(21, outputs, inputs, scale=inputs ** -0.5), 0, gap)
    assert workspace(engine, x, weight) == 0
    bias, residual, grad = made(22, outputs), around(made(23, points, outputs), 0, gap), around(made(24, points, outputs), gap, 0)
    _, z = check_linear(engine, x, weight, bias, 'tanh', residual)
    check_gradient(engine, grad, x, weight, bias, 'linear', None)
    if gap == 0:
        check_gradient(engine, grad, x, weight, None, 'tanh', z)


def test_the_gathered_gradient_takes_no_parts(engine):
    size = ctypes.c_size_t()
    for points, outputs, inputs in GATHERED:  # the sides exchanged
        grad, x, weight = made(25, points, outputs), made(26, points, inputs), made(27, outputs, inputs)
        assert engine.lib.cpde_linear_gradient_workspace(0, grad.data_ptr(), outputs, 1, x.data_ptr(), inputs, points, inputs, outputs,
                                                         weight.data_ptr(), inputs, 1, ctypes.byref(size)) == native.OK
        assert size.value == 0
        whole = operators.linear_gradient(engine, grad, x, weight)
        alone = operators.linear_gradient(engine, grad, x, weight, need=(True, False))
        assert same_bits(whole[0], alone[0]) and alone[1] is None
        within(alone[0], *oracle.linear_gradient(grad, x, weight, 'linear', None)[0])


# Sums of one sign of 16-bit products. The tensor core cuts 2048 terms toward zero, which oracle.chain bounds (3.5e-5); what is
# added of them, and the joined splits, is rounded to nearest, at most 2^-24 each time.
def one_sign(terms):
    return oracle.chain(2048, BF16) + (terms / 2048 + 8) * oracle.E


@pytest.mark.parametrize('kind', [BF16, F16])
@pytest.mark.parametrize('points,inputs,outputs', [(1 << 18, 1024, 1024), (100001, 520, 1032), (1 << 17, 2048, 256)])
def test_long_sums_of_one_sign(engine, kind, points, inputs, outputs):
    """The gradient of the weights over many points whose terms have one sign, as behind a sigmoid, in FP32."""
    x, grad = (torch.sigmoid(made(120 + i, points, n)).to(kind) for i, n in enumerate((inputs, outputs)))
    _, dweight, _ = operators.linear_gradient(engine, grad, x, torch.zeros((outputs, inputs), dtype=kind, device='cuda'),
                                              need=(False, True), dtype=F32)
    want = sum(grad[a:a + 32768].double().t() @ x[a:a + 32768].double() for a in range(0, points, 32768))
    assert ((dweight.double() - want).abs() <= (one_sign(points) + 2 * oracle.E) * want).all()


@pytest.mark.parametrize('kind', [BF16, F16])
@pytest.mark.parametrize('points,inputs,outputs', [(2048, 65536, 512), (600, 9000, 1024), (40, 1 << 20, 16)])
def test_long_rows_of_one_sign(engine, kind, points, inputs, outputs):
    x, weight = (torch.sigmoid(made(122 + i, n, inputs)).to(kind) for i, n in enumerate((points, outputs)))
    y, _ = operators.linear(engine, x / 64, weight)
    want = sum((x / 64)[:, a:a + 65536].double() @ weight[:, a:a + 65536].double().t() for a in range(0, inputs, 65536))
    within(y, want, (one_sign(inputs) + oracle.ROUNDING[kind] * (1 + 2 * one_sign(inputs))) * want)


# FP32 against 64 bits in norm, on the routes of three parts. Parts are exact (3 x 8 bits); left out are products below 2^-25 of
# |x||w|, at random signs. Inside a slab at most 24 times a sum is cut toward zero, by half of 2^-23 of it on average; a slab's sum is
# some sqrt(64) of the result's sqrt(K) terms, and the cuts of the slabs add up at random: 24 * 2^-24 = 1.4e-6 of the result where
# all cuts of a slab fall on its full sum, 0.7e-6 where the sum grows along them. Roundings of 2^-24 between slabs add at random.
# The bound is 1e-6; products of two parts leave 2^-17 |x||w|, 4e-6 of the result (test_layers_bounds_host).
NORM = 1e-6


@pytest.mark.parametrize('points,inputs,outputs', [(1300, 2000, 1000), (1500, 264, 600), (65536, 128, 128), (40001, 100, 77), (129, 4096, 520),
                                                   (2050, 192, 384), (70000, 16, 8)])
@pytest.mark.parametrize('activation', ['linear', 'tanh'])
def test_float32_in_norm(engine, points, inputs, outputs, activation):
    x, weight, bias = made(30, points, inputs), made(31, outputs, inputs, scale=inputs ** -0.5), made(32, outputs)
    grad = made(33, points, outputs)
    y, z = operators.linear(engine, x, weight, bias, activation, keep=True)
    want = oracle.linear(x, weight, bias, activation, None)
    got = operators.linear_gradient(engine, grad, x, weight, bias, activation, z)
    for a, b in zip((y, z, *got), (*want[:2], *(v for v, _ in oracle.linear_gradient(grad, x, weight, activation, z)))):
        assert (a - b).norm() <= NORM * b.norm(), float((a - b).norm() / b.norm())


@pytest.mark.parametrize('kind,points,inputs,outputs', [(F32, 1500, 264, 600), (F32, 40001, 100, 77), (BF16, 1500, 264, 600), (F16, 1500, 264, 600),
                                                        (BF16, 1501, 257, 603), (F16, 1501, 257, 603)])
def test_a_bad_row_stays_in_its_row_of_a_tile(engine, kind, points, inputs, outputs):
    """NaN, infinite and largest values in one point change nothing of the others; the largest value's own row stays right."""
    x, weight = made(40, points, inputs, dtype=kind), made(41, outputs, inputs, dtype=kind, scale=0.1)
    clean, _ = operators.linear(engine, x, weight)
    at = points // 2
    keep = torch.arange(points, device='cuda') != at
    for bad in (float('nan'), float('inf'), torch.finfo(kind).max, -torch.finfo(kind).max):
        x[at, 3] = bad
        got, _ = operators.linear(engine, x, weight)
        assert same_bits(got[keep], clean[keep])
        if bad != bad:
            assert got[at].isnan().all()
        elif bad == float('inf'):
            assert not got[at].isfinite().any()
        else:
            want, _, bound, _ = oracle.linear(x[at:at + 1], weight, None, 'linear', None)
            fits = want.abs() < 0.99 * torch.finfo(kind).max
            assert fits.sum() > 0.9 * outputs
            assert ((got[at].double() - want[0]).abs() <= bound[0])[fits[0]].all()


def test_float32_range_of_tiles(engine):
    """Rows of very different sizes keep the error of FP32 each, up to the largest numbers and down to small ones."""
    scale = torch.tensor([1e-30, 1e-20, 1e-10, 1e-3, 1, 1e5, 1e15, 1e25, 1e36], device='cuda')
    for points, inputs, outputs in ((1503, 264, 600), (40001, 100, 77)):
        x = made(42, points, inputs) * scale.repeat(points // 9 + 1)[:points, None]
        weight = made(43, outputs, inputs, scale=0.1)
        assert (workspace(engine, x, weight) == 0) == (inputs == 100)
        check_linear(engine, x, weight, None, 'linear')
        # Few terms a row, so that the largest numbers' sums stay finite.
        x = torch.full_like(x, torch.finfo(F32).max)
        weight.zero_()
        weight[torch.arange(outputs), torch.arange(outputs) % inputs] = torch.tensor([1.0, 0.5, 1e-30], device='cuda').repeat(outputs // 3 + 1)[:outputs]
        y, _ = operators.linear(engine, x, weight)
        want = x[:1].double() @ weight.double().t()
        assert ((y.double() - want).abs() <= 2.0 ** -22 * want).all()


@pytest.mark.parametrize('kind', [BF16, F16])
@pytest.mark.parametrize('points,inputs,outputs', [(1500, 264, 600), (1501, 257, 603), (20000, 64, 72)])
def test_parameters_of_float32_on_tiles(engine, kind, points, inputs, outputs):
    x, weight, bias = made(50, points, inputs, dtype=kind), made(51, outputs, inputs, dtype=kind, scale=0.1), made(52, outputs)
    grad = made(53, points, outputs, dtype=kind)
    for activation in ('linear', 'sigmoid'):
        _, z = check_linear(engine, x, weight, bias, activation)
        z = None if activation == 'linear' else z
        _, dweight, dbias = check_gradient(engine, grad, x, weight, bias, activation, z, dtype=F32)
        assert dweight.dtype == dbias.dtype == F32
        _, dweight, dbias = operators.linear_gradient(engine, grad, x, weight, bias, activation, z)
        assert dweight.dtype == kind and dbias.dtype == F32


@pytest.mark.parametrize('kind', [BF16, F16])
@pytest.mark.parametrize('points,inputs,outputs', [(1500, 264, 600), (1501, 257, 603), (20000, 64, 72), (70, 40, 24), (4096, 1024, 1024)])
def test_float32_gradients_of_16_bit_layers(engine, kind, points, inputs, outputs):
    """Two numbers of the type hold a term to 2^-16. Cuts of sums of random signs, 2 * 2048 / 16 at most before they are taken out,
    each below 2^-24 of what has been reached on average, leave 1.5e-5; the slope's roundings are some 2^-20. Together below 2^-15:
    terms rounded once to bfloat16 leave 1e-3, to float16 1e-4."""
    x, weight, bias, grad = (made(54 + i, *s, dtype=kind) for i, s in enumerate(((points, inputs), (outputs, inputs), (outputs,), (points, outputs))))
    for activation in ACTIVATIONS[1:]:
        z = operators.linear(engine, x, weight / inputs ** 0.5, bias, activation, keep=True)[1]
        _, dweight, dbias = check_gradient(engine, grad, x, weight, bias, activation, z, dtype=F32)
        dz = grad.double() * oracle.slope(z.double(), activation)
        for got, want in ((dweight, dz.t() @ x.double()), (dbias, dz.sum(0))):
            assert (got.double() - want).norm() <= 2.0 ** -15 * want.norm(), float((got.double() - want).norm() / want.norm())
        alone = operators.linear_gradient(engine, grad, x, weight, None, activation, z, need=(False, True), dtype=F32)[1]
        assert same_bits(alone, dweight)


@pytest.mark.parametrize('kind', [BF16, F16])
def test_float32_gradients_of_bad_values(engine, kind):
    """Infinite terms and those that overflow the type stay infinite."""
    x, weight, grad = (made(58 + i, *s, dtype=kind).abs() for i, s in enumerate(((1500, 264), (600, 264), (1500, 600))))
    z = torch.ones_like(grad)
    grad[7, 3] = float('inf')
    grad[9, 5] = torch.finfo(kind).max  # times a slope of silu above 1, if the type holds no more
    z[9, 5] = 2.0
    _, dweight, _ = operators.linear_gradient(engine, grad, x, weight, None, 'silu', z, need=(False, True), dtype=F32)
    assert (dweight[3] == float('inf')).all()
    assert (dweight[5] == float('inf')).all()
    keep = [i for i in range(600) if i not in (3, 5)]
    assert dweight[keep].isfinite().all()


@pytest.mark.parametrize('kind', KINDS)
def test_needs_on_tiles(engine, kind):
    x, weight, bias, grad = (made(60 + i, *s, dtype=kind) for i, s in enumerate(((1500, 264), (600, 264), (600,), (1500, 600))))
    for activation in ('linear', 'silu'):
        z = None if activation == 'linear' else operators.linear(engine, x, weight, bias, activation, keep=True)[1]
        whole = operators.linear_gradient(engine, grad, x, weight, bias, activation, z)
        for need in ((True, False), (False, True), (False, False)):
            for b in (bias, None):
                got = operators.linear_gradient(engine, grad, x, weight, b, activation, z, need=need)
                for part, want, there in zip(got, whole, (*need, b is not None)):
                    assert (part is None) != there and (part is None or same_bits(part, want))


@pytest.mark.parametrize('kind', KINDS)
def test_captured_tiles(engine, kind):
    """A step of forward, gradient and update in a graph, replayed on other inputs."""
    x, weight, bias, grad = (made(70 + i, *s, dtype=kind) for i, s in enumerate(((1500, 264), (600, 264), (600,), (1500, 600))))
    momentum = torch.zeros_like(weight)

    def step(x):
        y, z = operators.linear(engine, x, weight, bias, 'silu', keep=True)
        dx, dweight, dbias = operators.linear_gradient(engine, grad, x, weight, bias, 'silu', z)
        return (y, dx, dweight, dbias, *operators.muon(engine, weight, dweight, momentum, 0.1))

    held = x.clone()
    step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for seed in (80, 81):
        held.copy_(made(seed, 1500, 264))
        graph.replay()
        for a, b in zip(out, step(held)):
            assert same_bits(a, b)


@pytest.mark.parametrize('kind', KINDS)
def test_autograd_of_tiles(engine, kind):
    """The autograd function with all of its arguments and with fewer."""
    x, weight, bias, grad = (made(90 + i, *s, dtype=kind) for i, s in enumerate(((3, 500, 264), (600, 264), (600,), (3, 500, 600))))
    for arguments in ((x, weight), (x, weight, bias), (x, weight, bias, 'silu'), (x, weight, bias, 'silu', grad)):
        leaves = [a.clone().requires_grad_() if isinstance(a, torch.Tensor) else a for a in arguments]
        operators.Linear.apply(engine, *leaves).backward(grad)
        activation = arguments[3] if len(arguments) > 3 else 'linear'
        b = arguments[2] if len(arguments) > 2 else None
        z = None if activation == 'linear' else operators.linear(engine, x, weight, b, activation, keep=True)[1]
        want = operators.linear_gradient(engine, grad, x, weight, b, activation, z)
        for leaf, part in zip(leaves[:3], want):
            assert same_bits(leaf.grad, part)
        if len(leaves) > 4:
            assert same_bits(leaves[4].grad, grad)


# --- larger matrices ---------------------------------------------------------------

@pytest.mark.parametrize('kind,momentum_kind', [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize('rows,columns', [(300, 515), (515, 300), (700, 384), (257, 1030)])
def test_muon_of_larger_matrices(engine, kind, momentum_kind, rows, columns):
    """Both sides above 256, where steps of 16-bit weights multiply one part: the bounds of the small ones."""
    weight, grad = made(100, rows, columns, dtype=kind), update(101, rows, columns, dtype=kind)
    momentum = update(104, rows, columns, dtype=momentum_kind)
    for nesterov, decay in ((True, 0.0), (False, 0.1)):
        new_weight, new_momentum = operators.muon(engine, weight, grad, momentum, 0.02, 0.9, nesterov, decay)
        m = 0.9 * momentum.double() + 0.1 * grad.double()
        u = 0.9 * m + 0.1 * grad.double() if nesterov else m
        size = 0.9 * momentum.double().abs() + 0.1 * grad.double().abs()
        within(new_momentum, m, (oracle.ROUNDING[momentum_kind] * (1 + 4 * oracle.E) + 4 * oracle.E) * size + oracle.TINY[momentum_kind])
        step = oracle.orthogonalize(u)
        off = (oracle.orthogonalize_modelled(u, kind, step=True) - step).norm()
        s = max(1.0, rows / columns) ** 0.5
        want = (1 - 0.02 * decay) * weight.double() - 0.02 * s * step
        bound = 0.02 * s * (8 * off + 2.0 ** -20 * step.norm()) + (oracle.ROUNDING[kind] + 4 * oracle.E) * want.norm()
        assert (new_weight.double() - want).norm() <= bound
        # The step itself, where the weights are zeros: nothing is left of it to hide behind the weights' rounding.
        alone, _ = operators.muon(engine, torch.zeros_like(weight), grad, momentum, 0.02, 0.9, nesterov, decay)
        want = -0.02 * s * step
        bound = 0.02 * s * (8 * off + 2.0 ** -20 * step.norm()) + (oracle.ROUNDING[kind] + 4 * oracle.E) * want.norm()
        bound += oracle.TINY[kind] * (rows * columns) ** 0.5
        assert (alone.double() - want).norm() <= bound
        w, m = weight.clone(), momentum.clone()
        operators.muon(engine, w, grad, m, 0.02, 0.9, nesterov, decay, inplace=True)
        assert same_bits(w, new_weight) and same_bits(m, new_momentum)


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('shape', [(3, 300, 515), (2, 700, 384), (2, 129, 257), (300, 257, 260)])
def test_orthogonalize_batches_of_larger_matrices(engine, kind, shape):
    x = update(110, *shape, dtype=kind)
    got = operators.orthogonalize(engine, x)
    for at in {0, 1, shape[0] - 1}:
        close(got[at], x[at], kind)
        assert same_bits(got[at], operators.orthogonalize(engine, x[at]))
