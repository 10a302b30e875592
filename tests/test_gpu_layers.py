"""Linear layers, their gradients, orthogonalised matrices and the optimiser step against 64-bit forms of the same formulas
(layer_oracle, which also derives the bounds)."""
import ctypes

import pytest

torch = pytest.importorskip('torch')

import layer_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [F32, BF16, F16]
ACTIVATIONS = ['linear', 'sigmoid', 'tanh', 'silu']


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e


def made(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * scale).to(dtype)


def within(got, want, bound):
    got, want, bound = (t.reshape(want.shape) for t in (got.to(torch.float64), want, bound))
    wrong = ~((got - want).abs() <= bound)
    assert not wrong.any(), (int(wrong.sum()), float((got - want).abs().max()), float(bound.min()))


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check_linear(engine, x, weight, bias, activation, residual=None):
    y, z = operators.linear(engine, x, weight, bias, activation, residual, keep=True)
    assert y.shape == z.shape == (*x.shape[:-1], weight.shape[0]) and y.dtype == z.dtype == x.dtype
    want_y, want_z, bound_y, bound_z = oracle.linear(x, weight, bias, activation, residual)
    within(z, want_z, bound_z)
    within(y, want_y, bound_y)
    again, none = operators.linear(engine, x, weight, bias, activation, residual)
    assert none is None and same_bits(again, y)
    return y, z


def check_gradient(engine, grad, x, weight, bias, activation, z, dtype=None):
    got = operators.linear_gradient(engine, grad, x, weight, bias, activation, z, dtype=dtype)
    again = operators.linear_gradient(engine, grad, x, weight, bias, activation, z, dtype=dtype)
    want = oracle.linear_gradient(grad, x, weight, activation, z, dtype)
    assert got[0].shape == x.shape and got[1].shape == weight.shape
    assert got[0].dtype == x.dtype and got[1].dtype == (dtype or weight.dtype)
    for a, b, (value, bound) in zip(got, again, want):
        if a is None:
            assert bias is None
            continue
        assert same_bits(a, b)
        within(a, value, bound)
    return got


# --- linear layers -----------------------------------------------------------

SIZES = [(1, 1, 1), (2, 3, 5), (1, 64, 64), (7, 1, 130), (130, 7, 1), (64, 128, 64), (129, 65, 257), (257, 48, 128),
         (300, 100, 77), (1, 4096, 520), (16, 1000, 1024), (5, 640, 33), (700, 129, 1), (900, 130, 8), (3000, 64, 3), (3001, 600, 7), (70000, 16, 8), (3, 20, 17000), (1000, 512, 256), (2050, 192, 384)]


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('points,inputs,outputs', SIZES)
def test_linear_and_gradient(engine, kind, points, inputs, outputs):
    for at, activation in enumerate(ACTIVATIONS):
        x, weight = made(1, points, inputs, dtype=kind), made(2, outputs, inputs, dtype=kind, scale=inputs ** -0.5)
        bias = made(3, outputs, dtype=kind) if at % 2 else None
        residual = made(4, points, outputs, dtype=kind) if at > 1 else None
        _, z = check_linear(engine, x, weight, bias, activation, residual)
        check_gradient(engine, made(5, points, outputs, dtype=kind), x, weight, bias, activation,
                       None if activation == 'linear' else z)


@pytest.mark.parametrize('kind,points,inputs,outputs', [(BF16, 4096, 2048, 2048), (F16, 1111, 1536, 4104), (F32, 1300, 2000, 1000),
                                                        (F32, 65536, 128, 128), (BF16, 100000, 64, 96), (F16, 33, 8192, 2048),
                                                        (BF16, 513, 8192, 513)])
def test_larger_layers(engine, kind, points, inputs, outputs):
    x, weight = made(1, points, inputs, dtype=kind), made(2, outputs, inputs, dtype=kind, scale=inputs ** -0.5)
    bias, residual = made(3, outputs, dtype=kind), made(4, points, outputs, dtype=kind)
    _, z = check_linear(engine, x, weight, bias, 'silu', residual)
    check_gradient(engine, made(5, points, outputs, dtype=kind), x, weight, bias, 'silu', z)


@pytest.mark.parametrize('kind', KINDS)
def test_layouts(engine, kind):
    """Rows with strides and at odd addresses, transposed and broadcast arrays, further leading dimensions."""
    whole, weights = made(6, 90, 200, dtype=kind), made(7, 200, 200, dtype=kind, scale=0.1)
    grads = made(8, 90, 200, dtype=kind)
    for x, weight, grad in ((whole[:, 8:72], weights[:40, 16:80], grads[:, :40]), (whole[:, 3:68], weights[1:34, 5:70], grads[:, 1:34]),
                            (whole[::2, 1:2], weights[:, :1], grads[::2]), (whole[:64].t(), weights[:50, :64], grads[0, :50].expand(200, 50)),
                            (whole[:1].expand(17, 200), weights.t(), grads[:17]),
                            (whole.view(9, 10, 200)[:, ::3, :24], weights[:16, :24], grads.view(9, 10, 200)[:, ::3, 4:20]),
                            (whole[0, :33], weights[:, :33], grads[0])):
        residual = grad * 2
        _, z = check_linear(engine, x, weight, None, 'tanh', residual)
        padded = torch.zeros((*z.shape[:-1], z.shape[-1] + 3), dtype=kind, device='cuda')
        padded[..., 2:-1] = z
        check_gradient(engine, grad, x, weight, None, 'tanh', padded[..., 2:-1])


@pytest.mark.parametrize('kind', [BF16, F16])
def test_parameters_of_float32(engine, kind):
    x, weight, bias = made(9, 70, 40, dtype=kind), made(10, 24, 40, dtype=kind, scale=0.2), made(11, 24)
    _, z = check_linear(engine, x, weight, bias, 'sigmoid')
    _, dweight, dbias = check_gradient(engine, made(12, 70, 24, dtype=kind), x, weight, bias, 'sigmoid', z, dtype=F32)
    assert dweight.dtype == dbias.dtype == F32
    dbias = operators.linear_gradient(engine, made(12, 70, 24, dtype=kind), x, weight, bias, 'sigmoid', z)[2]
    assert dbias.dtype == F32


def test_needs(engine):
    x, weight, bias, grad = made(13, 30, 20), made(14, 10, 20), made(15, 10), made(16, 30, 10)
    z = operators.linear(engine, x, weight, bias, 'silu', keep=True)[1]
    whole = operators.linear_gradient(engine, grad, x, weight, bias, 'silu', z)
    for need in ((True, False), (False, True), (False, False)):
        for b in (bias, None):
            got = operators.linear_gradient(engine, grad, x, weight, b, 'silu', z, need=need)
            for part, want, there in zip(got, whole, (*need, b is not None)):
                assert (part is None) != there and (part is None or torch.equal(part, want))


@pytest.mark.parametrize('kind', KINDS)
def test_no_points(engine, kind):
    x, weight, bias = made(17, 0, 20, dtype=kind), made(18, 10, 20, dtype=kind), made(19, 10, dtype=kind)
    y, z = operators.linear(engine, x, weight, bias, 'tanh', keep=True)
    assert y.shape == z.shape == (0, 10)
    dx, dweight, dbias = operators.linear_gradient(engine, y, x, weight, bias, 'tanh', z)
    assert dx.shape == (0, 20) and not dweight.any() and not dbias.any()


@pytest.mark.parametrize('kind', KINDS)
def test_a_bad_row_stays_in_its_row(engine, kind):
    """NaN, infinite and largest values in one point change nothing of the others."""
    for points, inputs, outputs in ((40, 64, 64), (300, 130, 33), (1, 64, 64), (700, 256, 256)):
        x, weight = made(20, points, inputs, dtype=kind), made(21, outputs, inputs, dtype=kind, scale=0.1)
        clean, _ = operators.linear(engine, x, weight)
        at = points // 2
        for bad in (float('nan'), float('inf'), torch.finfo(kind).max):
            x[at, 3 % inputs] = bad
            got, _ = operators.linear(engine, x, weight)
            keep = torch.arange(points, device='cuda') != at
            assert same_bits(got[keep], clean[keep])
            if bad != bad:
                assert got[at].isnan().all()
            elif bad == float('inf'):
                assert not got[at].isfinite().any()


def test_float32_range(engine):
    """Rows of very different sizes keep the error of FP32 each, up to the largest numbers and down to small ones."""
    x = made(22, 9, 96) * torch.tensor([1e-30, 1e-20, 1e-10, 1e-3, 1, 1e5, 1e15, 1e25, 1e36], device='cuda')[:, None]
    weight = made(23, 40, 96, scale=0.1)
    check_linear(engine, x, weight, None, 'linear')
    huge = torch.full((2, 8), torch.finfo(F32).max, device='cuda')
    one = torch.zeros((3, 8), device='cuda')
    one[0, 0], one[1, 1], one[2, 2] = 1.0, 0.5, 1e-30
    y, _ = operators.linear(engine, huge, one)
    want = huge.double() @ one.double().t()
    assert ((y.double() - want).abs() <= 2.0 ** -22 * want).all()


def test_gradient_against_differences(engine):
    """Central differences of the FP32 forward: with steps of 1e-2 along a direction the truncation is below 1e-4 of the
    third derivative's scale, and rounding of a sum of 600 values to FP32 over the step below 1e-4 of the sum's terms."""
    x, weight, bias, grad = made(24, 30, 24), made(25, 20, 24, scale=0.3), made(26, 20), made(27, 30, 20)
    for activation in ACTIVATIONS:
        def loss(x, weight, bias):
            return float((operators.linear(engine, x, weight, bias, activation)[0].double() * grad.double()).sum())

        z = operators.linear(engine, x, weight, bias, activation, keep=True)[1]
        for at, part in enumerate(operators.linear_gradient(engine, grad, x, weight, bias, activation, z)):
            v = made(28, *part.shape)
            v /= v.norm()
            ahead, back = ([t + (h * v if i == at else 0) for i, t in enumerate((x, weight, bias))] for h in (1e-2, -1e-2))
            slope = (loss(*ahead) - loss(*back)) / 2e-2
            assert abs(slope - float((part * v).sum())) < 2e-3 * float(grad.norm())


# --- orthogonalised matrices -----------------------------------------------------

def update(seed, *shape, dtype=F32, scale=1e-3):
    """Strong directions over a weak rest, as a layer's gradient has them."""
    r = min(8, *shape[-2:])
    strong = made(seed, *shape[:-1], r) / torch.arange(1, r + 1, device='cuda') @ made(seed + 1, *shape[:-2], r, shape[-1])
    return (scale * (strong + 0.05 * made(seed + 2, *shape))).to(dtype)


def close(got, x, kind, **options):
    """Within eight times what the roundings of the parts do in 64 bits, and half a unit of the result's type."""
    want = oracle.orthogonalize(x, **options)
    off = (oracle.orthogonalize_modelled(x, kind, **options) - want).norm()
    bound = 8 * off + 2.0 ** -20 * want.norm() + oracle.ROUNDING[got.dtype] * want.norm()
    assert (got.to(torch.float64) - want).norm() <= bound, (float((got.to(torch.float64) - want).norm() / want.norm()),
                                                              float(bound / want.norm()))


MATRICES = [(1, 1), (1, 7), (7, 1), (3, 5), (24, 40), (40, 24), (20, 128), (128, 20), (64, 64), (128, 256), (250, 120), (72, 200), (65, 64), (128, 128), (130, 257), (500, 129),
            (77, 1000), (256, 256), (512, 384), (1024, 320)]


@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('rows,columns', MATRICES)
def test_orthogonalize(engine, kind, rows, columns):
    x = update(30, rows, columns, dtype=kind)
    got = operators.orthogonalize(engine, x)
    assert got.shape == x.shape and got.dtype == kind
    close(got, x, kind)
    assert same_bits(got, operators.orthogonalize(engine, x))


@pytest.mark.parametrize('kind,rows,columns', [(BF16, 1024, 4096), (F32, 1024, 1024), (F16, 3000, 700)])
def test_orthogonalize_larger(engine, kind, rows, columns):
    x = update(33, rows, columns, dtype=kind)
    close(operators.orthogonalize(engine, x), x, kind)


@pytest.mark.parametrize('kind', KINDS)
def test_orthogonalize_batches(engine, kind):
    for shape in ((4, 128, 128), (3, 17, 90), (2, 300, 40), (0, 5, 6)):
        x = update(36, *shape, dtype=kind)
        got = operators.orthogonalize(engine, x)
        assert got.shape == x.shape
        for part, matrix in zip(got, x):
            close(part, matrix, kind)


def test_orthogonalize_steps_and_coefficients(engine):
    x = update(39, 60, 90)
    cubic, strong = (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)
    for options in (dict(steps=1), dict(steps=12), dict(coefficients=cubic, steps=9), dict(coefficients=strong),
                    dict(coefficients=[(4.0, -8.0, 5.0), (3.0, -3.5, 1.5), strong], steps=6), dict(coefficients=(1.0, 0.0, 0.0)),
                    dict(eps=1.0)):
        close(operators.orthogonalize(engine, x, **options), x, F32, **options)
    whole = operators.orthogonalize(engine, x, coefficients=cubic, steps=30)
    assert (whole @ whole.t() - torch.eye(60, device='cuda')).abs().max() < 1e-4


def test_orthogonalize_scales_and_layouts(engine):
    """The result does not depend on the matrix's size, from sizes whose squares overflow FP32 to small ones; any layout."""
    x = update(42, 50, 70, scale=1.0)
    for scale in (1e-3, 1e18, 1e25):
        close(operators.orthogonalize(engine, x * scale), x * scale, F32)
    base = operators.orthogonalize(engine, x)
    assert same_bits(operators.orthogonalize(engine, x.t().contiguous().t()), base)
    wide = torch.zeros((50, 99), device='cuda')
    wide[:, 3:73] = x
    assert same_bits(operators.orthogonalize(engine, wide[:, 3:73]), base)


@pytest.mark.parametrize('kind', KINDS)
def test_orthogonalize_zeros_and_bad_values(engine, kind):
    x = update(45, 3, 40, 64, dtype=kind, scale=1.0)
    x[1] = 0
    got = operators.orthogonalize(engine, x)
    assert not got[1].any()
    for bad in (float('nan'), float('inf')):
        x[1, 2, 3] = bad
        spoiled = operators.orthogonalize(engine, x)
        assert not spoiled[1].isfinite().any()
        assert same_bits(spoiled[0], got[0]) and same_bits(spoiled[2], got[2])


# --- the optimiser step ------------------------------------------------------------

@pytest.mark.parametrize('kind,momentum_kind', [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize('rows,columns', [(1, 1), (24, 40), (20, 128), (128, 20), (128, 128), (200, 72), (33, 515), (640, 256)])
def test_muon(engine, kind, momentum_kind, rows, columns):
    weight, grad = made(50, rows, columns, dtype=kind), update(51, rows, columns, dtype=kind)
    momentum = update(54, rows, columns, dtype=momentum_kind)
    for nesterov, decay, scale in ((True, 0.0, None), (False, 0.1, 0.3)):
        new_weight, new_momentum = operators.muon(engine, weight, grad, momentum, 0.02, 0.9, nesterov, decay, scale)
        m = 0.9 * momentum.double() + 0.1 * grad.double()
        u = 0.9 * m + 0.1 * grad.double() if nesterov else m
        size = 0.9 * momentum.double().abs() + 0.1 * grad.double().abs()
        within(new_momentum, m, (oracle.ROUNDING[momentum_kind] * (1 + 4 * oracle.E) + 4 * oracle.E) * size + oracle.TINY[momentum_kind])
        step = oracle.orthogonalize(u)
        off = (oracle.orthogonalize_modelled(u, kind, step=True) - step).norm()
        s = max(1.0, rows / columns) ** 0.5 if scale is None else scale
        want = (1 - 0.02 * decay) * weight.double() - 0.02 * s * step
        bound = 0.02 * s * (8 * off + 2.0 ** -20 * step.norm()) + (oracle.ROUNDING[kind] + 4 * oracle.E) * want.norm()
        assert (new_weight.double() - want).norm() <= bound
        w, m = weight.clone(), momentum.clone()
        version = w._version
        a, b = operators.muon(engine, w, grad, m, 0.02, 0.9, nesterov, decay, scale, inplace=True)
        assert a is w or a.data_ptr() == w.data_ptr()
        assert same_bits(w, new_weight) and same_bits(m, new_momentum) and w._version > version
        assert same_bits(b, m)


def test_optimiser(engine):
    """Steps of the class are those of the function; parameters without gradients are left alone."""
    a, b = torch.nn.Parameter(made(60, 24, 40)), torch.nn.Parameter(made(61, 8, 8))
    optimiser = operators.Muon(engine, [a, b], lr=0.1, beta=0.8, weight_decay=0.01)
    weight, momentum, before = a.detach().clone(), torch.zeros_like(a), b.detach().clone()
    for step in range(3):
        a.grad = update(62 + step, 24, 40)
        optimiser.step()
        weight, momentum = operators.muon(engine, weight, a.grad, momentum, 0.1, 0.8, True, 0.01)
        assert same_bits(a.detach(), weight) and same_bits(optimiser.state[a]['momentum'], momentum)
    assert torch.equal(b, before)
    with pytest.raises(ValueError, match='matrices'):
        operators.Muon(engine, [torch.nn.Parameter(made(63, 5))])


# --- together ------------------------------------------------------------------------

class Trunk(torch.nn.Module):
    def __init__(self, engine, widths):
        super().__init__()
        self.engine = engine
        self.weights = torch.nn.ParameterList([made(70 + i, o, c, scale=c ** -0.5) for i, (c, o) in enumerate(zip(widths, widths[1:]))])
        self.biases = torch.nn.ParameterList([made(80 + i, o, scale=0.1) for i, o in enumerate(widths[1:])])

    def forward(self, x, own):
        for i, (w, b) in enumerate(zip(self.weights, self.biases)):
            last = i + 1 == len(self.weights)
            residual = x if w.shape[0] == w.shape[1] else None
            if own:
                x = operators.Linear.apply(self.engine, x, w, b, 'linear' if last else 'tanh', residual)
            else:
                y = x @ w.t() + b
                y = y if last else torch.tanh(y)
                x = y if residual is None else residual + y
        return x


def test_a_network_trains(engine):
    """Gradients of a small trunk with the operators against torch's in 64 bits, then steps on them: the layers' chain keeps
    each gradient's error below 1e-5 of its norm (each layer's is some 1e-7, and there are five)."""
    trunk = Trunk(engine, [3, 128, 128, 128, 2])
    x, target = made(90, 777, 3), made(91, 777, 2)
    (trunk(x, True) - target).square().mean().backward()
    twin = Trunk(engine, [3, 128, 128, 128, 2])
    twin.double()
    (twin(x.double(), False) - target.double()).square().mean().backward()
    for a, b in zip(trunk.parameters(), twin.parameters()):
        assert (a.grad - b.grad).norm() <= 1e-5 * b.grad.norm()
    before = [w.detach().clone() for w in trunk.weights]
    operators.Muon(engine, list(trunk.weights)[1:3], lr=0.05).step()
    for i, (w, old) in enumerate(zip(trunk.weights, before)):
        if i in (1, 2):
            want = old.double() - 0.05 * oracle.orthogonalize(0.95 * 0.05 * w.grad + 0.05 * w.grad)
            assert (w - want).norm() <= 1e-5 * want.norm()
        else:
            assert torch.equal(w, old)


def test_captured(engine):
    """A step of forward, gradient and update in a graph, replayed on other inputs."""
    x, weight, bias, grad = made(92, 200, 96), made(93, 64, 96, scale=0.1), made(94, 64), made(95, 200, 64)
    momentum = torch.zeros_like(weight)

    def step(x, weight, momentum):
        y, z = operators.linear(engine, x, weight, bias, 'silu', keep=True)
        dx, dweight, dbias = operators.linear_gradient(engine, grad, x, weight, bias, 'silu', z)
        return (y, dx, dweight, dbias, *operators.muon(engine, weight, dweight, momentum, 0.1))

    held = x.clone()
    step(held, weight, momentum)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, weight, momentum)
    for seed in (96, 97):
        held.copy_(made(seed, 200, 96))
        graph.replay()
        for a, b in zip(out, step(held, weight, momentum)):
            assert same_bits(a, b)


def test_streams(engine):
    """Calls on three streams at once give what they give alone."""
    cases = [(made(100 + i, 1500 + 7 * i, 256, dtype=BF16), made(110 + i, 512, 256, dtype=BF16, scale=0.1), update(120 + i, 200, 150))
             for i in range(3)]

    def call(x, weight, matrix):
        y, z = operators.linear(engine, x, weight, None, 'tanh', keep=True)
        return (y, *operators.linear_gradient(engine, y, x, weight, None, 'tanh', z)[:2], operators.orthogonalize(engine, matrix))

    want = [call(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for stream, c in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(call(*c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(same_bits(p, q) for p, q in zip(a, b))


def test_workspace_is_not_read(engine):
    """The C entry with a workspace full of NaNs, and results between guards that stay."""
    lib = engine.lib
    for kind, code, p, c, o in ((F32, 0, 150, 72, 136), (BF16, 1, 150, 72, 136), (F32, 0, 700, 1500, 900), (BF16, 1, 33, 4096, 136),
                                (BF16, 1, 40, 75, 30)):
        x, weight = made(130, p, c, dtype=kind), made(131, o, c, dtype=kind)
        size = ctypes.c_size_t()
        args = (code, x.data_ptr(), c, p, c, o, weight.data_ptr(), c)
        assert lib.cpde_linear_workspace(*args, ctypes.byref(size)) == native.OK
        work = torch.full((size.value // 4 + 64,), float('nan'), device='cuda')
        y = torch.full((p * o + 256,), 7.0, dtype=kind, device='cuda')
        status = lib.cpde_linear(engine.handle, *args, 0, None, 2, None, 0, y[128:].data_ptr(), None, work.data_ptr(), size.value,
                                 torch.cuda.current_stream().cuda_stream or 1)
        assert status == native.OK
        assert (y[:128] == 7).all() and (y[128 + p * o:] == 7).all()
        assert same_bits(y[128:128 + p * o].view(p, o), operators.linear(engine, x, weight, None, 'tanh')[0])


@pytest.mark.parametrize('rows,columns', [(24, 40), (40, 24), (128, 128), (100, 77), (16, 250), (140, 136), (300, 50)])
def test_orthogonalize_writes_its_own(engine, rows, columns):
    """The C entry between guards, with a workspace full of NaNs, for one matrix and for three."""
    lib, coefficients = engine.lib, (ctypes.c_double * 3)(*oracle.QUINTIC)
    for matrices in (1, 3):
        x = update(132, matrices, rows, columns)
        count, size = x.numel(), ctypes.c_size_t()
        assert lib.cpde_orthogonalize_workspace(0, matrices, rows, columns, ctypes.byref(size)) == native.OK
        work = torch.full((size.value // 4 + 64,), float('nan'), device='cuda')
        out = torch.full((count + 256,), 7.0, device='cuda')
        status = lib.cpde_orthogonalize(engine.handle, 0, x.data_ptr(), matrices, rows, columns, 5, coefficients, 1, 1e-7,
                                        out[128:].data_ptr(), work.data_ptr(), size.value,
                                        torch.cuda.current_stream().cuda_stream or 1)
        assert status == native.OK
        assert (out[:128] == 7).all() and (out[128 + count:] == 7).all()
        assert same_bits(out[128:128 + count].view(x.shape), operators.orthogonalize(engine, x))
        for part, matrix in zip(out[128:128 + count].view(x.shape), x):
            close(part, matrix, F32)


def test_refusals(engine):
    x, weight, bias, grad = made(140, 6, 8), made(141, 4, 8), made(142, 4), made(143, 6, 4)
    z = made(144, 6, 4)

    def refused(call, match):
        with pytest.raises((ValueError, native.EngineError), match=match):
            call()

    refused(lambda: operators.linear(engine, x, weight[:, :7]), 'shape')
    refused(lambda: operators.linear(engine, x, weight.half()), 'one type')
    refused(lambda: operators.linear(engine, x.double(), weight.double()), 'float32')
    refused(lambda: operators.linear(engine, x, weight, bias[:3]), 'bias')
    refused(lambda: operators.linear(engine, x.half(), weight.half(), bias.bfloat16()), 'bias')
    refused(lambda: operators.linear(engine, x, weight, activation='relu'), 'activation')
    refused(lambda: operators.linear(engine, x, weight, residual=x), 'residual')
    refused(lambda: operators.linear(engine, x, weight, residual=grad.half()), 'residual')
    refused(lambda: operators.linear(engine, x, weight.cpu()), 'device')
    refused(lambda: operators.linear(engine, x, weight.clone().requires_grad_()), 'requires gradients')
    refused(lambda: operators.linear(engine, x[:, :0], weight[:, :0]), 'positive')
    refused(lambda: operators.linear_gradient(engine, grad, x, weight, activation='tanh'), 'z is needed')
    refused(lambda: operators.linear_gradient(engine, grad[:5], x, weight), 'grad')
    refused(lambda: operators.linear_gradient(engine, grad, x, weight, activation='tanh', z=z[:, :3]), 'z must')
    refused(lambda: operators.linear_gradient(engine, grad, x, weight, dtype=F16), 'dtype')
    refused(lambda: operators.orthogonalize(engine, x[0]), 'shape')
    refused(lambda: operators.orthogonalize(engine, x, steps=0), 'steps')
    refused(lambda: operators.orthogonalize(engine, x, eps=0.0), 'eps')
    refused(lambda: operators.orthogonalize(engine, x, eps=float('nan')), 'eps')
    refused(lambda: operators.orthogonalize(engine, x, coefficients=(1.0, 2.0)), 'triples')
    refused(lambda: operators.orthogonalize(engine, x, coefficients=(1.0, float('nan'), 0.0)), 'finite')
    refused(lambda: operators.orthogonalize(engine, x, coefficients=(9.0, 0.0, 0.0)), 'singular')
    refused(lambda: operators.orthogonalize(engine, x, coefficients=[(1.0, 0.0, 0.0)] * 6), 'triples')
    refused(lambda: operators.orthogonalize(engine, x[:, :0]), 'rows')
    refused(lambda: operators.muon(engine, x, x[:5], x, 0.1), 'shape')
    refused(lambda: operators.muon(engine, x, x.half(), x, 0.1), 'grad')
    refused(lambda: operators.muon(engine, x.half(), x.half(), x.bfloat16(), 0.1), 'momentum')
    refused(lambda: operators.muon(engine, x, x, x, 0.1, beta=1.0), 'beta')
    refused(lambda: operators.muon(engine, x, x, x, float('inf')), 'finite')
    refused(lambda: operators.muon(engine, x.t(), x.t(), x.t(), 0.1, inplace=True), 'contiguous')
    refused(lambda: operators.muon(engine, x.clone().requires_grad_(), x, x, 0.1), 'requires gradients')
    # At the C entry; a layer so wide that its operands are made into parts needs a workspace.
    wide = made(145, 2048, 2048)
    size = ctypes.c_size_t()
    assert engine.lib.cpde_linear_workspace(0, wide.data_ptr(), 2048, 2048, 2048, 2048, wide.data_ptr(), 2048,
                                            ctypes.byref(size)) == native.OK and size.value > 0
    work = torch.empty(size.value + 256, dtype=torch.uint8, device='cuda')
    y = torch.empty_like(wide)
    for bad in (dict(workspace=0), dict(workspace=work.data_ptr() + 16), dict(bytes=size.value - 1), dict(y=0), dict(x=0),
                dict(y=y.data_ptr() + 1), dict(stride=2047), dict(kind=3), dict(activation=4), dict(bias_type=2)):
        got = dict(kind=0, x=wide.data_ptr(), stride=2048, bias_type=0, activation=1, y=y.data_ptr(), workspace=work.data_ptr(),
                   bytes=size.value)
        got.update(bad)
        status = engine.lib.cpde_linear(engine.handle, got['kind'], got['x'], got['stride'], 2048, 2048, 2048, wide.data_ptr(),
                                        2048, got['bias_type'], None, got['activation'], None, 0, got['y'], None,
                                        got['workspace'], got['bytes'], None)
        assert status == native.REJECTED, bad


def test_autograd(engine):
    """The gradients that are wanted and no others, and what the function's own gradients are."""
    x, weight, bias, residual = made(150, 5, 9, 16), made(151, 32, 16, scale=0.2), made(152, 32), made(153, 5, 9, 32)
    grad = made(154, 5, 9, 32)
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias, residual)]
    y = operators.Linear.apply(engine, *leaves[:3], 'silu', leaves[3])
    y.backward(grad)
    z = operators.linear(engine, x, weight, bias, 'silu', keep=True)[1]
    want = operators.linear_gradient(engine, grad, x, weight, bias, 'silu', z)
    for leaf, part in zip(leaves, (*want, grad)):
        assert torch.equal(leaf.grad, part)
    for wanted in range(4):
        leaves = [t.clone().requires_grad_(i == wanted) for i, t in enumerate((x, weight, bias, residual))]
        operators.Linear.apply(engine, *leaves[:3], 'silu', leaves[3]).backward(grad)
        for i, (leaf, part) in enumerate(zip(leaves, (*want, grad))):
            assert (leaf.grad is not None) == (i == wanted) and (i != wanted or torch.equal(leaf.grad, part))
