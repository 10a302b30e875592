"""Device-tensor operators at offsets beyond 2^31 elements and at the sizes between which they change their kernels. Large
results are spot-checked on the device; tolerances as in test_gpu_operators.py."""
import numpy as np
import pytest

torch = pytest.importorskip('torch')

import operator_oracle as oracle  # noqa: E402
from cpde_b200 import native, operators  # noqa: E402
from operator_oracle import EPS, ROUNDING, wide  # noqa: E402
from test_gpu_operators import check_gradient, check_norm, made, norm_inputs, some_ids  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope='module')
def engine():
    torch.cuda.init()
    with native.Engine(0) as e:
        yield e
    torch.cuda.empty_cache()


def test_embedding_table_beyond_32_bit_offsets(engine):
    rows, channels = 1100000, 2048
    assert rows * channels > 1 << 31
    table = torch.empty((rows, channels), dtype=BF16, device='cuda')
    ids = torch.tensor([0, rows - 1, 5, rows - 2, 1048576, 1048575], device='cuda')
    table[ids] = made(1, len(ids), channels, dtype=BF16)
    assert torch.equal(operators.embedding(engine, table, ids), table[ids])


def test_embedding_gradient_beyond_32_bit_offsets(engine):
    rows, channels = 1100000, 2048
    ids = torch.tensor([0, rows - 1, 5, rows - 2, 1048576, 1048575, rows - 1], device='cuda')
    grad = made(2, len(ids), channels, dtype=BF16)
    got = operators.embedding_gradient(engine, grad, ids, rows)
    assert torch.equal(got[ids[:6]][[0, 2, 3, 4, 5]], grad[[0, 2, 3, 4, 5]])
    assert torch.equal(got[rows - 1], (grad[1].float() + grad[6].float()).to(BF16))
    assert int(torch.count_nonzero(got.view(torch.int16).any(1))) == 6


def test_embedding_many_tokens_beyond_32_bit_offsets(engine):
    tokens, channels = 2200000, 1024
    table = made(3, 7, channels, dtype=BF16)
    ids = torch.arange(tokens, device='cuda') % 7
    out = operators.embedding(engine, table, ids)
    at = torch.tensor([0, tokens - 1, tokens - 2, 2097151, 2097152, 2097153], device='cuda')
    assert torch.equal(out[at], table[ids[at]])
    got = operators.embedding_gradient(engine, out, ids, 7, scale=1 / 65536, dtype=F32)
    counts = torch.bincount(ids, minlength=7)[:, None]
    want = wide(table) * wide(counts) / 65536
    assert (abs(wide(got) - want) <= (tokens / 7 + 2) * EPS * abs(want)).all()


def test_dropout_beyond_32_bit_offsets(engine):
    count = (1 << 31) + 4096
    x = torch.ones(count, dtype=BF16, device='cuda')
    y = operators.dropout(engine, x, 0.25, 3, 4)
    for first in (0, (1 << 31) - 64, 1 << 31, count - 64):
        words = oracle.philox(range(first // 8, first // 8 + 8), 4, 3)
        keep = words.astype('<u4').view('<u2').reshape(-1) >= 16384
        assert np.array_equal(wide(y[first:first + 64]) != 0, keep)


@pytest.mark.parametrize('n,p,c,groups', [(2, 1100000, 1024, 8), (600, 3600, 1024, 32)])
def test_group_norm_beyond_32_bit_offsets(engine, n, p, c, groups):
    x = torch.empty((n, p, c), dtype=BF16, device='cuda')
    x.copy_(made(5, 1, 997, c, dtype=BF16).expand(n, 997, c)[:, torch.arange(p, device='cuda') % 997])
    x[-1] += 3
    y, mean, rstd = operators.group_norm(engine, x, groups, activation='silu')
    dx, _, _ = operators.group_norm_gradient(engine, x, x, mean, rstd, groups, activation='silu')
    last = x[-1].double().view(p, groups, -1)
    m, v = last.mean((0, 2)), last.var((0, 2), unbiased=False)
    assert torch.allclose(mean[-1].double(), m, rtol=0, atol=64 * EPS * 8)
    assert torch.allclose(rstd[-1].double(), (v + 1e-5).rsqrt(), rtol=64 * EPS * 8, atol=0)
    xhat = (last - m[:, None]) * (v + 1e-5).rsqrt()[:, None]
    f = torch.sigmoid(xhat)
    assert (y[-1].double().view_as(xhat) - xhat * f).norm() <= (64 * EPS * 8 + ROUNDING[BF16]) * (xhat * f).norm()
    h = last * f * (1 + xhat * (1 - f))
    want = (h - h.mean((0, 2), keepdim=True) - xhat * (h * xhat).mean((0, 2), keepdim=True)) * (v + 1e-5).rsqrt()[:, None]
    assert (dx[-1].double().view_as(want) - want).norm() <= (64 * EPS * 64 + ROUNDING[BF16]) * h.norm()


# --- sizes around which the kernels change ----------------------------------------

@pytest.mark.parametrize('tokens,rows,channels', [(1023, 256, 1024), (1024, 256, 1024), (1025, 256, 1024),
                                                  (1024, 256, 1032), (512, 262144, 1), (1, 1, 8), (33, 40, 520)])
def test_gradient_of_few_tokens(engine, tokens, rows, channels):
    grad = made(10, tokens, channels)
    for skew in (False, True):
        check_gradient(engine, grad, some_ids(11, tokens, rows, absent=True, skew=skew), rows)


@pytest.mark.parametrize('tokens', [65535, 65536, 65537, 148 * 32 * 512 - 1, 148 * 32 * 512 + 1])
def test_gradient_sort_launches(engine, tokens):
    """The sort by one cluster, by one wave of tiles and by two."""
    grad = made(12, tokens, 2, dtype=BF16)
    check_gradient(engine, grad, some_ids(13, tokens, 70000, skew=True), 70000, dtype=F32)


@pytest.mark.parametrize('length', [1, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 600])
@pytest.mark.parametrize('lead', [0, 1, 5, 64, 70])
def test_gradient_runs_across_chunks(engine, length, lead):
    """One run of equal rows at every place relative to the chunks' borders, between runs of one token."""
    tokens = 40000
    ids = torch.arange(tokens, device='cuda')
    ids[lead:lead + length] = lead
    ids[20000:20000 + 3 * length] = 20000
    check_gradient(engine, made(14, tokens, 8), ids[torch.randperm(tokens, device='cuda')], tokens)


@pytest.mark.parametrize('rows,channels', [(30000, 2048), (30011, 1032), (200000, 260)])
def test_gradient_clears_a_large_table(engine, rows, channels):
    """Tables whose rows without a token are cleared by the sums' launch."""
    ids = some_ids(15, 3000, rows, absent=True, skew=True)
    ids[0], ids[1] = 0, rows - 1
    grad = made(16, 3000, channels)
    grad[(ids < 0) | (ids >= rows)] = float('nan')  # absent tokens' gradients are not read
    got = operators.embedding_gradient(engine, grad, ids, rows)
    again = operators.embedding_gradient(engine, grad, ids, rows)
    assert torch.equal(got, again)
    there = (ids >= 0) & (ids < rows)
    want = torch.zeros((rows, channels), dtype=torch.float64, device='cuda')
    want.index_add_(0, ids[there], grad[there].double())
    size = torch.zeros_like(want).index_add_(0, ids[there], grad[there].double().abs())
    terms = torch.bincount(ids[there], minlength=rows)[:, None]
    assert bool(((got.double() - want).abs() <= (terms + 1) * EPS * size).all())


@pytest.mark.parametrize('n,p,c,groups', [
    (1, 3000, 64, 8), (1, 30000, 64, 8), (3, 5000, 96, 4), (70, 90, 192, 12), (300, 33, 64, 16), (2, 2000, 1024, 2),
    (1, 513, 32, 1), (9, 1500, 40, 5), (130, 700, 128, 8)])
@pytest.mark.parametrize('kind', [F32, BF16])
def test_group_norm_cluster_sizes(engine, n, p, c, groups, kind):
    """Slabs in clusters of 1 to 16, more items than clusters, tiles that are no power of two."""
    x, weight, bias = norm_inputs(n, p, c, kind)
    check_norm(engine, x, groups, weight, bias, 'silu')
    lengths = torch.randint(0, p + 1, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(9)).cuda()
    check_norm(engine, x, groups, weight, bias, 'tanh', lengths)


def test_group_norm_unaligned_parameters(engine):
    x, weight, bias = norm_inputs(3, 200, 64, BF16)
    w, b = torch.empty(65, device='cuda')[1:], torch.empty(67, device='cuda')[3:]
    w.copy_(weight)
    b.copy_(bias)
    check_norm(engine, x, 4, w, b, 'silu')
    w16, b16 = torch.empty(65, dtype=BF16, device='cuda')[1:], torch.empty(67, dtype=BF16, device='cuda')[3:]
    w16.copy_(weight)
    b16.copy_(bias)
    check_norm(engine, x, 4, w16, b16, 'silu')
