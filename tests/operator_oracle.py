"""The device-tensor operators in 64 bits on the host, from their definitions."""
import numpy as np
import torch

EPS = 2.0 ** -24  # half a unit in the last place of FP32, relative
# Half the spacing of the type's numbers at 1, relative: its significands have 24, 8 and 11 bits.
ROUNDING = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Smallest absolute rounding: half the spacing of the type's subnormal numbers.
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def wide(t):
    return t.detach().cpu().to(torch.float64).numpy()


def philox(index, offset, seed):
    """Philox4x32-10 of 64-bit counters; (len(index), 4) 32-bit words."""
    mask = 0xFFFFFFFF
    out = np.zeros((len(index), 4), np.uint32)
    for at, i in enumerate(index):
        x = [int(i) & mask, int(i) >> 32, offset & mask, offset >> 32]
        k = [seed & mask, seed >> 32]
        for _ in range(10):
            p, q = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
            x = [(q >> 32) ^ x[1] ^ k[0], q & mask, (p >> 32) ^ x[3] ^ k[1], p & mask]
            k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
        out[at] = x
    return out


def kept(count, rate, seed, offset):
    """(kept elements, factor of the kept ones)."""
    words = philox(range((count + 7) // 8), offset, seed)
    halves = words.astype('<u4').view('<u2').reshape(-1)[:count]
    threshold = int(np.floor(rate * 65536 + 0.5))
    return halves >= threshold, 65536 / (65536 - threshold) if threshold < 65536 else 0.0


def dropped(x, rate, seed, offset):
    keep, factor = kept(x.size, rate, seed, offset)
    keep = keep.reshape(x.shape)
    return np.where(keep, np.where(keep, x, 0.0) * factor, 0.0)


def activated(z, name):
    return {'linear': lambda: z, 'sigmoid': lambda: 1 / (1 + np.exp(-z)), 'tanh': lambda: np.tanh(z),
            'silu': lambda: z / (1 + np.exp(-z))}[name]()


def slope(z, name):
    f = 1 / (1 + np.exp(-z))
    return {'linear': lambda: np.ones_like(z), 'sigmoid': lambda: f * (1 - f), 'tanh': lambda: 1 - np.tanh(z) ** 2,
            'silu': lambda: f + z * f * (1 - f)}[name]()


def group_norm(x, groups, weight, bias, eps, activation, lengths, rate, seed, offset, grad=None):
    """(y, mean, rstd) and, with ``grad``, (dx, dweight, dbias) of float64 arrays."""
    n, p, c = x.shape
    width = c // groups
    weight = np.ones(c) if weight is None else weight
    bias = np.zeros(c) if bias is None else bias
    y, dx = np.zeros(x.shape), np.zeros(x.shape)
    mean, rstd = np.zeros((n, groups)), np.zeros((n, groups))
    dweight, dbias = np.zeros(c), np.zeros(c)
    z = np.zeros(x.shape)
    for i in range(n):
        m = p if lengths is None else min(max(int(lengths[i]), 0), p)
        for g in range(groups):
            cs = slice(g * width, (g + 1) * width)
            part = x[i, :m, cs]
            if m:
                mean[i, g] = part.mean()
                rstd[i, g] = 1 / np.sqrt(part.var() + eps)
            z[i, :m, cs] = (part - mean[i, g]) * rstd[i, g] * weight[cs] + bias[cs]
        y[i, :m] = activated(z[i, :m], activation)
    y = dropped(y, rate, seed, offset) if rate else y
    for i in range(n):
        y[i, (p if lengths is None else min(max(int(lengths[i]), 0), p)):] = 0
    if grad is None:
        return y, mean, rstd
    h = dropped(grad, rate, seed, offset) if rate else grad
    for i in range(n):
        m = p if lengths is None else min(max(int(lengths[i]), 0), p)
        for g in range(groups if m else 0):
            cs = slice(g * width, (g + 1) * width)
            xhat = (x[i, :m, cs] - mean[i, g]) * rstd[i, g]
            hh = h[i, :m, cs] * slope(z[i, :m, cs], activation)
            dbias[cs] += hh.sum(0)
            dweight[cs] += (hh * xhat).sum(0)
            wh = hh * weight[cs]
            dx[i, :m, cs] = rstd[i, g] * (wh - wh.mean() - xhat * (wh * xhat).mean())
    return y, mean, rstd, dx, dweight, dbias
