"""Group norm and its gradient in 64 bits with the statistics given, and how far FP32 arithmetic may be off.

e = 2^-24 is the relative error of an FP32 operation, u half a unit in the last place of the array's type. All bounds are
first order and by element; Z = |d rstd w| + |b| with d = x - mean, K the longest chain of additions in a sum of ``points``
points (a thread's own points, at most 512, then the threads' and the blocks').

* z = d (w rstd) + b: three roundings of the factors, one of d, two of b's scaling and one of the sum: 5 e Z.
* The activations: sigmoid's exponential and reciprocal 2 and 1 units, tanh 2 units: at most 10 e of 1 + |a|. Their slopes
  (at most 1.1) change by at most 0.77 a unit of z and are evaluated to 32 e: e (32 + 4 Z).
* h = g act'(z), g = factor dy of the kept: e |g| (40 + 4 Z).
* Sums add K e of their terms' absolute sum; means over the channels of a group (width + 8) e more; what is left of dx is 8 e
  of its three terms.
* The statistics: deviations from a value of the group: the mean is off by at most (K + 8) e of the largest deviation and
  64 e of the largest value (64 or fewer means are joined), the variance by twice that times the deviations and by 2 K e of the
  largest deviation squared.
"""
import numpy as np

EPS = 2.0 ** -24


def kept(count, rate, seed, offset):
    """operator_oracle.kept by whole arrays."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    at = np.arange((count + 7) // 8, dtype=np.uint64)
    x = [at & low, at >> half, np.full_like(at, offset & 0xFFFFFFFF), np.full_like(at, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> half) ^ x[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ x[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack(x, 1).astype('<u4').view('<u2').reshape(-1)[:count]
    threshold = int(np.floor(rate * 65536 + 0.5))
    return halves >= threshold, 65536 / (65536 - threshold) if threshold < 65536 else 0.0


class Norm:
    """A call in 64 bits: ``x`` and ``grad`` (n, p, c), ``weight`` and ``bias`` (c,) or None, ``lengths`` a list or None."""

    def __init__(self, x, groups, weight, bias, eps, activation, lengths, rate, seed, offset):
        self.n, self.p, self.c = x.shape
        self.groups, self.width, self.eps, self.activation = groups, self.c // groups, eps, activation
        counts = np.full(self.n, self.p) if lengths is None else np.clip(lengths, 0, self.p)
        self.counts = counts
        self.mask = (np.arange(self.p) < counts[:, None])[:, :, None, None]
        self.values = np.maximum(counts, 1)[:, None] * self.width  # of a group
        self.x = np.where(self.mask, self.split(x), 0.0)
        self.w = (np.ones(self.c) if weight is None else weight).reshape(groups, -1)
        self.b = (np.zeros(self.c) if bias is None else bias).reshape(groups, -1)
        self.keep, self.factor = kept(x.size, rate, seed, offset) if rate else (np.ones(x.size, bool), 1.0)
        self.keep = self.split(self.keep.reshape(x.shape))
        self.chain = 64 + min(self.p, 512)

    def split(self, a):
        return a.reshape(self.n, self.p, self.groups, self.width)

    def statistics(self):
        """(mean, rstd) and their bounds, all (n, groups)."""
        mean = self.x.sum((1, 3)) / self.values
        d = np.where(self.mask, self.x - mean[:, None, :, None], 0.0)
        var = (d ** 2).sum((1, 3)) / self.values
        some = (self.counts > 0)[:, None]
        rstd = some / np.sqrt(var + self.eps)
        most, far = abs(self.x).max((1, 3), initial=0.0), 2 * abs(d).max((1, 3), initial=0.0)
        off = (self.chain + 8) * EPS * far + 64 * EPS * most
        off_var = 2 * off * far + off ** 2 + 2 * self.chain * EPS * far ** 2
        low = np.maximum(var - off_var, 0.0) + self.eps  # rstd moves most downwards in the variance
        return mean, rstd, off, some * (1 / np.sqrt(low) * (1 + 4 * EPS) - 1 / np.sqrt(var + self.eps))

    def _z(self, mean, rstd):
        d = np.where(self.mask, self.x - mean[:, None, :, None], 0.0)
        r = rstd[:, None, :, None]
        return d, r, d * r * self.w + self.b, abs(d * r * self.w) + abs(self.b)

    def forward(self, mean, rstd, u, tiny):
        """y and its bound, with the statistics given."""
        _, _, z, size = self._z(mean, rstd)
        with np.errstate(over='ignore'):
            f = 1 / (1 + np.exp(-z))
        a = {'linear': z, 'sigmoid': f, 'tanh': np.tanh(z), 'silu': z * f}[self.activation]
        there = self.mask & self.keep
        y = np.where(there, a * self.factor, 0.0)
        bound = self.factor * EPS * (6 * size + 10 * (abs(a) + (self.activation != 'linear'))) + u * abs(y) + tiny
        return y.reshape(self.n, self.p, -1), np.where(there, bound, 0.0).reshape(self.n, self.p, -1)

    def gradient(self, grad, mean, rstd, u, tiny):
        """((dx, bound), (dweight, bound), (dbias, bound)), with the statistics given; dweight's and dbias' bounds without
        their rounding."""
        d, r, z, size = self._z(mean, rstd)
        with np.errstate(over='ignore'):
            f = 1 / (1 + np.exp(-z))
        slope = {'linear': np.ones_like(z), 'sigmoid': f * (1 - f), 'tanh': 1 - np.tanh(z) ** 2,
                 'silu': f + z * f * (1 - f)}[self.activation]
        g = np.where(self.mask & self.keep, self.split(grad), 0.0) * self.factor
        h, off = g * slope, EPS * abs(g) * (40 + 4 * size)
        xhat = d * r

        def summed(v, off):
            return v.sum(1), off.sum(1) + (self.chain + 8) * EPS * abs(v).sum(1)

        def mean_of(v, off):  # of w times the channels' sums
            total, wide = (v * self.w).sum(2) / self.values, ((off + 8 * EPS * abs(v)) * abs(self.w)).sum(2) / self.values
            return total[:, None, :, None], (wide + (self.width + 8) * EPS * (abs(v * self.w)).sum(2) / self.values)[:, None, :, None]

        by_h, by_xhat = summed(h, off), summed(h * xhat, off * abs(xhat) + 3 * EPS * abs(h * xhat))
        (m1, off1), (m2, off2) = mean_of(*by_h), mean_of(*by_xhat)
        dx = np.where(self.mask, r * (self.w * h - m1 - xhat * m2), 0.0)
        terms = abs(self.w * h) + abs(m1) + abs(xhat * m2)
        bound = r * (abs(self.w) * off + off1 + abs(xhat) * off2 + 8 * EPS * terms) + u * abs(dx) + tiny

        def over_instances(v, off):
            return v.sum(0).reshape(-1), (off.sum(0) + (self.n * 16 + 128) * EPS * abs(v).sum(0)).reshape(-1)

        shape = (self.n, self.p, self.c)
        return ((dx.reshape(shape), np.where(self.mask, bound, 0.0).reshape(shape)), over_instances(*by_xhat),
                over_instances(*by_h))
