"""A family of solutions in one network, and where to sample next.

The engine solves u'' = -k^2 u with u(0) = 0, u'(0) = k for a few wavenumbers k, each by training a small network on the
equation's residual. A conditioned trunk then learns the whole family: a latent code per instance is looked up, added to
features of its points, normalised by groups over them with an activation and dropout, and added back to the trunk through
another dropout. The point counts differ from instance to instance. With dropout kept on in evaluation, the spread over
masks says at which points the family is least known: there the next collocation points belong.

    python examples/field_family.py            # needs a B200 and the built library
"""
import argparse
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cpde_b200 import native, operators  # noqa: E402
from cpde_b200.expressions import Expression, glorot_like, quadrature_inputs, table  # noqa: E402
from cpde_b200.wire import Writer  # noqa: E402

CHANNELS, GROUPS, RATE, SEED = 64, 8, 0.1, 20


def solve(engine, k, points, epochs):
    """u at ``points`` of a network that the engine trains on the residual and the conditions at 0."""
    layers = [1, 32, 32, 1]
    net = engine.network(layers, glorot_like(layers, seed=int(10 * k)))
    costs = []
    for text, x, weight in ((f'(u_xx+{k * k}*u)**2', points, 1.0 / len(points)), (f'u**2+(u_x-{k})**2', points[:1], 10.0)):
        t = table(['', 'x', 'xx'], 'x')
        data = engine.data(quadrature_inputs(x[:, None], t), t)
        e = Expression(text, table=t, variables='x', outputs='u', count=len(x))
        costs.append(engine.integral(net, data, len(x), np.asarray(e.nodes, np.int32), np.asarray(e.constants, np.float64),
                                     e.field_array(), np.full(len(x), weight)))
    body = (Writer().put('Q', net).array(costs, 'u8').put('Q', epochs).put('i', 0).put('i', 1).put('f', 0.01).put('i', 0)
            .put('f', 0.0))
    for value in (0, 1, 0, 0, 0):  # nothing is logged, evaluated or saved
        body.put('i', value)
    engine.train(body.string('').put('i', 0).bytes())
    t = table([''], 'x')
    return engine.download(engine.evaluate(net, engine.data(quadrature_inputs(points[:, None], t), t)))[0, 0]


class Trunk(torch.nn.Module):
    """Instance codes and point features to a field, with the engine's operators."""

    def __init__(self, engine, instances):
        super().__init__()
        self.engine = engine
        self.codes = torch.nn.Parameter(torch.randn(instances, CHANNELS))
        self.features = torch.nn.Linear(1, CHANNELS)
        self.inner = torch.nn.Linear(CHANNELS, CHANNELS)
        self.weight, self.bias = torch.nn.Parameter(torch.ones(CHANNELS)), torch.nn.Parameter(torch.zeros(CHANNELS))
        self.head = torch.nn.Linear(CHANNELS, 1)

    def forward(self, ids, x, lengths, step):
        h = operators.Embedding.apply(self.engine, self.codes, ids, 0.5) + torch.sin(4 * self.features(x))
        # Each place and step has masks of its own: they are numbered by the offset.
        n = operators.GroupNorm.apply(self.engine, self.inner(h), self.weight, self.bias, GROUPS, 1e-5, 'silu', lengths, RATE,
                                      SEED, 2 * step)
        return self.head(operators.Dropout.apply(self.engine, n, RATE, SEED, 2 * step + 1, h))[..., 0]


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument('--points', type=int, default=256)
    parser.add_argument('--epochs', type=int, default=400, help='epochs of each solution')
    parser.add_argument('--steps', type=int, default=400, help='steps of the family')
    parser.add_argument('--masks', type=int, default=32, help='evaluations with dropout kept on')
    args = parser.parse_args(argv)
    wavenumbers = [1.0, 1.5, 2.0, 2.5]
    torch.manual_seed(0)
    with native.Engine(0) as engine:
        points = np.linspace(0.0, 1.0, args.points)
        fields = torch.tensor(np.stack([solve(engine, k, points, args.epochs) for k in wavenumbers])).float().cuda()
        exact = np.sin(np.outer(wavenumbers, points))
        print('solutions: largest error', float(abs(fields.cpu().numpy() - exact).max()))
        # An instance knows its field at its first points only, the later ones at fewer.
        n = len(wavenumbers)
        lengths = torch.tensor([args.points * (n - i) // n for i in range(n)], dtype=torch.int32, device='cuda')
        known = torch.arange(args.points, device='cuda') < lengths[:, None]
        ids = torch.arange(n, device='cuda')[:, None].expand(n, args.points)
        x = torch.tensor(points, device='cuda').float().expand(n, -1)[..., None]
        trunk = Trunk(engine, n).cuda()
        optimizer = torch.optim.Adam(trunk.parameters(), lr=1e-2)
        losses = []
        for step in range(args.steps):
            loss = ((trunk(ids, x, lengths, step) - fields).square() * known).sum() / known.sum()
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
            losses.append(loss.detach())
        losses = torch.stack(losses).tolist()
        print('family: loss', losses[0], '->', losses[-1])
        with torch.no_grad():
            draws = torch.stack([trunk(ids, x, None, args.steps + i) for i in range(args.masks)])
        spread = draws.std(0)
        worst = spread.flatten().topk(8).indices.tolist()
        print('sample next (wavenumber, x):', [(wavenumbers[i // args.points], round(float(points[i % args.points]), 3))
                                               for i in worst])
        return losses, spread


if __name__ == '__main__':
    main()
