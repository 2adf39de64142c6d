"""8-bit states of ``AdamWMulti`` over many steps: they follow the gradients as 32-bit states do.

A rounding of the second moment between neighbouring codes lo < hi is unbiased in v = r^2.  Where a step moves v by d out of a gap
of q between codes, it adds a variance of at most d q.  Gaps are 0.18 v on average over a binade and at most 0.27 v.
Steady: d is on average at most (1 - b2) v (E|g^2 / v - 1| = 0.97 for Gaussian g), and the average forgets at 1 - b2, so the
relative variance of v settles at 0.18 (1 - b2) / (1 - b2^2) <= 0.09, whatever b2.
Shrinking: while v falls as e^-s it forgets no faster than it falls, so the relative variance grows by 0.18 for each e-fold of the
fall, 4.6 of them for gradients ten times smaller, and is back at 0.09 some e-folds later.
With x = log(1 + variance), v taken as log-normal: the mean of v is right, the median of its root off by e^(-x / 4), the norm of
the update, sqrt(mean 1 / v), by e^(x / 2).  The first moment adds 0.09^2 / 6 / (1 - b1^2) = 0.7 % of variance to the update.  A
twentieth is left for the samples (4096 values: 1.5 % at a variance of 0.9) and for what the estimates round off.
"""
import math

import pytest
import torch

from maester_b200.ops import reference as ref
from maester_b200.optimizers import AdamWMulti

N = 4096


def _gradient(kind, step, size, g):
    noise = torch.randn(N, generator=g) * size
    if kind == "noise":
        return noise
    if kind == "constant":
        return size.clone()
    return noise * (1.0 if step < 300 else 0.1)           # shrinking


@pytest.mark.parametrize("b2", [0.95, 0.99, 0.999])
@pytest.mark.parametrize("kind", ["noise", "constant", "shrinking"])
def test_states_follow_the_gradients(kind, b2):
    size = torch.exp(torch.randn(N, generator=torch.Generator().manual_seed(1)))    # (values of a block differ a hundredfold)
    kw = dict(lr=1e-3, betas=(0.9, b2), eps=1e-12, weight_decay=0.0)
    a, b = (torch.nn.Parameter(torch.zeros(N)) for _ in range(2))
    eight, full = AdamWMulti([a], state_bits=8, **kw), AdamWMulti([b], state_bits=32, **kw)
    g = torch.Generator().manual_seed(2)
    for step in range(2000):
        a.grad = b.grad = _gradient(kind, step, size, g)
        if step + 1 in (2, 10, 100, 299, 400, 1000, 2000):
            before = a.detach().clone(), b.detach().clone()
        eight.step()
        full.step()
        if step + 1 in (2, 10, 100, 299, 400, 1000, 2000):
            (m8, v8), (m32, v32) = eight._moments(a), full._moments(b)
            fall = min((step + 1 - 300) * (1 - b2), 4.6) if kind == "shrinking" and step >= 300 else 0.0
            settled = kind == "shrinking" and (step + 1 - 300) * (1 - b2) > 10.0
            x = math.log(1 + 0.09 + (0.0 if settled else 0.18 * fall))
            level = ((v8 / size ** 2).sum() / (v32 / size ** 2).sum()).item()   # (values that a block lifts count little)
            root = (v8 / v32).sqrt().median().item()
            update = ((a.detach() - before[0]).norm() / (b.detach() - before[1]).norm()).item()
            assert 0.95 < level < 1.05, (step + 1, level)
            assert 0.95 * math.exp(-x / 4) < root < 1.05, (step + 1, root)
            assert 0.95 < update < 1.05 * math.exp(x / 2), (step + 1, update)
            if kind == "constant":
                assert 0.95 < (m8 / m32).mean() < 1.05
