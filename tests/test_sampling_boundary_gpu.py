"""Draws whose target lies next to the border between two tokens."""
import numpy as np
import pytest

from test_sampling_gpu import check

pytestmark = pytest.mark.gpu


def rows_next_to_a_border(n, lo, hi):
    """(x, u): rows of two logits, 0 and x, with u (1 + exp x) above or below 1 by lo .. hi units of 2^-44."""
    r, xs, us = np.random.default_rng(1), [], []
    while len(xs) < n:
        u = (0.5 + r.uniform(2.0 ** -13, 2.0 ** -9, 1 << 16)).astype(np.float32)
        w = u.astype(np.longdouble)
        x = np.log((1 - w) / w).astype(np.float32)         # the border; what this rounding leaves says on which side the target is
        beyond = np.abs(w * (1 + np.exp(x.astype(np.longdouble))) - 1) * 2.0 ** 44
        take = (beyond >= lo) & (beyond <= hi)
        xs += list(x[take])
        us += list(u[take])
    return np.stack([np.zeros(n, np.float32), np.array(xs[:n])], 1), np.array(us[:n])


@pytest.mark.parametrize("lo,hi", [(0.4, 0.6), (0.6, 1.0), (1.0, 5.0)])
def test_tokens_next_to_a_border(dev, lo, hi):
    """The best weight is 2^44 units, exactly; the other one is off by half a unit and 0.15 more (9e-15, where its series ends), and u = 1/2 of that moves the
    target: 0.33 units."""
    x, u = rows_next_to_a_border(400, lo, hi)
    check(dev, x, u)
