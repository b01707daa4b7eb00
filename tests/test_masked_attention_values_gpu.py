"""Values that are infinite or no numbers in rows of the cache that some queries of a call see and others do not: the first have them in their results, the others are
what the definition gives from the keys that they see.  Paths and tolerances as in test_masked_attention_undefined_gpu.py."""
import numpy as np
import pytest

from test_masked_attention_gpu import attention
from test_masked_attention_undefined_gpu import call_of, cases, put, run

pytestmark = pytest.mark.gpu


def compare(c, got):
    reached = 0
    for s, m in enumerate(c.masks):
        with np.errstate(invalid="ignore"):
            want, off = attention(c.values[0][s], c.values[1][s], c.values[2][s], m, c.scale, c.B.bf16)
            want *= 0.7
            fine = np.isfinite(want)
            assert np.array_equal(np.where(fine, 0.0, want), np.where(fine, 0.0, got[s]), equal_nan=True)
            assert (np.abs(got[s] - want)[fine] <= off[fine]).all()
        reached += int((~fine).sum())
    return reached


@cases
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["first", "last", "middle", "all of some"])
def test_a_value_that_is_not_finite(dev, path, kind, value, where):
    c = call_of(dev, path, kind, 600)
    t, heads = c.values[0].shape[1:3]
    rows = 0
    for s in (0, c.values[0].shape[0] // 2):
        some = np.nonzero(c.masks[s].any(0) & ~c.masks[s].all(0))[0]
        j = {"first": some[:1], "last": some[-1:], "middle": some[len(some) // 2:][:1], "all of some": some}[where]
        c.values[2][s, -1, j, 5] = value
        c.values[2][s, -1, j[:1], c.dims[5] - 1] = value
        rows += c.masks[s][:, j].any(1).sum()
    put(c, 2)
    assert compare(c, run(dev, c, path)) >= rows > 0


@cases
def test_infinities_of_both_signs(dev, path, kind):
    """Two that one query sees are NaN together, one alone is not; and one that every query sees."""
    c = call_of(dev, path, kind, 650)
    for s in (0, c.values[0].shape[0] - 1):
        some = np.nonzero(c.masks[s].any(0) & ~c.masks[s].all(0))[0]
        every = np.nonzero(c.masks[s].all(0))[0]
        c.values[2][s, 0, some[0], 9:12] = np.inf
        c.values[2][s, 0, some[-1], 9:12] = -np.inf
        c.values[2][s, 0, every[len(every) // 2], 11:14] = -np.inf
    put(c, 2)
    assert compare(c, run(dev, c, path)) > 0
