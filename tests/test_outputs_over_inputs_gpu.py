"""Operators of generation whose outputs would lie over what other sequences or rows of the call still read: refused, by the elements that the call uses.  Nothing is
launched."""
import numpy as np
import pytest

from test_draft_rows_gpu import I32
from ug_b200 import DType, UgError

pytestmark = pytest.mark.gpu


def over(dev, s, dtype, n):
    """The first n values of s as another type of 4 bytes."""
    return dev.wrap(s.device_ptr, dtype, n)


def refused(dev, call):
    before = dev.launch_count
    with pytest.raises(UgError) as e:
        call()
    assert e.value.code == 1 and dev.launch_count == before


def test_attention(dev):
    q, k, v, pos = dev.zeros(64), dev.zeros(512), dev.zeros(512), I32(dev, [0] * 64)
    bad = over(dev, pos, DType.F32, 64)
    refused(dev, lambda: dev.window_attend(q, k, v, pos, bad, 1, 2, 4, 1, 8, 8, 64, 0, 4, 1.0))
    refused(dev, lambda: dev.tree_attend(q, k, v, pos, I32(dev, [-1, 0]), bad, 1, 2, 4, 1, 8, 8, 64, 1.0))
    refused(dev, lambda: dev.tree_attend(q, k, v, I32(dev, [0]), pos, bad, 1, 2, 4, 1, 8, 8, 64, 1.0))
    # behind the elements that the call uses the slices may meet
    long = dev.zeros(128)
    before = dev.launch_count
    dev.window_attend(long, k, v, pos, dev.wrap(long.device_ptr + 4 * 64, DType.F32, 64), 1, 2, 4, 1, 8, 8, 64, 0, 4, 1.0)
    dev.synchronize()
    assert dev.launch_count > before


def test_inputs_of_nodes(dev):
    n = dict(pre=dev.zeros(96), cos=dev.zeros(128), sin=dev.zeros(128), pos=I32(dev, [0, 0]), parents=I32(dev, [-1, 0] * 2), q=dev.zeros(32), k=dev.zeros(512), v=dev.zeros(512))
    for a in ("pre", "cos", "sin", "pos", "parents"):
        for o in ("q", "k", "v"):
            swap = dict(n)
            big = dev.zeros(512)
            swap[o], swap[a] = big, over(dev, big, DType.I32 if a in ("pos", "parents") else DType.F32, 512)
            refused(dev, lambda: dev.tree_inputs(*swap.values(), 2, 2, 1, 1, 8, 8, 8, True, False, 1e-5, 32))
    dev.tree_inputs(*n.values(), 2, 2, 1, 1, 8, 8, 8, True, False, 1e-5, 32)
    dev.synchronize()


def test_kept_rows(dev):
    k, v, i = dev.zeros(512), dev.zeros(512), I32(dev, [0] * 8)
    for at in range(3):
        for cache in (k, v):
            args = [i, i, i]
            args[at] = over(dev, cache, DType.I32, 512)
            refused(dev, lambda: dev.cache_keep(k, v, *args, 2, 1, 8, 8, 32, 2))


@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p", "u"])
def test_sampling(dev, name):
    rows, vocab = 3, 50
    x, both = dev.zeros(rows * vocab), dev.slice_from_values(np.full(rows + 1, 0, np.int32))
    kind = DType.I32 if name == "top_k" else DType.F32
    for out in ("tokens", "prob"):
        given = dict(u=dev.zeros(rows), tokens=dev.allocate_uninit(DType.I32, rows), prob=dev.zeros(rows))
        given[name] = dev.wrap(both.device_ptr + 4, kind, rows)
        given[out] = dev.wrap(both.device_ptr, DType.I32 if out == "tokens" else DType.F32, rows)
        u, tokens = given.pop("u"), given.pop("tokens")
        refused(dev, lambda: dev.sample(x, u, tokens, rows, vocab, **given))


def test_a_share_in_the_place_of_its_random_number(dev):
    """Row by row, which is no overlap with another row's."""
    rows, vocab = 64, 50
    x, tokens = dev.zeros(rows * vocab), dev.allocate_uninit(DType.I32, rows)
    u = np.linspace(0, 0.99, rows).astype(np.float32)
    both = dev.slice_from_values(u)
    dev.sample(x, both, tokens, rows, vocab, prob=both)
    dev.synchronize()
    assert tokens.to_vec().tolist() == [int(np.floor(float(r) * vocab)) for r in u] and np.allclose(both.to_vec(), 1 / vocab, rtol=2.0 ** -23)
