"""Attention over a window or a tree where a row's softmax is undefined or takes in infinities: a NaN in the query or in a key that is seen, scores of -inf.
What the definition gives does not depend on whether the keys ran in one piece, in slices, or spread over the warps of a CTA.  Tolerances are those of
test_masked_attention_gpu.py."""
import numpy as np
import pytest

from test_draft_rows_gpu import tree
from test_masked_attention_gpu import Call, attention
from ug_b200 import synth

pytestmark = pytest.mark.gpu
# name: (bf16, values of a head, query and key heads, positions, cache rows, sequences, kernels of a call)
PATHS = {"ffma": (False, 64, 4, 2, 3, 100, 1, 1), "ffma, slices": (False, 64, 4, 2, 3, 2048, 1, 2), "ffma, 64 rows, slices": (False, 128, 4, 2, 40, 2048, 1, 2),
         "one group": (True, 64, 4, 2, 3, 100, 1, 1), "one group, slices": (True, 64, 4, 2, 3, 2048, 1, 2), "one group, 128, slices": (True, 128, 8, 1, 9, 2048, 2, 2),
         "two groups": (True, 128, 4, 2, 70, 100, 1, 1), "two groups, slices": (True, 64, 4, 2, 70, 2048, 1, 2), "spread": (True, 64, 4, 2, 3, 2304, 75, 2)}
cases = pytest.mark.parametrize("path,kind", [(p, k) for p in PATHS for k in ("window", "tree")])


def call_of(dev, path, kind, seed, full=False, **kw):
    """A call that takes this path: caches full to the last row, or from nothing to that where there are many sequences."""
    bf16, d, heads, kv, t, t_max, b, _ = PATHS[path]
    r = synth.rng(90 + seed)
    pos = [t_max - t] + [int(x) for x in (np.full(b - 1, t_max - t) if full else r.integers(0, t_max - t, b - 1))]
    parents = np.array([tree(91 + seed + s, t) for s in range(b)]) if kind == "tree" else None
    return Call(dev, bf16, b, t, heads, kv, d, d, t_max, pos, parents=parents, sinks=2, window=2100 if b > 1 else t_max * 3 // 4, seed=seed, **kw)


def put(c, which):
    """The host's queries, keys or values (0, 1, 2), changed, as the device's."""
    x = c.values[which].ravel().astype(np.float32)
    c.keep[which].copy_host_to_device(synth.to_bf16_bits(x) if c.B.bf16 else x, bf16=c.B.bf16)


def run(dev, c, path):
    before = dev.launch_count
    c.run()
    assert dev.launch_count - before == PATHS[path][-1]    # sliced or not, as the name says
    dev.synchronize()
    return c.read()


def compare(c, got, undefined):
    """undefined [b, t, heads]: rows of NaN, all of each; the others as the definition gives them."""
    assert np.isnan(got[undefined]).all()
    for s, m in enumerate(c.masks):
        if undefined[s].all():
            continue
        with np.errstate(invalid="ignore"):
            want, off = attention(c.values[0][s], c.values[1][s], c.values[2][s], m, c.scale, c.B.bf16)
        fine = ~undefined[s]
        assert (np.abs(got[s][fine] - 0.7 * want[fine]) <= off[fine]).all()


@cases
def test_queries_that_are_not_numbers(dev, path, kind):
    c = call_of(dev, path, kind, 200)
    b, t, heads = c.values[0].shape[:3]
    undefined = np.zeros((b, t, heads), bool)
    for s, i, h, x in ((0, 0, 0, 5), (0, t - 1, heads - 1, 0), (b - 1, t // 2, 1, 63)):
        c.values[0][s, i, h, x] = np.nan
        undefined[s, i, h] = True
    put(c, 0)
    compare(c, run(dev, c, path), undefined)


@cases
@pytest.mark.parametrize("where", ["first", "last", "self", "middle"])
def test_seen_keys_that_are_not_numbers(dev, path, kind, where):
    c = call_of(dev, path, kind, 300)
    b, t, heads = c.values[0].shape[:3]
    share = heads // c.values[1].shape[1]
    undefined = np.zeros((b, t, heads), bool)
    for s in (0, b // 2):
        seen = np.nonzero(c.masks[s].any(0))[0]
        j = {"first": seen[0], "last": seen[-1], "self": c.pos[s], "middle": seen[len(seen) // 2]}[where]
        c.values[1][s, 0, j, 7] = np.nan
        undefined[s, :, :share] = c.masks[s][:, j, None]
    put(c, 1)
    compare(c, run(dev, c, path), undefined)


@cases
def test_rows_whose_only_keys_in_a_slice_are_not_numbers(dev, path, kind):
    """All keys of the second half: whatever the slices, some rows see nothing but NaN in one of them and numbers in others."""
    c = call_of(dev, path, kind, 350)
    t_max = c.values[1].shape[2]
    c.values[1][:, 0, t_max // 2:] = np.nan
    put(c, 1)
    share = c.values[0].shape[2] // c.values[1].shape[1]
    undefined = np.zeros(c.values[0].shape[:3], bool)
    for s, m in enumerate(c.masks):
        undefined[s, :, :share] = m[:, t_max // 2:].any(1)[:, None]
    compare(c, run(dev, c, path), undefined)


@cases
def test_scores_of_minus_infinity(dev, path, kind):
    """Where all are, 0 / 0; where some are, these weigh nothing.  Every score of the others is finite."""
    c = call_of(dev, path, kind, 400, full=True)
    c.values[0][..., 5] = 1.0
    share = c.values[0].shape[2] // c.values[1].shape[1]
    undefined = np.zeros(c.values[0].shape[:3], bool)
    for s, m in enumerate(c.masks):
        seen = np.nonzero(m.any(0))[0]
        if s == 0:                                         # everything that the first group sees
            c.values[1][s, 0, seen, 5] = -np.inf
            undefined[s, :, :share] = True
        rest = seen[(seen % 3 == 1) & (seen < c.pos[s])]   # a third of the committed positions, of every group
        c.values[1][s, :, rest, 5] = -np.inf
        c.masks[s] = m & ~np.isin(np.arange(m.shape[1]), rest)
    put(c, 0)
    put(c, 1)
    compare(c, run(dev, c, path), undefined)
