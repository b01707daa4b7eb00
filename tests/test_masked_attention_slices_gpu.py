"""Sequences that are not there or not valid, where the keys of the others run in slices or spread over the warps of a CTA, and caches that are mostly empty."""
import numpy as np
import pytest

from test_draft_rows_gpu import I32
from test_masked_attention_gpu import Call
from test_masked_attention_undefined_gpu import PATHS, call_of, run
from ug_b200 import UgError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path,kind,what", [(p, k, w) for p in PATHS for k in ("window", "tree") for w in ("absent", "negative", "behind the cache", "tree") if w != "tree" or k == "tree"])
def test_sequences_that_are_left_alone(dev, path, kind, what):
    """Their outputs stay as they were, whatever the scratch of the slices holds; the others are done."""
    bf16, d, heads, kv, t, t_max, b, launches = PATHS[path]
    c = call_of(dev, path, kind, 500)
    run(dev, c, path)                                      # leaves its sums in the scratch
    two = b + 2                                            # in front of, between and behind the valid ones
    bad = [0, 2] if b == 1 else [0, b // 2, two - 1]
    pos, good = np.empty(two, np.int32), [s for s in range(two) if s not in bad]
    pos[bad] = {"absent": -1, "negative": -2, "behind the cache": t_max - t + 1, "tree": t_max // 2}[what]
    pos[good] = [t_max - t - s for s in range(len(good))]
    parents = None
    if kind == "tree":
        parents = np.tile(np.arange(t) - 1, (two, 1))
        if what == "tree":
            parents[bad, t - 1] = t - 1                    # its own parent
    ok = np.where(np.isin(np.arange(two), bad), 0, pos)    # for the definition: what is bad is not looked at
    c = Call(dev, bf16, two, t, heads, kv, d, d, t_max, ok, parents=None if kind != "tree" else np.tile(np.arange(t) - 1, (two, 1)), sinks=2, window=c.window, seed=510)
    c.pos_s = I32(dev, pos)
    if kind == "tree":
        c.parents_s = I32(dev, parents)
    for s in bad:
        c.masks[s] = None
    if what == "absent":
        run(dev, c, path)
    else:
        with pytest.raises(UgError) as e:
            run(dev, c, path)
        assert e.value.code == 1
    c.check()


@pytest.mark.parametrize("bf16,d,heads,kv,t", [(True, 64, 32, 4, 24), (True, 128, 8, 2, 70), (False, 64, 4, 2, 9), (False, 128, 2, 1, 1)])
@pytest.mark.parametrize("pos", [[0], [300, -1, 0], [1, 127, 128]])
def test_caches_that_are_mostly_empty(dev, bf16, d, heads, kv, t, pos):
    """Many slices by the cache's length, of which hardly any has keys."""
    for kind in ("tree", "window"):
        parents = np.tile(np.arange(t) - 1, (len(pos), 1)) if kind == "tree" else None
        Call(dev, bf16, len(pos), t, heads, kv, d, d, 16384, pos, parents=parents, sinks=4, window=16000, seed=520).run().check()
