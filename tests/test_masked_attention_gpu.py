"""Attention over a window and the first positions, and of drafted trees, through the C ABI against the definition in 64 bits.

How far an output may be off, with w the weights that add up to 1 and A = sum w |v|: a score is a sum of dq products in 32 bits, off by 2 dq 2^-24 times the
sum of the products' sizes (a tensor core cuts off where another unit rounds: twice half a step), its way into the exponent and the exponential by 8 steps more,
and this moves numerator and denominator; the sums over n keys are off by 2 n 2^-24 at most.  In bf16 the weights are rounded (2^-8 A) and the output is (2^-8 of it)."""
import numpy as np
import pytest
import torch

from hybrid_cases import Buf
from test_draft_rows_gpu import I32, tree
from ug_b200 import DType, UgError, synth
from ug_b200._lib import lib

pytestmark = pytest.mark.gpu
f64 = np.float64


def window_mask(pos, t, n, sinks, window):
    i, j = pos + np.arange(t)[:, None], np.arange(n)
    return (j <= i) & ((j > i - window) | (j < sinks))


def tree_mask(pos, parents, n):
    m = np.zeros((len(parents), n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, :pos] = True
        m[i, pos + i] = True
    return m


def attention(q, k, v, mask, scale, bf16):
    """q [t, heads, dq], k / v [kv, n, ...], mask [t, n]; what the mask leaves out is never looked at.  (output, how far it may be off)"""
    t, heads, dq = q.shape
    share, out, off = heads // k.shape[0], np.empty((t, heads, v.shape[2])), np.empty((t, heads, v.shape[2]))
    for i in range(t):
        see = np.nonzero(mask[i])[0]
        for h in range(heads):
            kk, vv = k[h // share, see], v[h // share, see]
            s = kk @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ vv
            size = (2 * dq + 8) * (np.abs(kk) @ np.abs(q[i, h])).max() * scale
            off[i, h] = (2 * size + 16 + 2 * see.size + (2.0 ** 16 if bf16 else 0)) * 2.0 ** -24 * (w @ np.abs(vv)) + (2.0 ** -8 if bf16 else 2.0 ** -24) * np.abs(out[i, h])
    return out, off


class Call:
    """Buffers of one call, position by position what the definition gives, everything that no query sees NaN."""

    def __init__(self, dev, bf16, b, t, heads, kv, dq, dv, t_max, pos, parents=None, sinks=0, window=0, shift=0, seed=0, std=1.0, spoil=True):
        self.dev, self.B, self.dims = dev, Buf(dev, bf16), (b, t, heads, kv, dq, dv, t_max)
        self.pos, self.parents, self.sinks, self.window = np.array(pos), parents, sinks, window
        x = [synth.normal(seed + 7, (b, t, heads, dq), std), synth.normal(seed + 8, (b, kv, t_max, dq)), synth.normal(seed + 9, (b, kv, t_max, dv))]
        self.masks = [None if p < 0 else window_mask(p, t, t_max, sinks, window) if parents is None else tree_mask(p, parents[s], t_max) for s, p in enumerate(pos)]
        for s, m in enumerate(self.masks if spoil else []):
            hidden = ~m.any(0) if m is not None else np.ones(t_max, bool)
            x[1][s][:, hidden] = np.nan
            x[2][s][:, hidden] = np.nan if s % 2 == 0 else np.inf
        size = 2 if bf16 else 4
        part = lambda s: dev.wrap(s.device_ptr + shift * size, s.dtype, len(s) - shift)
        got = [self.B.act(np.r_[np.zeros(shift, np.float32), a.ravel()]) for a in x]
        self.keep = [g[0] for g in got]
        self.values = [g[1][shift:].reshape(a.shape) for g, a in zip(got, x)]
        self.whole = self.B.act(np.full(shift + b * t * heads * dv, 7.0))[0]
        self.q, self.k, self.v, self.out = (part(s) for s in self.keep + [self.whole])
        self.scale, self.shift = 1.3 * dq ** -0.5, shift
        self.pos_s = I32(dev, pos)
        self.parents_s = None if parents is None else I32(dev, parents)

    def run(self):
        b, t, heads, kv, dq, dv, t_max = self.dims
        if self.parents is None:
            self.dev.window_attend(self.q, self.k, self.v, self.pos_s, self.out, b, t, heads, kv, dq, dv, t_max, self.sinks, self.window, self.scale, 0.7)
        else:
            self.dev.tree_attend(self.q, self.k, self.v, self.pos_s, self.parents_s, self.out, b, t, heads, kv, dq, dv, t_max, self.scale, 0.7)
        return self

    def read(self):
        b, t, heads, _, _, dv, _ = self.dims
        return self.B.read(self.whole, (-1,))[self.shift:].reshape(b, t, heads, dv)

    def check(self):
        self.dev.synchronize()
        got = self.read()
        for s, m in enumerate(self.masks):
            if m is None:
                assert (got[s] == 7.0).all()               # left as it was
                continue
            with np.errstate(invalid="ignore"):
                want, off = attention(self.values[0][s], self.values[1][s], self.values[2][s], m, self.scale, self.B.bf16)
            assert np.isfinite(got[s]).all()
            assert (np.abs(got[s] - 0.7 * want) <= off).all(), (s, float(np.max(np.abs(got[s] - 0.7 * want) / off)))


HEADS = [(False, 8, 16), (False, 64, 64), (False, 72, 40), (False, 256, 200), (True, 64, 64), (True, 64, 128), (True, 128, 64), (True, 128, 128), (True, 72, 40),
         (True, 256, 136)]


@pytest.mark.parametrize("bf16,dq,dv", HEADS)
@pytest.mark.parametrize("heads,kv,t,t_max,pos,sinks,window", [
    (1, 1, 1, 16, [0], 0, 1), (8, 2, 1, 640, [300, -1, 0, 639], 4, 100), (3, 3, 1, 333, [65, 127], 70, 64), (32, 2, 1, 512, [450], 1, 300),
    (4, 4, 5, 200, [0, 63, 190], 0, 3), (8, 1, 70, 300, [0, 130], 5, 64), (10, 2, 33, 129, [96, -1], 64, 17), (16, 1, 200, 520, [320], 3, 128), (34, 2, 3, 80, [62, 5], 0, 80),
    (6, 2, 65, 65, [0], 2, 2 ** 40)])
def test_window(dev, bf16, dq, dv, heads, kv, t, t_max, pos, sinks, window):
    Call(dev, bf16, len(pos), t, heads, kv, dq, dv, t_max, pos, sinks=sinks, window=window).run().check()


@pytest.mark.parametrize("bf16,dq,dv", HEADS)
@pytest.mark.parametrize("heads,kv,t,t_max,pos", [
    (1, 1, 1, 1, [0]), (4, 2, 1, 130, [64, 0, -1]), (8, 1, 24, 333, [300, 17, 63]), (3, 3, 128, 300, [0, 172]), (10, 2, 64, 128, [64, -1, 1]), (32, 4, 7, 700, [693]),
    (24, 1, 33, 90, [57, 31])])
def test_tree(dev, bf16, dq, dv, heads, kv, t, t_max, pos):
    parents = np.array([tree(40 + s, t) for s in range(len(pos))])
    Call(dev, bf16, len(pos), t, heads, kv, dq, dv, t_max, pos, parents=parents).run().check()


@pytest.mark.parametrize("bf16,dq,dv,share,t,kind", [(True, 64, 64, 1, 1, "window"), (True, 64, 64, 8, 1, "window"), (True, 64, 64, 32, 1, "tree"), (True, 128, 128, 4, 1, "window"),
                                                     (True, 128, 64, 5, 6, "tree"), (True, 40, 96, 3, 10, "window"), (False, 64, 64, 4, 1, "window"), (True, 128, 128, 8, 4, "tree"),
                                                     (True, 64, 64, 11, 3, "window")])
def test_many_sequences_over_long_caches(dev, bf16, dq, dv, share, t, kind):
    """Few rows each of more sequences than the GPU has SMs, over thousands of keys: lengths of one key to all, first positions and windows that meet and do not."""
    b, kv, t_max, r = 75, 2, 2304, synth.rng(77)
    pos = [int(p) for p in r.integers(0, t_max - t, b)]
    pos[3], pos[10], pos[11], pos[40], pos[41] = 0, -1, t_max - t, 127, 128
    parents = np.array([tree(80 + s, t) for s in range(b)]) if kind == "tree" else None
    Call(dev, bf16, b, t, share * kv, kv, dq, dv, t_max, pos, parents=parents, sinks=70, window=2100).run().check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
def test_shapes_of_trees(dev, bf16, kind):
    """A chain is a causal block, a star sees its root, roots see no other node; across every border of 32 and 64 nodes."""
    t, pos = 128, [61, 0]
    parents = {"chain": np.arange(t) - 1, "star": np.minimum(np.arange(t) - 1, 0), "roots": np.full(t, -1)}[kind]
    Call(dev, bf16, 2, t, 4, 2, 64, 64, 200, pos, parents=np.array([parents] * 2)).run().check()


@pytest.mark.parametrize("bf16,d", [(False, 64), (True, 64), (True, 128)])
@pytest.mark.parametrize("t", [1, 3, 130])
@pytest.mark.parametrize("shift", [0, 1])
def test_one_key_stands_out(dev, bf16, d, t, shift):
    """A key that outweighs the others by exp(40), one at a time at the borders of window, first positions and tiles: queries that see it return its value,
    the others do not."""
    t_max, pos, sinks, window = 700, 400, 5, 200
    for far in (0, 4, 5, 63, 64, 200, 201, 202, 255, 256, 399, 400, 400 + t - 1):
        c = Call(dev, bf16, 1, t, 4, 2, d, d, t_max, [pos], sinks=sinks, window=window, shift=shift, spoil=False)
        q, k = np.zeros((1, t, 4, d)), 0.05 * synth.normal(3, (1, 2, t_max, d)).astype(f64)
        q[..., 5], k[..., 5] = 10.0, 0.0
        k[:, :, far, 5] = 4.0 * d ** 0.5 / 1.3
        for dst, x in ((0, q), (1, k)):
            host = np.r_[np.zeros(shift), x.ravel()].astype(np.float32)
            c.keep[dst].copy_host_to_device(synth.to_bf16_bits(host) if bf16 else host, bf16=bf16)
            c.values[dst] = (synth.bf16_bits_to_f32(synth.to_bf16_bits(host)) if bf16 else host).astype(f64)[shift:].reshape(x.shape)
        c.run().check()
        seen = c.masks[0][:, far]
        got = c.read()[0]
        assert np.max(np.abs(got[seen] - 0.7 * c.values[2][0, :, far].repeat(2, 0)), initial=0.0) < 0.03


@pytest.mark.parametrize("bf16", [False, True])
def test_large_scores_and_sums(dev, bf16):
    """Scores of some hundreds: the maximum has to run along; long rows: the sums stay in 32 bits."""
    Call(dev, bf16, 1, 40, 8, 2, 64, 64, 700, [600], sinks=3, window=650, std=60.0, seed=50).run().check()
    c = Call(dev, bf16, 1, 2, 4, 1, 64, 64, 70000, [69990], sinks=0, window=70000, std=0.0, seed=51).run()
    dev.synchronize()
    got, want = c.read()[0], 0.7 * np.stack([c.values[2][0, 0, :n].mean(0) for n in (69991, 69992)])
    # equal weights are exact in 16 bits; sums over tiles of 64: (70000 / 64 + 64) steps of an average |v| of 0.8 and a rounding
    assert (np.abs(got - want[:, None]) <= 1200 * 2.0 ** -24 * 0.8 + (2.0 ** -8 if bf16 else 2.0 ** -24) * np.abs(want[:, None])).all()


@pytest.mark.parametrize("bf16,d", [(False, 64), (True, 64), (True, 128)])
@pytest.mark.parametrize("shift", [0, 1])
def test_sequences_are_independent(dev, bf16, d, shift):
    """A sequence alone and in a batch, at another place and beside longer ones: the same to within the order of its sums."""
    pos = [500, 3, 130, 257]
    for parents in (None, np.array([tree(60 + s, 20) for s in range(4)])):
        kw = dict(parents=parents, sinks=0 if parents is not None else 3, window=0 if parents is not None else 150, shift=shift)
        Call(dev, bf16, 4, 20, 8, 2, d, d, 520, pos, **kw).run().check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t,t_max,pos,parents", [(3, 64, [62, 0], None), (3, 64, [-2, 0], None), (1, 64, [64, 0], None), (1, 64, [2 ** 31 - 1, 0], None),
                                                 (3, 64, [62, 0], [[-1, 0, 1]] * 2), (3, 64, [0, 0], [[0, 0, 1], [-1, 0, 0]]), (3, 64, [0, 0], [[-1, 2, 1], [-1, 0, 0]]),
                                                 (3, 64, [0, 0], [[-1, -2, 1], [-1, -1, -1]]), (40, 64, [5, 0], [list(range(40)), list(range(-1, 39))])])
def test_bad_positions_and_trees(dev, bf16, t, t_max, pos, parents):
    """The bad sequence is left as it was, the other one is done."""
    c = Call(dev, bf16, 2, t, 4, 2, 64, 64, t_max, [0, 0], sinks=1, window=10, spoil=False, parents=None if parents is None else np.array([[-1] * t, parents[1]]))
    c.pos_s = I32(dev, pos)
    if parents is not None:
        c.parents_s = I32(dev, parents)
    c.run()
    with pytest.raises(UgError) as e:
        dev.synchronize()
    assert e.value.code == 1
    c.masks[0] = None
    c.check()


def test_refusals(dev):
    z = lambda n: dev.zeros(n)
    i, h = I32(dev, [0] * 64), Buf(dev, True).out(4096)
    q, k, v, o = z(64), z(512), z(512), z(64)
    ok = [q, k, v, i, o, 1, 2, 4, 1, 8, 8, 64, 0, 4, 1.0]
    cases = [(2, {0: h, 4: h}), (2, {0: i, 4: i}), (2, {3: q}), (2, {4: h}), (2, {1: h}), (3, {0: z(60)}), (3, {4: z(60)}), (3, {1: z(511)}), (3, {11: 65}), (3, {6: 65, 11: 64}), (3, {7: 3, 8: 2}), (3, {8: 0}),
             (3, {9: 12}), (3, {10: 0}), (6, {9: 264, 0: z(4 * 2 * 264), 1: z(64 * 264)}), (1, {13: 0}), (1, {4: q}), (1, {4: k}), (3, {3: I32(dev, [0]), 5: 2, 6: 1})]
    for code, swap in cases:
        args = [swap.get(n, x) for n, x in enumerate(ok)]
        with pytest.raises(UgError) as e:
            dev.window_attend(*args)
        assert e.value.code == code, swap
        if code == 1 and 13 in swap:
            continue
        args[12:14] = []
        with pytest.raises(UgError) as e:
            dev.tree_attend(*args[:4], i, *args[4:])
        assert e.value.code == code, swap
    with pytest.raises(UgError) as e:
        dev.tree_attend(z(129 * 8), z(2048), z(2048), i, I32(dev, np.arange(129) - 1), z(129 * 8), 1, 129, 1, 1, 8, 8, 256, 1.0)
    assert e.value.code == 6
    with pytest.raises(UgError) as e:
        dev.tree_attend(q, k, v, i, q, o, 1, 2, 4, 1, 8, 8, 64, 1.0)
    assert e.value.code == 2
    dev.window_attend(q, k, v, i, o, 0, 2, 4, 1, 8, 8, 64, 0, 4, 1.0)
    dev.window_attend(q, k, v, i, o, 1, 0, 4, 1, 8, 8, 64, 0, 4, 1.0)
    assert lib.ugb_window_attend(None, *[None] * 5, 1, 1, 1, 1, 8, 8, 8, 0, 1, 1.0, 1.0) == 1
    assert lib.ugb_tree_attend(None, *[None] * 6, 1, 1, 1, 1, 8, 8, 8, 1.0, 1.0) == 1


@pytest.mark.parametrize("bf16", [False, True])
def test_captured_and_replayed(dev, bf16):
    """A graph of both operators, each with scratch of its own, replayed at positions that change on the device."""
    parents = np.array([tree(70 + s, 12) for s in range(2)])
    a = Call(dev, bf16, 2, 2, 8, 2, 64, 64, 600, [0, 0], sinks=2, window=400, spoil=False)
    b = Call(dev, bf16, 2, 12, 8, 2, 64, 64, 600, [0, 0], parents=parents, spoil=False)
    a.run()
    b.run()
    dev.synchronize()
    stream, graph = torch.cuda.ExternalStream(lib.ugb_device_stream(dev._h)), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a.run()
        b.run()
    for pos in ([500, 31], [7, 588]):
        for c in (a, b):
            c.pos_s.copy_host_to_device(np.array(pos, np.int32))
            c.masks = [window_mask(p, 2, 600, 2, 400) if c is a else tree_mask(p, parents[s], 600) for s, p in enumerate(pos)]
        with torch.cuda.stream(stream):
            graph.replay()
        a.check()
        b.check()
