"""Generation with drafted trees, all operators together: head inputs by depth, attention over the cache and the ancestors, sampling at every node, the
accepted nodes' rows kept.  What is generated has to be what one token after the other gives."""
import numpy as np
import pytest

from hybrid_cases import Buf
from oracle import zidevik_ref as Z
from sampling_ref import choose
from test_draft_rows_gpu import I32
from ug_b200 import DType, synth

pytestmark = pytest.mark.gpu
VOCAB, WIDTH, HEADS, KV, T_MAX, BASE = 61, 96, 6, 2, 96, 200.0


class OneLayer:
    """Embedding, one attention layer, output head: projections on the host, attention over an exact cache in 64 bits."""

    def __init__(self, dim, seed=5):
        self.dim, r = dim, lambda i, *s: synth.normal(seed + i, s).astype(np.float64)
        self.embed = r(0, VOCAB, WIDTH)
        self.pre_w = r(1, WIDTH, (HEADS + 2 * KV) * dim) * WIDTH ** -0.5
        self.out_w = r(2, HEADS * dim, WIDTH) * (HEADS * dim) ** -0.5
        self.scale = 1.5 * dim ** -0.5

    def pre(self, tokens):
        return self.embed[tokens] @ self.pre_w

    def logits(self, tokens, attended):
        return (0.5 * self.embed[tokens] + 2.0 * attended.reshape(*np.shape(tokens), -1) @ self.out_w) @ self.embed.T * 0.3

    def full(self, tokens, window=None, sinks=0):
        """Logits of every position of one sequence."""
        t = len(tokens)
        x = self.pre(tokens)
        h = x[:, :(HEADS + KV) * self.dim].reshape(t, -1, self.dim)
        h = Z.rotate(h, np.arange(t), BASE, self.dim)
        q, k, v = h[:, :HEADS], h[:, HEADS:], x[:, (HEADS + KV) * self.dim:].reshape(t, KV, self.dim)
        k, v = (a.repeat(HEADS // KV, 1) for a in (k, v))
        s = np.einsum("ihd,jhd->hij", q, k) * self.scale
        i, j = np.arange(t)[:, None], np.arange(t)
        s[:, (j > i) | (j <= i - (window or t)) & (j >= sinks)] = -np.inf
        w = np.exp(s - s.max(-1, keepdims=True))
        return self.logits(np.array(tokens), np.einsum("hij,jhd->ihd", w / w.sum(-1, keepdims=True), v))


class OnDevice:
    def __init__(self, dev, bf16, model, batch):
        self.dev, self.B, self.m, self.batch = dev, Buf(dev, bf16), model, batch
        self.k, self.v = (self.B.act(np.full((batch, KV, T_MAX, model.dim), np.nan))[0] for _ in range(2))       # rows that nothing has written
        angle = np.arange(T_MAX)[:, None] * BASE ** (-2.0 * np.arange(model.dim // 2) / model.dim)
        self.cos, self.sin = self.B.f32(np.cos(angle)), self.B.f32(np.sin(angle))

    def nodes(self, pos, tokens, parents, window=None, sinks=0):
        """Logits [batch, t, vocab] of nodes at the cache's end, on the device."""
        d, t, dim = self.dev, tokens.shape[1], self.m.dim
        pos_s, par_s = I32(d, pos), I32(d, parents)
        q, out = self.B.out(self.batch * t * HEADS * dim), self.B.out(self.batch * t * HEADS * dim)
        d.tree_inputs(self.B.act(self.m.pre(tokens))[0], self.cos, self.sin, pos_s, par_s, q, self.k, self.v, self.batch, t, HEADS, KV, dim, dim, dim, True, False,
                      1e-5, T_MAX)
        if window is None:
            d.tree_attend(q, self.k, self.v, pos_s, par_s, out, self.batch, t, HEADS, KV, dim, dim, T_MAX, self.m.scale)
        else:
            d.window_attend(q, self.k, self.v, pos_s, out, self.batch, t, HEADS, KV, dim, dim, T_MAX, sinks, window, self.m.scale)
        return self.m.logits(tokens, self.B.read(out, (self.batch, t, HEADS, dim)))

    def sample(self, logits, u, **settings):
        rows = logits.reshape(-1, VOCAB).astype(np.float32)
        tokens = self.dev.allocate_uninit(DType.I32, len(rows))
        s = {n: self.dev.slice_from_values(np.full(len(rows), v, np.int32 if n == "top_k" else np.float32)) for n, v in settings.items()}
        self.dev.sample(self.B.f32(rows), self.B.f32(np.asarray(u)), tokens, len(rows), VOCAB, **s)
        got = tokens.to_vec()
        assert got.tolist() == [choose(x, float(np.float32(w)), **{n: int(v) if n == "top_k" else float(np.float32(v)) for n, v in settings.items()})[0]
                                for x, w in zip(rows, np.asarray(u).ravel())]
        return got.reshape(logits.shape[:-1])

    def keep(self, pos, paths, most):
        path = np.array([p + [0] * (most - len(p)) for p in paths], np.int32)
        self.dev.cache_keep(self.k, self.v, I32(self.dev, pos), I32(self.dev, path), I32(self.dev, [len(p) for p in paths]), self.batch, KV, self.m.dim, self.m.dim,
                            T_MAX, most)


def near(got, want, bf16):
    """f32: chains of a hundred products; bf16: inputs, keys, values, probabilities and outputs rounded to 2^-8 of a value of about the largest logit."""
    return np.max(np.abs(got - want)) <= (2.5e-2 if bf16 else 2e-5) * np.max(np.abs(want))


@pytest.mark.parametrize("bf16,dim", [(False, 24), (True, 64), (True, 128), (True, 40)])
def test_drafted_trees_give_what_single_steps_give(dev, bf16, dim):
    m, batch, most, draft = OneLayer(dim), 3, 4, synth.rng(9)
    d = OnDevice(dev, bf16, m, batch)
    prompt = synth.tokens(7, (batch, 11), VOCAB)
    u = synth.uniform(8, (batch, T_MAX), 0, 1)             # one random number per position, whoever draws there
    settings = dict(temperature=0.8, top_k=20, top_p=0.95)
    pos, rows = [0] * batch, [list(p) for p in prompt]
    logits = d.nodes(pos, prompt, [np.arange(11) - 1] * batch)
    assert all(near(logits[b], m.full(prompt[b]), bf16) for b in range(batch))
    pos = [11] * batch
    last = d.sample(logits[:, -1], u[:, 10], **settings)
    accepted = 0
    for _ in range(6):
        # the root is the last token; below it a guess that is right two times out of three, beside wrong ones, three levels deep
        tokens, parents = np.empty((batch, 13), np.int64), np.empty((batch, 13), np.int64)
        for b in range(batch):
            t, p, level, seq = [int(last[b])], [-1], [0], list(rows[b]) + [int(last[b])]
            for depth in range(most - 1):
                x = m.full(seq)[-1].astype(np.float32)
                right = choose(x, float(u[b, pos[b] + depth]), **{n: float(np.float32(v)) if n != "top_k" else v for n, v in settings.items()})[0]
                guesses = [right if draft.random() < 0.67 else int(draft.integers(VOCAB))] + [int(g) for g in draft.integers(0, VOCAB, 3)]
                draft.shuffle(guesses)
                at = level[0] if depth == 0 else len(t) - 4 + chosen
                chosen = guesses.index(right) if right in guesses else 0
                for g in guesses:
                    t.append(g)
                    p.append(at)
                seq.append(right)
            tokens[b], parents[b] = t, p
        logits = d.nodes(pos, tokens, parents)
        depth = np.zeros((batch, 13), np.int64)
        for i in range(1, 13):
            depth[:, i] = depth[np.arange(batch), parents[:, i]] + 1
        choice = d.sample(logits, np.take_along_axis(u, np.array(pos)[:, None] + depth, 1), **settings)
        paths = []
        for b in range(batch):
            path, node = [], 0
            while node is not None:
                path.append(node)
                assert near(logits[b, node], m.full(rows[b] + [int(tokens[b, n]) for n in path])[-1], bf16)
                below = [i for i in range(13) if parents[b, i] == node and tokens[b, i] == choice[b, node]]
                node = below[0] if below and len(path) < most else None
            rows[b] += [int(tokens[b, n]) for n in path]
            last[b] = choice[b, path[-1]]
            paths.append(path)
            accepted += len(path)
        d.keep(pos, paths, most)
        pos = [p + len(q) for p, q in zip(pos, paths)]
    assert accepted > 6 * batch                            # drafts were taken
    dev.synchronize()
    for b in range(batch):                                 # and a step after all that, by one token
        assert len(rows[b]) == pos[b]
    logits = d.nodes(pos, np.array(last)[:, None], [[-1]] * batch)
    assert all(near(logits[b, 0], m.full(rows[b] + [int(last[b])])[-1], bf16) for b in range(batch))


@pytest.mark.parametrize("bf16,dim", [(False, 24), (True, 64), (True, 128)])
def test_windowed_portions_and_steps(dev, bf16, dim):
    """A prompt in portions of any length and single steps behind it: every position sees its window and the first positions."""
    m, batch, window, sinks = OneLayer(dim), 2, 9, 3
    d = OnDevice(dev, bf16, m, batch)
    tokens = synth.tokens(11, (batch, 60), VOCAB)
    want = [m.full(tokens[b], window, sinks) for b in range(batch)]
    at = 0
    for n in (1, 17, 2, 30, 1, 1, 8):
        got = d.nodes([at] * batch, tokens[:, at:at + n], [np.arange(n) - 1] * batch, window, sinks)
        assert all(near(got[b], want[b][at:at + n], bf16) for b in range(batch))
        at += n
    dev.synchronize()
