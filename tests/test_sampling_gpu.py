"""Sampling through the C ABI against its definition in 64 bits (sampling_ref.py): tokens equal, shares within a rounding to 32 bits
(2^-24 of the value) and the unit of the sums (2^-45 of the best weight for each of the vocabulary's tokens at most, twice for numerator and
total)."""
import numpy as np
import pytest
import torch

from sampling_ref import choose
from ug_b200 import DType, UgError, synth
from ug_b200._lib import lib
from ug_b200.kabidra import Config, Layer, Model

pytestmark = pytest.mark.gpu
SETTINGS = ("temperature", "top_k", "top_p", "min_p")


def sample(dev, x, u, bf16=False, ld=None, logits=None, **settings):
    """(tokens, prob) of the rows of x; settings are arrays of one value per row."""
    rows, vocab = x.shape
    if logits is None:
        logits = dev.slice_from_values(synth.to_bf16_bits(x).ravel() if bf16 else x.astype(np.float32).ravel(), bf16=bf16)
    s = {n: dev.slice_from_values(np.asarray(v, np.int32 if n == "top_k" else np.float32)) for n, v in settings.items()}
    tokens, prob = dev.slice_from_values(np.full(rows, -7, np.int32)), dev.slice_from_values(np.full(rows, -7, np.float32))
    dev.sample(logits, dev.slice_from_values(np.asarray(u, np.float32)), tokens, rows, vocab, prob=prob, ld=ld, **s)
    return tokens, prob


def check(dev, x, u, bf16=False, **settings):
    if bf16:
        x = synth.bf16_bits_to_f32(synth.to_bf16_bits(np.asarray(x, np.float32)))
    x = np.asarray(x, np.float32)
    tokens, prob = sample(dev, x, u, bf16, **settings)
    dev.synchronize()
    tokens, prob = tokens.to_vec(), prob.to_vec()
    for r in range(len(x)):
        token, share = choose(x[r], float(np.float32(u[r])), **{n: (int if n == "top_k" else lambda a: float(np.float32(a)))(v[r]) for n, v in settings.items()})
        assert tokens[r] == token, (r, {n: v[r] for n, v in settings.items()})
        assert abs(prob[r] - share) <= 2.0 ** -24 * share * 1.01 + x.shape[1] * 2.0 ** -44


def logits_of(seed, rows, vocab, std=2.5):
    return synth.normal(seed, (rows, vocab), std)


def mixed(seed, rows, vocab):
    """Settings of every kind, off ones among them."""
    r = synth.rng(seed)
    pick = lambda on, off, share: np.where(r.random(rows) < share, off, on)
    return dict(temperature=pick(r.uniform(0.3, 2.0, rows), 0.0, 0.1).astype(np.float32), top_k=pick(r.integers(1, 2 * vocab + 1, rows), 0, 0.4).astype(np.int32),
                top_p=pick(r.uniform(0.05, 1.0, rows), 1.0, 0.4).astype(np.float32), min_p=pick(r.uniform(0, 0.2, rows), 0.0, 0.5).astype(np.float32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 2), (40, 17), (33, 513), (64, 4099), (9, 32000), (160, 1024), (3, 50257), (2, 131075), (1, 262144)])
def test_against_the_definition(dev, bf16, rows, vocab):
    u = synth.uniform(1, (rows,), 0.0, 1.0)
    check(dev, logits_of(2, rows, vocab), np.minimum(u, 1 - 2.0 ** -24), bf16, **mixed(3, rows, vocab))


@pytest.mark.parametrize("settings", [dict(), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=50, top_p=0.5),
                                      dict(temperature=1.5, top_k=300, min_p=0.01), dict(top_p=1e-6), dict(min_p=1.0), dict(top_k=1), dict(temperature=1e-30),
                                      dict(top_p=3.0, top_k=2 ** 31 - 1)])
def test_each_setting_alone(dev, settings):
    """Over the whole range of random numbers, its ends among them."""
    rows, vocab = 65, 2000
    u = np.r_[np.linspace(0, 1, rows - 1, endpoint=False), 1 - 2.0 ** -24]
    check(dev, np.tile(logits_of(4, 1, vocab), (rows, 1)), u, **{n: [v] * rows for n, v in settings.items()})


@pytest.mark.parametrize("vocab", [7, 600, 40000])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.37), dict(top_k=5, top_p=0.5), dict(min_p=1.0), dict(temperature=0.0)])
def test_equal_logits_go_by_index(dev, vocab, settings):
    u = np.r_[0.0, 0.2, 0.5, 0.77, 1 - 2.0 ** -24]
    x = np.full((5, vocab), 1.25)
    x[1, vocab // 2:] = -3.0
    x[2] = np.arange(vocab) % 2
    x[3] = 0.0
    x[3, ::2] = -0.0                                       # equal to 0
    check(dev, x, u, **{n: [v] * 5 for n, v in settings.items()})


@pytest.mark.parametrize("vocab", [9, 20001])
def test_masked_logits(dev, vocab):
    """-inf, NaN, the lowest value and +inf in masked places; rows of nothing, of one token, of few."""
    low = np.finfo(np.float32).min
    x = logits_of(5, 10, vocab)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[2, vocab - 1] = -5.0
    x[3] = low
    x[4, ::2] = -np.inf
    x[5, 1::2] = np.nan
    x[6, : vocab - 2] = low
    x[7, 3] = x[7, 5] = np.inf
    x[8] = np.inf
    x[9, 2:] = -np.inf
    x[3, 1::3] = -np.inf
    u = np.full(10, 0.6)
    for settings in (dict(), dict(top_k=4), dict(top_p=0.8), dict(top_k=vocab - 1, top_p=0.9, min_p=0.05), dict(temperature=0.0)):
        check(dev, x, u, **{n: [v] * 10 for n, v in settings.items()})


def test_wide_range_of_values(dev):
    """Logits of many orders of magnitude on both sides of zero, and neighbours that differ by one unit."""
    x = np.concatenate([s * 2.0 ** np.arange(-126, 12) for s in (-1, 1)]).astype(np.float32)[None].repeat(8, 0)
    x[4:] = np.nextafter(np.float32(8), np.float32(9)) + np.arange(x.shape[1], dtype=np.float32) * np.float32(2.0 ** -20)
    u = np.tile([0.1, 0.5, 0.9, 0.999], 2)
    for settings in (dict(temperature=1e20), dict(temperature=1e-45, top_p=0.5), dict(top_k=10), dict(temperature=300.0, top_p=0.9), dict(temperature=1e4, top_k=200, top_p=0.7)):
        check(dev, x, u, **{n: [v] * 8 for n, v in settings.items()})


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_apart_and_unaligned(dev, bf16, shift):
    """Rows ld apart whose gaps hold large values, from a base that is no multiple of 16 bytes."""
    rows, vocab, ld = 5, 1003, 1007
    x = logits_of(6, rows, vocab)
    full = np.full(shift + rows * ld, 1e30, np.float32)
    for r in range(rows):
        full[shift + r * ld:shift + r * ld + vocab] = x[r]
    s = dev.slice_from_values(synth.to_bf16_bits(full) if bf16 else full, bf16=bf16)
    part = dev.wrap(s.device_ptr + shift * (2 if bf16 else 4), s.dtype, len(full) - shift - (ld - vocab))
    settings = dict(top_k=[100] * rows, top_p=[0.9] * rows)
    u = np.linspace(0, 0.99, rows)
    got = sample(dev, x, u, ld=ld, logits=part, **settings)
    want = sample(dev, x, u, bf16, **settings)
    assert np.array_equal(got[0].to_vec(), want[0].to_vec()) and np.array_equal(got[1].to_vec(), want[1].to_vec())


@pytest.mark.parametrize("vocab", [7000, 12000])
def test_a_row_is_the_same_in_any_batch(dev, vocab):
    """However many CTAs share a row: 1, 2 or 4."""
    n = 4
    x, u, s = logits_of(7, n, vocab, 1.0), synth.uniform(8, (n,), 0, 1), dict(temperature=[1.3] * n, top_k=[0, 5000, 0, 0], top_p=[1, 0.9, 0.99, 0.5])
    one = [sample(dev, x[i:i + 1], u[i:i + 1], **{k: v[i:i + 1] for k, v in s.items()}) for i in range(n)]
    for times in (8, 80, 160):
        tokens, prob = sample(dev, np.tile(x, (times, 1)), np.tile(u, times), **{k: list(v) * times for k, v in s.items()})
        assert tokens.to_vec().tolist() == [int(t.to_vec()[0]) for t, _ in one] * times
        assert prob.to_vec().tolist() == [float(p.to_vec()[0]) for _, p in one] * times


@pytest.mark.parametrize("name,value", [("temperature", -0.5), ("temperature", np.nan), ("temperature", np.inf), ("temperature", 2e20), ("top_k", -1), ("top_p", 0.0), ("top_p", np.nan),
                                        ("min_p", -0.1), ("min_p", 1.5), ("min_p", np.nan), ("u", 1.0), ("u", -0.1), ("u", np.nan)])
def test_values_outside_their_range(dev, name, value):
    """The row is left as it was, the others are done."""
    x = logits_of(9, 3, 700)
    given = dict(temperature=[1.0] * 3, top_k=[5] * 3, top_p=[0.9] * 3, min_p=[0.1] * 3, u=[0.3] * 3)
    want = sample(dev, x, **{k: list(v) for k, v in given.items()})[0].to_vec()
    given[name][1] = value
    tokens, prob = sample(dev, x, **given)
    with pytest.raises(UgError) as e:
        dev.synchronize()
    assert e.value.code == 1
    assert tokens.to_vec().tolist() == [want[0], -7, want[2]] and prob.to_vec()[1] == -7


def test_refusals(dev):
    x, u, t = dev.zeros(64), dev.zeros(2), dev.allocate_uninit(DType.I32, 2)
    for code, call in ((2, lambda: dev.sample(t, u, t, 1, 2)),                                    # logits of a type without a kernel
                       (2, lambda: dev.sample(x, u, u, 2, 32)), (2, lambda: dev.sample(x, t, t, 2, 32)),
                       (2, lambda: dev.sample(x, u, t, 2, 32, top_k=u)), (3, lambda: dev.sample(x, u, t, 2, 33)),
                       (3, lambda: dev.sample(x, u, t, 3, 16)), (3, lambda: dev.sample(x, u, t, 1, 32, ld=16)), (3, lambda: dev.sample(x, u, t, 2, 0)),
                       (6, lambda: dev.sample(x, u, t, 0, 262145)), (3, lambda: dev.sample(x, u, t, 2, 32, prob=dev.zeros(1))),
                       (1, lambda: dev.sample(x, u, t, 2, 32, prob=x))):
        with pytest.raises(UgError) as e:
            call()
        assert e.value.code == code
    dev.sample(x, u, t, 0, 32)                             # no rows: nothing happens
    assert lib.ugb_sample(None, *[None] * 8, 1, 1, 1) == 1


def test_captured_and_replayed(dev):
    """A graph of two calls reads new logits and random numbers at each replay."""
    rows, vocab = 3, 5000
    bufs = [dev.zeros(rows * vocab), dev.zeros(rows)]
    outs = [dev.allocate_uninit(DType.I32, rows) for _ in range(2)]
    p = dev.slice_from_values(np.full(rows, 0.8, np.float32))
    dev.sample(bufs[0], bufs[1], outs[0], rows, vocab)
    dev.synchronize()
    stream, graph = torch.cuda.ExternalStream(lib.ugb_device_stream(dev._h)), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        dev.sample(bufs[0], bufs[1], outs[0], rows, vocab)
        dev.sample(bufs[0], bufs[1], outs[1], rows, vocab, top_p=p)
    for seed in (10, 11):
        x, u = logits_of(seed, rows, vocab), synth.uniform(seed + 5, (rows,), 0, 1)
        bufs[0].copy_host_to_device(x.ravel())
        bufs[1].copy_host_to_device(u)
        with torch.cuda.stream(stream):
            graph.replay()
        dev.synchronize()
        assert outs[0].to_vec().tolist() == [choose(x[r], float(u[r]))[0] for r in range(rows)]
        assert outs[1].to_vec().tolist() == [choose(x[r], float(u[r]), top_p=float(np.float32(0.8)))[0] for r in range(rows)]


def small_model(dev, batch, dtype=DType.F32):
    cfg = Config(vocab=320, width=112, eps=1e-5, taps=3, layers=[Layer("mingru", {"width": 144}, 160)])
    return Model.new(cfg, synth.kabidra_weights(cfg, 21), dev, batch, 64, dtype)


def test_models_feed_the_sampled_tokens(dev):
    """The choice is that of the definition on the logits that the model reports, and the next step is the one that an explicit token gives."""
    batch, prompt = 3, synth.tokens(12, (3, 9), 320)
    m, other = small_model(dev, batch), small_model(dev, batch)
    with pytest.raises(UgError):
        m.sample(0.5)                                      # nothing to sample from yet
    prob = dev.zeros(batch)
    m.prefill(prompt)
    other.prefill(prompt)
    for i in range(4):
        u, x = synth.uniform(30 + i, (batch,), 0, 1), m.logits()
        m.sample(u, temperature=1.2, top_k=[5, 0, 50], top_p=0.95, prob=prob)
        want = [choose(x[r], float(u[r]), float(np.float32(1.2)), [5, 0, 50][r], float(np.float32(0.95))) for r in range(batch)]
        assert m.next_tokens().tolist() == [t for t, _ in want]
        assert np.allclose(prob.to_vec(), [p for _, p in want], rtol=2.0 ** -23, atol=320 * 2.0 ** -44)
        m.decode(1)
        other.fwd(np.array([t for t, _ in want], np.int32))
        assert np.array_equal(m.logits(), other.logits())


def test_llama_feeds_the_sampled_tokens(dev):
    """The same of the Llama engine, through its captured step too."""
    from ug_b200 import llama
    cfg = llama.Config(hidden_size=256, intermediate_size=512, max_position_embeddings=128, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2, vocab_size=512)
    w, prompt = synth.llama_weights(cfg, 11), synth.tokens(15, (3, 7), 512)
    m, other = (llama.Model.new(cfg, w, dev, 3, 64) for _ in range(2))
    with pytest.raises(UgError):
        m.sample(0.5)
    m.prefill(prompt)
    other.prefill(prompt)
    for i in range(4):
        u, x = synth.uniform(40 + i, (3,), 0, 1), m.logits()
        m.sample(u, temperature=[1.5, 0.0, 0.7], top_k=100, min_p=0.01)
        want = [choose(x[r], float(u[r]), [1.5, 0.0, float(np.float32(0.7))][r], 100, 1.0, float(np.float32(0.01)))[0] for r in range(3)]
        assert m.next_tokens().tolist() == want
        m.decode(1)
        other.fwd(np.array(want, np.int32))
        assert np.array_equal(m.logits(), other.logits())
    m.close()
    other.close()
    assert lib.ugb_llama_sample(None, *[None] * 6) == 1 and lib.ugb_hybrid_sample(None, *[None] * 6) == 1


def test_generate_with_random_numbers(dev):
    from ug_b200.generate import generate
    m = small_model(dev, 2)
    prompt, u = synth.tokens(13, (2, 5), 320), synth.uniform(14, (6, 2), 0, 1)
    got = generate(m, prompt, 6, u=u, temperature=0.9, top_k=40)
    m.reset()
    m.prefill(prompt)
    for i in range(6):
        x = m.logits()
        want = [choose(x[r], float(u[i, r]), float(np.float32(0.9)), 40)[0] for r in range(2)]
        assert got[:, i].tolist() == want
        m.fwd(np.array(want, np.int32))
    m.logits()
    assert np.array_equal(generate(m, prompt, 6, u=u, top_k=1), generate(m, prompt, 6))
    with pytest.raises(UgError):
        generate(m, prompt, 6, temperature=0.9)
    with pytest.raises(UgError):
        generate(m, prompt, 6, u=u[:5])
