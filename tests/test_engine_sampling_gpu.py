"""Sampling over an engine's logits: where there are none, one sequence, a tensor-parallel rank."""
import numpy as np
import pytest

from sampling_ref import choose
from test_sampling_gpu import small_model
from ug_b200 import UgError, llama, synth

pytestmark = pytest.mark.gpu


def llama_model(dev, batch):
    cfg = llama.Config(hidden_size=256, intermediate_size=512, max_position_embeddings=128, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2, vocab_size=512)
    return llama.Model.new(cfg, synth.llama_weights(cfg, 11), dev, batch, 64)


def refused(m):
    with pytest.raises(UgError) as e:
        m.sample(0.5)
    assert e.value.code == 1


def test_a_position_alone_is_not_a_step(dev):
    """reset(pos > 0) leaves no logits of that position, on a fresh model and on a used one."""
    m = llama_model(dev, 2)
    m.reset(5)
    refused(m)
    prompt = synth.tokens(3, (2, 9), 512)
    m.reset()
    m.prefill(prompt)
    m.sample(0.5)
    m.reset(9)                                             # the position that the logits are of
    m.sample(0.5)
    m.reset(4)
    refused(m)
    m.fwd(prompt[:, 4])
    m.sample(0.5)
    m.reset()
    refused(m)
    m.decode(2)
    m.sample(0.5)
    dev.synchronize()
    m.close()


def test_a_recurrent_model_that_starts_again(dev):
    m = small_model(dev, 2)
    m.reset()
    refused(m)
    m.prefill(synth.tokens(3, (2, 9), 320))
    m.sample(0.5)
    m.reset(9)
    m.sample(0.5)
    m.reset()
    refused(m)
    m.fwd(np.array([1, 2], np.int32))
    m.sample(0.5)
    dev.synchronize()
    m.close()


def test_logits_of_a_timed_kernel_are_nobodys(dev):
    m = small_model(dev, 1)
    m.prefill(synth.tokens(3, (1, 9), 320))
    m.fwd(np.array([1], np.int32))
    m.sample(0.5)
    m.time_kernel("head", 1, 1)
    refused(m)
    m.reset()
    m.prefill(synth.tokens(3, (1, 9), 320))
    m.sample(0.5)
    dev.synchronize()
    m.close()


def test_one_sequence(dev):
    """The Llama engine's steps of one sequence, through the captured step too."""
    m, other, prompt = llama_model(dev, 1), llama_model(dev, 1), synth.tokens(15, (1, 7), 512)
    m.prefill(prompt)
    other.prefill(prompt)
    for i in range(4):
        u, x = synth.uniform(60 + i, (1,), 0, 1), m.logits()
        m.sample(u, temperature=1.5, top_k=100, top_p=0.9)
        want = choose(x[0], float(u[0]), 1.5, 100, float(np.float32(0.9)))[0]
        assert m.next_tokens().tolist() == [want]
        m.decode(1)
        other.fwd(np.array([want], np.int32))
        assert np.array_equal(m.logits(), other.logits())
    m.close()
    other.close()


def test_a_tensor_parallel_rank_is_refused(dev):
    cfg = llama.Config(hidden_size=256, intermediate_size=512, max_position_embeddings=128, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2, vocab_size=512)
    m = llama.Model(cfg, dev, 2, 64, tp=(0, 2))            # a rank that has not met its peer: nothing runs
    with pytest.raises(UgError) as e:
        m.sample(0.5)
    assert e.value.code == 6
    m.close()
