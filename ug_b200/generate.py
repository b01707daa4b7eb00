"""Generation with any model of the registry, as a function and as a command:

    python -m ug_b200.generate --model DIR --prompt 12,7,99 [--prompt 3,1,4] -n 32 [--chunk 512] [--dtype float32]
        [--temperature 0.8 --top-k 40 --top-p 0.95 --min-p 0.05 --seed 1]

Token ids in, token ids out (a tokenizer is not part of this package).  Prompts of one call are the rows of a batch and
share their length; a prompt is fed in portions of ``chunk`` positions, then every new token is one graph-replayed step
whose input is the device-side choice after the previous one: the best token, or with any of the sampling options one drawn from
the random numbers of ``--seed``.
"""
import argparse
import sys

import numpy as np

from .device import DType, UgError

DTYPES = {"bfloat16": DType.BF16, "float32": DType.F32}


def generate(model, prompts, n_new, chunk=None, reset=True, u=None, temperature=None, top_k=None, top_p=None, min_p=None):
    """int32 [batch, n_new] continuations of ``prompts`` (int32 [batch, t]): greedy ones, or with ``u`` (f32 [n_new, batch], random
    numbers of [0, 1)) sampled ones; the other settings are those of :meth:`EngineModel.sample`."""
    prompts = np.ascontiguousarray(prompts, dtype=np.int32)
    if prompts.ndim != 2 or prompts.shape[0] != model.batch or prompts.shape[1] < 1:
        raise UgError(3, f"prompts must be [batch={model.batch}, t >= 1], got {prompts.shape}")
    if u is None:
        if any(x is not None for x in (temperature, top_k, top_p, min_p)):
            raise UgError(1, "sampling needs the random numbers u")
    else:
        u = np.ascontiguousarray(u, dtype=np.float32)
        if u.shape != (n_new, model.batch):
            raise UgError(3, f"u must be [n_new={n_new}, batch={model.batch}], got {u.shape}")
        draws = model.dev.slice_from_values(u.reshape(-1))
        rows = [model.dev.wrap(draws.device_ptr + 4 * model.batch * i, DType.F32, model.batch) for i in range(n_new)]
        settings = [model._per_row(x, d) for x, d in ((temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    if reset:
        model.reset()
    t = prompts.shape[1]
    for lo in range(0, t, chunk or t):
        model.prefill(prompts[:, lo:lo + (chunk or t)])
    out = np.empty((model.batch, n_new), np.int32)
    for i in range(n_new):
        if i:
            model.decode(1)
        if u is not None:
            model.sample(rows[i], *settings)
        out[:, i] = model.next_tokens()
    model.dev.synchronize()
    return out


def main(argv=None):
    ap = argparse.ArgumentParser(prog="python -m ug_b200.generate", description="generation from token ids")
    ap.add_argument("--model", required=True, help="folder with config.json and .safetensors files")
    ap.add_argument("--prompt", action="append", required=True, metavar="IDS", help="comma-separated token ids; repeat for a batch")
    ap.add_argument("-n", "--new-tokens", type=int, default=32)
    ap.add_argument("--chunk", type=int, default=None, help="positions of the prompt per portion")
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bfloat16")
    ap.add_argument("--device", type=int, default=0)
    ap.add_argument("--temperature", type=float, default=None, help="sample: divides the logits (0: the best token)")
    ap.add_argument("--top-k", type=int, default=None, help="sample among the k best tokens (0: all)")
    ap.add_argument("--top-p", type=float, default=None, help="sample among the best tokens that hold this share of the probability")
    ap.add_argument("--min-p", type=float, default=None, help="sample among tokens of at least this share of the best one's probability")
    ap.add_argument("--seed", type=int, default=None, help="of the random numbers (sampling without it: 0)")
    a = ap.parse_args(argv)
    sampled = any(x is not None for x in (a.temperature, a.top_k, a.top_p, a.min_p, a.seed))
    for name, x, ok in (("temperature", a.temperature, lambda x: 0 <= x <= 1e20), ("top-k", a.top_k, lambda x: 0 <= x < 2 ** 31),
                        ("top-p", a.top_p, lambda x: np.float32(x) > 0), ("min-p", a.min_p, lambda x: 0 <= x <= 1), ("seed", a.seed, lambda x: x >= 0)):
        if x is not None and not ok(x):
            ap.error(f"--{name} {x} is outside its range")
    from . import registry
    from .device import Device
    prompts = [[int(x) for x in p.split(",")] for p in a.prompt]
    if len({len(p) for p in prompts}) != 1:
        ap.error("the prompts of a batch must have one length")
    dev = Device(a.device)
    model = registry.load(a.model, dev, len(prompts), len(prompts[0]) + a.new_tokens, DTYPES[a.dtype])
    u = np.random.default_rng(a.seed or 0).random((a.new_tokens, len(prompts)), dtype=np.float32) if sampled else None
    for row in generate(model, np.array(prompts, np.int32), a.new_tokens, a.chunk, u=u, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p,
                        min_p=a.min_p):
        print(",".join(str(t) for t in row))
    model.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
