"""The operators of generation beyond greedy steps, as cases that can be timed and checked.

`kind` says which operator a case runs; T is bf16 or f32, lengths of a batch are ragged:

  sample       rows, vocab, dtype, filters       one token per row of logits from given random numbers
  window       b, t, depth, sinks, window, ...   attention of t new positions over a cache, a sliding window and the first keys
  tree_inputs  b, t, depth, ...                  rotary positions by depth and cache append of t drafted nodes
  tree         b, t, depth, ...                  attention of t drafted nodes, each over the cache and its ancestors
  keep         b, nodes, most, depth, ...        the accepted nodes' cache rows moved behind the committed ones

Head layouts and vocabularies are those of the package's benchmark models or generic.
"""
import math
import random

import torch

own = False

_T = {"bf16": torch.bfloat16, "f32": torch.float32}


def _heads(heads, kv_heads, dq, dv, dtype="bf16"):
    return dict(heads=heads, kv_heads=kv_heads, dq=dq, dv=dv, dtype=dtype)


def listed():
    llama = _heads(32, 4, 64, 64)               # the 1.1B benchmark model
    wide = _heads(32, 8, 128, 128)
    return [
        # one user's chat: the token after a step of the benchmark model
        dict(name="sample_1x32000", kind="sample", rows=1, vocab=32000, dtype="f32", filters="all"),
        # a serving batch, every request with settings of its own, some greedy
        dict(name="sample_64x32000", kind="sample", rows=64, vocab=32000, dtype="f32", filters="mixed"),
        # 16-bit logits of a large vocabulary, full of equal values: a batch of rollouts with nothing but a nucleus
        dict(name="sample_256x131072", kind="sample", rows=256, vocab=131072, dtype="bf16", filters="nucleus"),
        # a step of a serving batch deep in its sequences
        dict(name="window_64x1_8192", kind="window", b=64, t=1, depth=8192, sinks=4, window=4096, **llama),
        # a document's next portion
        dict(name="window_4x2048_4096", kind="window", b=4, t=2048, depth=2048, sinks=16, window=1024, **wide),
        # the 32-bit form on a prompt of odd length that fills no tile
        dict(name="window_f32_1x777", kind="window", b=1, t=777, depth=200, sinks=5, window=333, **_heads(32, 4, 64, 64, "f32")),
        # one user's step with a tree of drafts
        dict(name="tree_1x24_2000", kind="tree", b=1, t=24, depth=2000, **llama),
        # a serving batch of large trees over deep caches
        dict(name="tree_16x64_8192", kind="tree", b=16, t=64, depth=8192, **wide),
        # what goes ahead of each of the two
        dict(name="tree_inputs_1x24", kind="tree_inputs", b=1, t=24, depth=2000, rot=64, interleaved=False, norm=False, **llama),
        dict(name="tree_inputs_64x64", kind="tree_inputs", b=64, t=64, depth=1024, rot=128, interleaved=True, norm=True, **wide),
        # and what comes behind the choice
        dict(name="keep_1x24_2000", kind="keep", b=1, nodes=24, most=6, depth=2000, **llama),
        dict(name="keep_64x64_1024", kind="keep", b=64, nodes=64, most=12, depth=1024, **wide),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "window", "window", "window", "tree", "tree", "tree_inputs", "keep"])
    if kind == "sample":
        vocab = _log(rng, 500, 200000)
        return dict(kind=kind, rows=_log(rng, 1, min(512, (1 << 25) // vocab)), vocab=vocab, dtype=rng.choice(["f32", "f32", "bf16"]),
                    filters=rng.choice(["all", "mixed", "mixed", "nucleus", "top", "none"]))
    f32 = rng.random() < 0.25
    share, kv = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 16]), rng.choice([1, 2, 4, 4, 8])
    dq, dv = rng.choice([(64, 64), (64, 64), (128, 128), (128, 128), (64, 128), (128, 64)] if not f32 else [(64, 64), (128, 128), (80, 80), (72, 40)])
    if not f32 and rng.random() < 0.1:
        dq, dv = 96, 96
    dims = _heads(share * kv, kv, dq, dv, "f32" if f32 else "bf16")
    t = 1 if kind == "window" and rng.random() < 0.4 else _log(rng, 2, 2048) if kind == "window" else rng.randint(1, rng.choice([32, 128]))
    # no more pairs of queries and keys, and no larger caches, than the largest listed cases have
    pairs = (1 << (26 if f32 or dq == 96 else 28)) // (share * kv * t)
    depth = _log(rng, 1, max(1, min(16384 if kind in ("window", "tree") else 2048, pairs - t)))
    most = min(pairs // (depth + t), (1 << 28) // (kv * (depth + t) * (dq + dv)), 25_000_000 // (t * (share + 2) * kv * dq))
    dims.update(b=_log(rng, 1, max(1, min(64, most))), depth=depth)
    if kind == "window":
        return dict(kind=kind, t=t, sinks=rng.choice([0, 1, 4, 16, 100]), window=_log(rng, 1, 8192), **dims)
    if kind == "tree":
        return dict(kind=kind, t=t, **dims)
    if kind == "tree_inputs":
        return dict(kind=kind, t=t, rot=rng.choice([0, dq // 2, dq, dq]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5, **dims)
    return dict(kind=kind, nodes=t, most=rng.randint(1, min(t, 16)), **dims)


# ------------------------------------------------------------------ inputs ---
def _normal(gen, shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _uniform(gen, shape, lo=0.0, hi=1.0):
    return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=gen)


def _whole(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(rng, case):
    """Committed positions of every sequence: one of the full depth, the others down to half of it."""
    return [case["depth"]] + [rng.randint(case["depth"] // 2, case["depth"]) for _ in range(case["b"] - 1)]


def _tree(rng, t):
    """Parents of t nodes as a drafter lists them: level by level, likely nodes have the children."""
    parents, level = [-1], [0]
    while len(parents) < t:
        nxt = []
        for at, node in enumerate(level):
            for _ in range(rng.choice([4, 3, 2] if at == 0 else [2, 1, 1, 0])):
                if len(parents) < t:
                    nxt.append(len(parents))
                    parents.append(node)
        level = nxt or [len(parents) - 1]
    return parents


def _t_max(case):
    return (case["depth"] + case.get("t", case.get("nodes", 0)) + 15) // 16 * 16


def prepare(case, seed):
    gen, rng = torch.Generator("cuda").manual_seed(seed), random.Random(seed)
    s, kind = dict(case), case["kind"]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = _normal(gen, (rows, vocab), std=2.0)             # most of a vocabulary is noise, some tokens stand out
        some = torch.randint(0, vocab, (rows, 32), device="cuda", generator=gen)
        s["logits"] = x.scatter_add(1, some, _uniform(gen, (rows, 32), 2.0, 9.0)).to(_T[case["dtype"]])
        s["u"] = _uniform(gen, (rows,)).clamp(max=1 - 2.0 ** -24)
        f = case["filters"]
        every = {"temperature": _uniform(gen, (rows,), 0.6, 1.3), "top_k": torch.randint(1, 200, (rows,), device="cuda", generator=gen, dtype=torch.int32),
                 "top_p": _uniform(gen, (rows,), 0.7, 0.99), "min_p": _uniform(gen, (rows,), 0.0, 0.1)}
        if f == "mixed":                                     # 0 and 1 stand for a filter that is off, a temperature of 0 for the best token
            off = _uniform(gen, (4, rows))
            every["temperature"][off[0] < 0.2] = 0.0
            every["top_k"][off[1] < 0.5] = 0
            every["top_p"][off[2] < 0.4] = 1.0
            every["min_p"][off[3] < 0.5] = 0.0
        has = {"all": every, "mixed": every, "nucleus": ("temperature", "top_p"), "top": ("temperature", "top_k"), "none": ("temperature",)}[f]
        s.update({n: every[n] if n in has else None for n in every})
        s["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["prob"] = torch.empty(rows, device="cuda")
        return s
    dtype, b, kv, dq, dv, t_max = _T[case["dtype"]], case["b"], case["kv_heads"], case["dq"], case["dv"], _t_max(case)
    s["pos"] = _whole(_lengths(rng, case))
    s["k"], s["v"] = _normal(gen, (b, kv, t_max, dq), dtype), _normal(gen, (b, kv, t_max, dv), dtype)
    if kind in ("tree", "tree_inputs"):
        s["parents"] = _whole([_tree(rng, case["t"]) for _ in range(b)])
    if kind in ("tree", "window"):
        s["q"] = _normal(gen, (b, case["t"], case["heads"], dq), dtype, 1.5)
        s["out"] = torch.empty((b, case["t"], case["heads"], dv), dtype=dtype, device="cuda")
    elif kind == "tree_inputs":
        s["pre"] = _normal(gen, (b, case["t"], (case["heads"] + kv) * dq + kv * dv), dtype)
        half = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        angle = torch.arange(t_max, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2.0 * half / max(1, case["rot"]))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q"] = torch.empty((b, case["t"], case["heads"], dq), dtype=dtype, device="cuda")
    else:
        # accepted nodes: the root and then nodes of deeper levels, which lie behind the rows that are written
        most, nodes, count, path = case["most"], case["nodes"], [], []
        for _ in range(b):
            n = min(rng.randint(1, most), 1 + max(0, nodes - most))
            p = [0] + sorted(rng.sample(range(most, nodes), n - 1)) if n > 1 else [0]
            count.append(n)
            path.append(p + [0] * (most - n))
        s["path"], s["count"] = _whole(path), _whole(count)
    return s


# ------------------------------------------------------------ the plain forms ---
def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    one = torch.ones(rows, 1, dtype=torch.float64, device=x.device)
    arg = lambda n, off: one * off if s[n] is None else s[n].double()[:, None]
    temperature, top_k, top_p, min_p = arg("temperature", 1), arg("top_k", 0), arg("top_p", 1), arg("min_p", 0)
    best = x.max(1, keepdim=True).values
    weight = torch.exp((x - best) / torch.where(temperature > 0, temperature, one))
    order = s["logits"].float().sort(dim=1, descending=True, stable=True).indices
    w = weight.gather(1, order)
    keep = (top_k == 0) | (torch.arange(vocab, device=x.device)[None] < top_k)
    w = w * keep
    total = w.sum(1, keepdim=True)
    keep = keep & ((top_p >= 1) | (w.cumsum(1) - w < top_p * total)) & (w >= min_p)
    kept = weight * torch.zeros_like(keep).scatter_(1, order, keep)
    running = kept.cumsum(1)
    total = running[:, -1:]
    token = (running <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    prob = kept.gather(1, token) / total
    greedy = temperature == 0
    token = torch.where(greedy, (x == best).to(torch.uint8).argmax(1, keepdim=True), token)
    return {"tokens": token[:, 0].to(torch.int32), "prob": torch.where(greedy, one, prob)[:, 0].float()}


def _plain_closure(parents):
    """[b, t, t]: whether node j is node i itself or an ancestor of it."""
    t = parents.shape[1]
    up = (parents[:, :, None] == torch.arange(t, device=parents.device)).double() + torch.eye(t, dtype=torch.float64, device=parents.device)
    return torch.linalg.matrix_power(up, 127) > 0


def _plain_attention(s):
    q, k, v, b, t = s["q"].float(), s["k"].float(), s["v"].float(), s["b"], s["t"]
    n = s["depth"] + t
    j, pos = torch.arange(n, device=q.device), s["pos"].long()
    if s["kind"] == "window":
        at = pos[:, None] + torch.arange(t, device=q.device)
        seen = (j <= at[..., None]) & ((j < s["sinks"]) | (j > at[..., None] - s["window"]))
    else:
        node = j - pos[:, None]                              # [b, n]
        mine = _plain_closure(s["parents"]).gather(2, node.clamp(0, t - 1)[:, None].expand(b, t, n))
        seen = (node < 0)[:, None] | ((node >= 0) & (node < t))[:, None] & mine
    share = s["heads"] // s["kv_heads"]
    rows = q.view(b, t, s["kv_heads"], share, -1).permute(0, 2, 1, 3, 4).reshape(b, s["kv_heads"], t * share, -1)
    score = (rows @ k[:, :, :n].transpose(2, 3)).view(b, s["kv_heads"], t, share, n).mul_(s["dq"] ** -0.5)
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(b, s["kv_heads"], t * share, n)
    out = (p @ v[:, :, :n]).view(b, s["kv_heads"], t, share, -1).permute(0, 2, 1, 3, 4)
    return out.reshape(b, t, s["heads"], -1).to(s["q"].dtype)


def _plain_inputs(s):
    b, t, kv, dq, dv, rot = s["b"], s["t"], s["kv_heads"], s["dq"], s["dv"], s["rot"]
    pre, pos, k, v = s["pre"].float(), s["pos"].long(), s["k"], s["v"]
    at = pos[:, None] + _plain_closure(s["parents"]).sum(2) - 1
    x = pre[..., :(s["heads"] + kv) * dq].view(b, t, -1, dq)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if s["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack([first, second], -1).flatten(-2) if s["interleaved"] else torch.cat([first, second], -1)
    x = torch.cat([turned, x[..., rot:]], -1)
    if s["norm"]:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    q, new = x[:, :, :s["heads"]].to(k.dtype), x[:, :, s["heads"]:].to(k.dtype)
    row = (pos[:, None] + torch.arange(t, device=k.device))[:, None]
    seq, head = torch.arange(b, device=k.device)[:, None, None], torch.arange(kv, device=k.device)[None, :, None]
    k[seq, head, row] = new.transpose(1, 2)
    v[seq, head, row] = s["pre"][..., (s["heads"] + kv) * dq:].view(b, t, kv, dv).transpose(1, 2)
    return {"q": q, "k": k, "v": v}


def _plain_keep(s):
    i = torch.arange(s["most"], device="cuda")
    pos = s["pos"].long()[:, None]
    to = (pos + i)[:, None]
    of = (pos + torch.where(i < s["count"][:, None], s["path"].long(), i))[:, None]
    seq, head = torch.arange(s["b"], device="cuda")[:, None, None], torch.arange(s["kv_heads"], device="cuda")[None, :, None]
    s["k"][seq, head, to] = s["k"][seq, head, of]
    s["v"][seq, head, to] = s["v"][seq, head, of]
    return {"k": s["k"], "v": s["v"]}


# ------------------------------------------------------------- the operators ---
_PROCESS = {}


def _handles(s):
    """The device handle that a program has, and its handles of the state's buffers."""
    from ug_b200.device import Device, DType
    if "dev" not in _PROCESS:
        _PROCESS["dev"] = Device(0)
    if "slices" not in s:
        code = {torch.bfloat16: DType.BF16, torch.float32: DType.F32, torch.int32: DType.I32}
        s["slices"] = {n: _PROCESS["dev"].wrap(x.data_ptr(), code[x.dtype], x.numel()) for n, x in s.items() if isinstance(x, torch.Tensor)}
    return _PROCESS["dev"], s["slices"]


def run(s):
    kind = s["kind"]
    if not own:
        if kind == "sample":
            return _plain_sample(s)
        if kind == "tree_inputs":
            return _plain_inputs(s)
        return _plain_keep(s) if kind == "keep" else _plain_attention(s)
    dev, h = _handles(s)
    if kind == "sample":
        dev.sample(h["logits"], h["u"], h["tokens"], s["rows"], s["vocab"], temperature=h.get("temperature"), top_k=h.get("top_k"),
                   top_p=h.get("top_p"), min_p=h.get("min_p"), prob=h["prob"])
        return {"tokens": s["tokens"], "prob": s["prob"]}
    b, kv, dq, dv, t_max = s["b"], s["kv_heads"], s["dq"], s["dv"], _t_max(s)
    if kind == "window":
        dev.window_attend(h["q"], h["k"], h["v"], h["pos"], h["out"], b, s["t"], s["heads"], kv, dq, dv, t_max, s["sinks"], s["window"], dq ** -0.5)
        return s["out"]
    if kind == "tree":
        dev.tree_attend(h["q"], h["k"], h["v"], h["pos"], h["parents"], h["out"], b, s["t"], s["heads"], kv, dq, dv, t_max, dq ** -0.5)
        return s["out"]
    if kind == "tree_inputs":
        dev.tree_inputs(h["pre"], h["cos"], h["sin"], h["pos"], h["parents"], h["q"], h["k"], h["v"], b, s["t"], s["heads"], kv, dq, dv, s["rot"],
                        s["interleaved"], s["norm"], 1e-5, t_max)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    dev.cache_keep(h["k"], h["v"], h["pos"], h["path"], h["count"], b, kv, dq, dv, t_max, s["most"])
    return {"k": s["k"], "v": s["v"]}


# ------------------------------------------------------------ what it costs ---
def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 28 * case["rows"], "flops": 4 * n}
    size = 2 if case["dtype"] == "bf16" else 4
    b, kv, dq, dv, heads = case["b"], case["kv_heads"], case["dq"], case["dv"], case["heads"]
    if kind == "keep":
        return {"bytes": 2 * b * (case["most"] + 1) / 2 * kv * (dq + dv) * size + 4 * b * (case["most"] + 2), "flops": 0}
    t = case["t"]
    if kind == "tree_inputs":
        return {"bytes": 2 * b * t * ((heads + kv) * dq + kv * dv) * size + 4 * b * (t + 1) + 4 * b * t * case["rot"], "flops": 6 * b * t * (heads + kv) * dq}
    mean = (case["depth"] + 0.75 * case["depth"] * (b - 1)) / b      # committed positions of a sequence
    if kind == "tree":
        pairs, keys = b * t * (mean + 6), b * (mean + t)
    else:
        last = mean + t
        each = lambda n: min(n, case["window"] + min(case["sinks"], max(0, n - case["window"])))
        pairs = b * t * (each(mean + 1) + each(mean + (t + 1) / 2) + each(last)) / 3
        keys = b * min(last, case["window"] + t - 1 + case["sinks"])
    return {"bytes": (b * t * heads * (dq + dv) + keys * kv * (dq + dv)) * size, "flops": 2 * pairs * heads * (dq + dv)}


# -------------------------------------------------- the same from the definition ---
def _exact_sample(s):
    """Row by row: tokens in the order of their logits (equal ones by index), cut, drawn by index."""
    tokens, probs = [], []
    get = lambda n, r, off: off if s[n] is None else float(s[n][r])
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    import numpy as np
    for r, x in enumerate(logits):
        temperature, k, p, low = (get(n, r, off) for n, off in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        if temperature == 0:
            tokens.append(int(np.argmax(x)))
            probs.append(1.0)
            continue
        order = np.lexsort((np.arange(x.size), -x))
        if k > 0:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / temperature)
        if p < 1:
            enough = np.nonzero(np.cumsum(w) >= p * w.sum())[0]
            end = int(enough[0]) + 1 if enough.size else order.size
            order, w = order[:end], w[:end]
        order, w = order[w >= low], w[w >= low]
        by_index = np.argsort(order)
        order, w = order[by_index], w[by_index]
        c = np.cumsum(w)
        at = min(int(np.searchsorted(c, u[r] * c[-1], side="right")), order.size - 1)
        tokens.append(int(order[at]))
        probs.append(w[at] / c[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}


def _ancestors(parents):
    """For each node the list of itself and its ancestors."""
    lists = []
    for i, p in enumerate(parents):
        lists.append(([] if p < 0 else lists[p]) + [i])
    return lists


def _exact_attention(s):
    b, t, heads, share = s["b"], s["t"], s["heads"], s["heads"] // s["kv_heads"]
    out = torch.empty(b, t, heads, s["dv"], dtype=torch.float64, device="cuda")
    for n in range(b):
        pos = int(s["pos"][n])
        hidden = torch.ones(t, pos + t, dtype=torch.bool, device="cuda")
        if s["kind"] == "tree":
            lists = _ancestors(s["parents"][n].tolist())
            hidden[:, :pos] = False
            rows = [i for i in range(t) for _ in lists[i]]
            hidden[rows, [pos + j for l in lists for j in l]] = False
        else:
            row = torch.arange(pos, pos + t, device="cuda")[:, None]
            back = row - torch.arange(pos + t, device="cuda")          # how far a key lies behind the query
            hidden = (back < 0) | (back >= s["window"]) & (row - back >= s["sinks"])
        for h in range(heads):
            k, v = s["k"][n, h // share, :pos + t].double(), s["v"][n, h // share, :pos + t].double()
            score = torch.einsum("id,jd->ij", s["q"][n, :, h].double(), k) / math.sqrt(s["dq"])
            out[n, :, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v
    return out


def _exact_inputs(s):
    b, t, heads, kv, dq, rot = s["b"], s["t"], s["heads"], s["kv_heads"], s["dq"], s["rot"]
    q, k, v = torch.empty(b, t, heads, dq, dtype=torch.float64, device="cuda"), s["k"].double(), s["v"].double()
    pair = [(2 * i, 2 * i + 1) if s["interleaved"] else (i, i + rot // 2) for i in range(rot // 2)]
    left, right = [p[0] for p in pair], [p[1] for p in pair]
    for n in range(b):
        pos = int(s["pos"][n])
        at = torch.tensor([pos + len(l) - 1 for l in _ancestors(s["parents"][n].tolist())], device="cuda")
        x = s["pre"][n, :, :(heads + kv) * dq].double().view(t, heads + kv, dq).clone()
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        z = torch.complex(x[..., left], x[..., right]) * turn
        x[..., left], x[..., right] = z.real, z.imag
        if s["norm"]:
            x = x * (x.square().sum(2, keepdim=True) / dq + 1e-5).rsqrt()
        q[n] = x[:, :heads]
        k[n, :, pos:pos + t] = x[:, heads:].transpose(0, 1)
        v[n, :, pos:pos + t] = s["pre"][n, :, (heads + kv) * dq:].double().view(t, kv, -1).transpose(0, 1)
    return {"q": q, "k": k, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s) if case["rows"] * case["vocab"] <= 1 << 25 else None
    if case["kind"] == "tree_inputs":
        return _exact_inputs(s)
    if case["kind"] != "keep":
        return _exact_attention(s)
    k, v = s["k"].double(), s["v"].double()
    for n in range(case["b"]):
        pos, rows = int(s["pos"][n]), s["path"][n, :int(s["count"][n])].tolist()
        for i, node in enumerate(rows):                     # node >= i: what a later row needs is still there
            k[n, :, pos + i], v[n, :, pos + i] = s["k"][n, :, pos + node].double(), s["v"][n, :, pos + node].double()
    return {"k": k, "v": v}
