"""Head inputs of drafted nodes and the rows that are kept of them, through the C ABI against numpy in 64 bits."""
import numpy as np
import pytest

from hybrid_cases import Buf, close
from oracle import zidevik_ref as Z
from test_zidevik_ops_gpu import half_split
from ug_b200 import DType, UgError, synth
from ug_b200._lib import lib

pytestmark = pytest.mark.gpu
I32 = lambda dev, x: x if hasattr(x, "_h") else dev.slice_from_values(np.ascontiguousarray(x, np.int32).ravel())


def tree(seed, t):
    """Parents of t nodes: chains, stars and everything between, several roots among them."""
    r = synth.rng(seed)
    return np.array([-1 if i == 0 or r.random() < 0.1 else int(r.integers(max(0, i - 6), i)) for i in range(t)], np.int32)


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return np.array(d)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("interleaved,norm", [(1, 1), (0, 1), (1, 0), (0, 0)])
@pytest.mark.parametrize("heads,kv,dim,vdim,rot,t,pos", [
    (2, 1, 8, 8, 8, 1, [0]), (6, 3, 64, 128, 32, 5, [31, 2, 990]), (4, 4, 72, 24, 36, 33, [0, -1, 100]), (3, 1, 256, 40, 128, 128, [63]), (5, 5, 40, 16, 0, 7, [4, 1017]),
    (8, 2, 128, 128, 128, 24, [500, 1, 1000, -1]), (32, 4, 64, 64, 64, 9, [777])])
def test_inputs_of_nodes(dev, bf16, interleaved, norm, heads, kv, dim, vdim, rot, t, pos):
    B, t_max, eps, base, b = Buf(dev, bf16), 1024, 1e-3, 500.0, len(pos)
    pre, pv = B.act(synth.normal(4, (b, t, (heads + kv) * dim + kv * vdim), 2.0))
    angle = np.arange(t_max)[:, None] * base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
    q, q0 = B.act(synth.normal(7, (b, t, heads, dim)))
    kc, k0 = B.act(synth.normal(5, (b, kv, t_max, dim)))
    vc, v0 = B.act(synth.normal(6, (b, kv, t_max, vdim)))
    parents = np.array([tree(20 + s, t) for s in range(b)])
    if b > 1:
        parents[-1] = np.arange(t) - 1                     # a chain
    dev.tree_inputs(pre, B.f32(np.cos(angle)), B.f32(np.sin(angle)), I32(dev, pos), I32(dev, parents), q, kc, vc, b, t, heads, kv, dim, vdim, rot,
                    interleaved, norm, eps, t_max)
    dev.synchronize()
    turn = Z.rotate if interleaved else half_split
    for s in range(b):
        if pos[s] < 0:
            continue                                       # left as it was
        x = pv[s, :, :(heads + kv) * dim].reshape(t, heads + kv, dim)
        x = turn(x, pos[s] + depths(parents[s]), base, rot) if rot else x
        x = Z.rms(x, eps) if norm else x
        q0[s] = x[:, :heads]
        k0[s, :, pos[s]:pos[s] + t] = x[:, heads:].transpose(1, 0, 2)
        v0[s, :, pos[s]:pos[s] + t] = pv[s, :, (heads + kv) * dim:].reshape(t, kv, vdim).transpose(1, 0, 2)
    assert close(B.read(q, q0.shape), q0, B.tol) and close(B.read(kc, k0.shape), k0, B.tol) and np.array_equal(B.read(vc, v0.shape), v0)


@pytest.mark.parametrize("bf16", [False, True])
def test_a_chain_is_a_block(dev, bf16):
    """Nodes that follow one another get what the positions of a block get, from buffers of any alignment too."""
    B, b, t, heads, kv, dim, t_max = Buf(dev, bf16), 1, 12, 6, 2, 64, 64
    size = 2 if bf16 else 4
    pre, _ = B.act(synth.normal(4, (1 + b * t * (heads + 2 * kv) * dim,)))
    angle = np.arange(t_max)[:, None] * 100.0 ** (-np.arange(dim // 2) / (dim // 2))
    cos, sin, pos, got = B.f32(np.cos(angle)), B.f32(np.sin(angle)), I32(dev, [17]), []
    for call in ("block", "nodes", "unaligned"):
        bufs = [B.act(np.zeros(1 + n))[0] for n in (b * t * heads * dim, b * kv * t_max * dim, b * kv * t_max * dim)]
        odd = [dev.wrap(s.device_ptr + size, s.dtype, len(s) - 1) for s in bufs + [pre]]
        src = dev.wrap(pre.device_ptr + size, pre.dtype, len(pre) - 1)
        if call == "block":
            even, _ = B.act(B.read(src, (len(src),)))
            dev.head_inputs(even, cos, sin, pos, *bufs, b, t, heads, kv, dim, dim, dim, False, True, 1e-5, t_max)
        else:
            parents = I32(dev, np.arange(t) - 1)
            q, k, v = odd[:3] if call == "unaligned" else bufs
            from_ = odd[3] if call == "unaligned" else even
            dev.tree_inputs(from_, cos, sin, pos, parents, q, k, v, b, t, heads, kv, dim, dim, dim, False, True, 1e-5, t_max)
        dev.synchronize()
        got.append([x.to_vec()[1:] if call == "unaligned" else x.to_vec()[:-1] for x in bufs])
    for want, nodes, unaligned in zip(*got):
        f = lambda x: (synth.bf16_bits_to_f32(x) if bf16 else x).astype(np.float64)
        assert close(f(nodes), f(want), B.tol) and np.array_equal(nodes, unaligned)


def inputs_call(dev, B, pos, parents, b=2, t=3, t_max=32, heads=2, kv=1, dim=8, vdim=8, rot=8, **swap):
    n = dict(pre=B.act(np.ones((b, t, (heads + kv) * dim + kv * vdim)))[0], cos=B.f32(np.ones((t_max, max(1, rot // 2)))), sin=B.f32(np.zeros((t_max, max(1, rot // 2)))),
             pos=I32(dev, pos), parents=I32(dev, parents), q=B.act(np.zeros((b, t, heads, dim)))[0], k=B.act(np.zeros((b, kv, t_max, dim)))[0],
             v=B.act(np.zeros((b, kv, t_max, vdim)))[0])
    n.update(swap)
    dev.tree_inputs(*n.values(), b, t, heads, kv, dim, vdim, rot, True, False, 1e-5, t_max)
    return n


@pytest.mark.parametrize("pos,parents", [([30, 0], [-1, 0, 1]), ([-2, 0], [-1, 0, 1]), ([2 ** 31 - 2, 0], [-1, 0, 1]), ([0, 0], [0, 0, 1]), ([0, 0], [-1, 2, 1]), ([0, 0], [-1, -2, 0]),
                                         ([0, 0], [-1, 0, 2 ** 31 - 1])])
def test_bad_trees_and_positions_of_inputs(dev, pos, parents):
    """The bad sequence is left as it was, the other one is done."""
    n = inputs_call(dev, Buf(dev, False), pos, [parents, [-1, 0, 0]])
    with pytest.raises(UgError) as e:
        dev.synchronize()
    assert e.value.code == 1
    assert not n["q"].to_vec()[:48].any() and not n["k"].to_vec()[:256].any() and not n["v"].to_vec()[:256].any()
    assert n["q"].to_vec()[48:].all() and n["k"].to_vec()[256:280].all() and n["v"].to_vec()[256:280].all()


def test_refusals_of_inputs(dev):
    F, H = Buf(dev, False), Buf(dev, True)
    ok = dict(pos=[0, 0], parents=[[-1, 0, 1]] * 2)
    cases = [(2, dict(q=H.act(np.zeros(48 * 2))[0])), (2, dict(k=H.act(np.zeros(512))[0])), (2, dict(parents=F.f32(np.zeros(6)))), (3, dict(pre=F.f32(np.zeros(10)))),
             (3, dict(pos=I32(dev, [0]))), (3, dict(dim=12)), (3, dict(rot=16)), (3, dict(rot=7)), (3, dict(kv=0)), (3, dict(t_max=2)), (3, dict(dim=264)), (3, dict(cos=F.f32(np.zeros(3))))]
    for code, swap in cases:
        with pytest.raises(UgError) as e:
            inputs_call(dev, F, **{**ok, **swap})
        assert e.value.code == code, swap
    big = F.f32(np.zeros(129 * 24))
    with pytest.raises(UgError) as e:
        inputs_call(dev, F, [0], np.arange(129) - 1, b=1, t=129, t_max=256)
    assert e.value.code == 6
    for swap in (dict(pre=big, q=big), dict(k=big, v=big)):
        with pytest.raises(UgError) as e:
            inputs_call(dev, F, **ok, **swap)
        assert e.value.code == 1
    inputs_call(dev, F, [0], [], b=1, t=0)
    assert lib.ugb_tree_inputs(None, *[None] * 8, 1, 1, 1, 1, 8, 8, 8, 0, 0, 1e-5, 8) == 1


def kept(k, pos, paths):
    """What the definition leaves: rows of the accepted nodes behind the committed ones."""
    out = k.copy()
    for s, (p, path) in enumerate(zip(pos, paths)):
        for i, node in enumerate(path if p >= 0 else []):
            out[s, :, p + i] = k[s, :, p + node]
    return out


def keep_call(dev, B, k, v, pos, paths, most, counts=None, shift=0):
    b, kv, t_max, dq = k.shape
    size = 2 if B.bf16 else 4
    pad = lambda x: np.r_[np.zeros(shift), x.ravel()]
    (ks, _), (vs, _) = B.act(pad(k)), B.act(pad(v))
    path = np.full((b, most), -99, np.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)] = p[:most]
    part = lambda s: dev.wrap(s.device_ptr + shift * size, s.dtype, len(s) - shift)
    dev.cache_keep(part(ks), part(vs), I32(dev, pos), I32(dev, path), I32(dev, [len(p) for p in paths] if counts is None else counts), b, kv, dq, v.shape[3], t_max, most)
    return lambda: [B.read(x, (-1,))[shift:].reshape(y.shape) for x, y in ((ks, k), (vs, v))]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kv,dq,dv", [(1, 8, 8), (3, 64, 128), (8, 128, 128), (2, 72, 40), (1, 1024, 24)])
@pytest.mark.parametrize("shift", [0, 1])
def test_kept_rows(dev, bf16, kv, dq, dv, shift):
    """Paths with and without overlap of what is read and written, of no node and of all."""
    B, t_max, most = Buf(dev, bf16), 160, 20
    pos = [0, 7, -1, 140, 30, 99, 32]
    paths = [[0, 2, 5, 6, 11], [], [3, 4], list(range(20)), [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [60], list(range(3, 43, 2))]
    _, k = B.act(synth.normal(1, (len(pos), kv, t_max, dq)))
    _, v = B.act(synth.normal(2, (len(pos), kv, t_max, dv)))
    got = keep_call(dev, B, k, v, pos, paths, most, shift=shift)
    dev.synchronize()
    for x, want in zip(got(), (kept(k, pos, paths), kept(v, pos, paths))):
        assert np.array_equal(x, want)


@pytest.mark.parametrize("pos,path,count", [(-2, [0, 1], None), (0, [1, 1], None), (0, [2, 1], None), (0, [-1, 3], None), (3, [1, 0], None), (0, [0, 32], None), (31, [0, 1], None), (0, [0, 1], 5), (0, [0, 1], -1), (32, [0], None),
                                            (2 ** 31 - 1, [0], None)])
def test_bad_paths(dev, pos, path, count):
    """The bad sequence is left as it was, the other one is done."""
    B = Buf(dev, True)
    k, v = (B.act(synth.normal(s, (2, 2, 32, 16)))[1] for s in (1, 2))
    got = keep_call(dev, B, k, v, [pos, 4], [path, [1, 3]], 4, [len(path) if count is None else count, 2])
    with pytest.raises(UgError) as e:
        dev.synchronize()
    assert e.value.code == 1
    for x, y in zip(got(), (k, v)):
        assert np.array_equal(x, kept(y, [-1, 4], [[], [1, 3]]))


def test_refusals_of_keep(dev):
    z, h, i = dev.zeros(512), Buf(dev, True).out(512), I32(dev, [0] * 8)
    w = dev.zeros(512)
    for code, args in ((2, (z, h, i, i, i, 1, 1, 8, 8, 32, 2)), (2, (i, i, i, i, i, 1, 1, 8, 8, 1, 1)), (2, (z, w, i, z, i, 1, 1, 8, 8, 32, 2)), (3, (z, w, i, i, i, 1, 1, 8, 8, 128, 2)), (3, (z, w, i, i, i, 9, 1, 8, 8, 1, 1)),
                       (3, (z, w, i, i, i, 1, 1, 12, 8, 32, 2)), (3, (z, w, i, i, i, 1, 0, 8, 8, 32, 2)), (6, (z, w, i, i, i, 0, 1, 8, 8, 32, 129)), (1, (z, z, i, i, i, 1, 1, 8, 8, 32, 2))):
        with pytest.raises(UgError) as e:
            dev.cache_keep(*args)
        assert e.value.code == code, args
    dev.cache_keep(z, w, i, i, i, 0, 1, 8, 8, 32, 2)
    dev.cache_keep(z, w, i, i, i, 1, 1, 8, 8, 32, 0)
    assert lib.ugb_cache_keep(None, *[None] * 5, 1, 1, 8, 8, 8, 1) == 1
