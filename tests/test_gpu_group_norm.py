"""GPU parity of the group normalisation (run with -m gpu), against numpy in 64 bits.

Bound. With u = 2^-24: the mean carries a few roundings of values up to max|x| =: A
over the group, so each deviation is off by at most 24 u A (a batch mean, its update
per batch and the joins over lanes and pieces: fewer than 24 roundings follow one
another for the sizes here), and the standard deviation by the same amount and 16 u of
itself. With z = (x - mean) / sd that makes |dz| <= 24 u A / sd * (1 + |z|) + 24 u |z|,
then y = z w + b adds 4 u (|z w| + |b|), and the activation is 1.13-Lipschitz and adds
8 u |y| + 2^-22 of its own (the reduced-precision exponential is good to 2 + |y| units).
"""
import math

import numpy as np
import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import norm_ops as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
EPS = 1e-5


def _act(y, act):
    if act == "relu":
        return np.maximum(y, 0)
    if act == "silu":
        return y / (1 + np.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))
    return y


def _want(x, groups, w, b, ptr, act):
    """(values, bounds) in 64 bits; rows of no graph are NaN."""
    n, c = x.shape
    x = x.astype(np.float64)
    want, bound = np.full((n, c), np.nan), np.zeros((n, c))
    spans = [(i, i + 1) for i in range(n)] if ptr is None else list(zip(ptr[:-1], ptr[1:]))
    cg = c // groups
    w = np.ones(c) if w is None else w.astype(np.float64)
    b = np.zeros(c) if b is None else b.astype(np.float64)
    for s, e in spans:
        if e <= s:
            continue
        v = x[s:e].reshape(e - s, groups, cg)
        d = v - v.mean(axis=(0, 2), keepdims=True)
        sd = np.sqrt((d * d).mean(axis=(0, 2), keepdims=True) + EPS)
        z = d / sd
        a = np.abs(v).max(axis=(0, 2), keepdims=True)
        dz = 24 * U * a / sd * (1 + np.abs(z)) + 24 * U * np.abs(z)
        z, dz = z.reshape(e - s, c), dz.reshape(e - s, c)
        y = z * w + b
        want[s:e] = _act(y, act)
        bound[s:e] = 1.13 * (dz * np.abs(w) + 4 * U * (np.abs(z * w) + np.abs(b))) + (8 + np.abs(y)) * U * np.abs(y) + 4 * U
    return want, bound


def _run(n, c, groups, ptr, act="none", seed=0, affine=True, index=torch.int32, shift=3.0, inplace=False, x=None):
    r = np.random.default_rng(seed)
    if x is None:
        x = (r.standard_normal((n, c)) * (0.3 + r.random(c)) + shift * r.standard_normal(c)).astype(np.float32)
    w = (1 + 0.3 * r.standard_normal(c)).astype(np.float32) if affine else None
    b = (0.3 * r.standard_normal(c)).astype(np.float32) if affine else None
    dx = torch.from_numpy(x).to(DEV)
    keep = torch.from_numpy(r.standard_normal((n, c)).astype(np.float32)).to(DEV)
    out = dx if inplace else keep.clone()
    dptr = None if ptr is None else torch.tensor(np.asarray(ptr), device=DEV).to(index)
    dw, db = (None, None) if not affine else (torch.from_numpy(w).to(DEV), torch.from_numpy(b).to(DEV))
    M.group_norm_forward_(dx, groups, dw, db, out, graph_ptr=dptr, eps=EPS, activation=act)
    want, bound = _want(x, groups, w, b, ptr, act)
    got = out.cpu().numpy().astype(np.float64)
    none = np.isnan(want)
    before = x if inplace else keep.cpu().numpy()
    assert np.array_equal(got[none], before.astype(np.float64)[none])
    err = np.abs(got - want)
    assert np.all(err[~none] <= bound[~none]), float(np.max(err[~none] / bound[~none]))
    if not inplace:
        again = keep.clone()
        M.group_norm_forward_(dx, groups, dw, db, again, graph_ptr=dptr, eps=EPS, activation=act)
        assert torch.equal(again, out)


CHANNELS = [(1, 1), (5, 1), (27, 3), (32, 32), (32, 4), (100, 10), (128, 128), (64, 8), (60, 5), (48, 3), (12, 3), (12, 12), (21, 7), (64, 1), (64, 64), (96, 8), (100, 4), (128, 8), (128, 32),
            (130, 2), (192, 3), (256, 16), (300, 100), (512, 1), (999, 27), (1024, 1), (1023, 1), (1280, 10), (2050, 1025)]


@pytest.mark.parametrize("c,groups", CHANNELS)
def test_nodes(c, groups):
    _run(77, c, groups, None, seed=c)


@pytest.mark.parametrize("c,groups", CHANNELS)
def test_graphs(c, groups):
    n = 1000
    _run(n, c, groups, [0, 5, 5, 6, 70, 134, 135, 500, 980], seed=c + 1)


@pytest.mark.parametrize("n,c,groups", [(1, 27, 3), (303, 27, 3), (20000, 9, 9), (70001, 14, 2), (5000, 128, 16)])
def test_many_narrow_nodes(n, c, groups):
    _run(n, c, groups, None, "relu", seed=n)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("graphs", [False, True])
def test_activations(act, graphs):
    _run(400, 48, 6, [0, 3, 200, 400] if graphs else None, act, seed=5)
    _run(9, 7, 1, [2, 9] if graphs else None, act, seed=6, affine=False)


@pytest.mark.parametrize("n,ptr", [(1, [0, 1]), (1, [0, 0]), (64, [0, 64]), (65, [0, 65]), (65, [0, 64, 65]),
                                   (128, [0, 64, 128]), (129, [0, 1, 129]), (200, [0, 65, 130, 195]),
                                   (700, [10, 10, 10, 80, 80, 650]), (640, [0, 320, 640]), (5000, [0, 5000]),
                                   (300, [299, 300]), (300, [300, 300]), (200, [64, 129, 193])])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_graph_bounds(n, ptr, index):
    _run(n, 32, 4, ptr, seed=n, index=index)


def test_many_empty_graphs():
    ptr = np.concatenate([np.zeros(50000), np.full(50000, 3), np.full(70000, 500), [777]]).astype(np.int64)
    _run(800, 16, 2, ptr, seed=1)


def test_many_random_graphs():
    r = np.random.default_rng(2)
    ptr = np.sort(r.integers(0, 20001, 900))
    _run(20000, 40, 5, ptr, "silu", seed=3)


def _check_wide(n, c, groups, ptr, seed):
    """The same bounds on the GPU, for row counts whose windows hold several long graphs."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, c, device=DEV, generator=g) + 2
    out = torch.full_like(x, 7.0)
    M.group_norm_forward_(x, groups, None, None, out, graph_ptr=ptr)
    ptr = ptr.long()
    seg = torch.searchsorted(ptr, torch.arange(n, device=DEV), right=True) - 1
    inside = (seg >= 0) & (seg < len(ptr) - 1)
    seg = seg.clamp(0, len(ptr) - 2)
    v = x.double().view(n, groups, -1)
    count = (ptr.diff().clamp(min=1) * (c // groups)).double()[:, None]
    zero = torch.zeros(len(ptr) - 1, groups, dtype=torch.float64, device=DEV)
    mean = zero.index_add(0, seg[inside], v.sum(2)[inside]) / count
    d = v - mean[seg][:, :, None]
    sd = (zero.index_add(0, seg[inside], d.square().sum(2)[inside]) / count + EPS).sqrt()[seg][:, :, None]
    z = d / sd
    biggest = float(x.abs().max())
    bound = 24 * U * biggest / sd * (1 + z.abs()) + 28 * U * z.abs()
    err = (out.double().view(n, groups, -1) - z).abs()
    assert bool((err <= bound)[inside].all())
    assert bool((out[~inside] == 7.0).all())


@pytest.mark.parametrize("rows,graphs", [(200_003, 8192), (300_000, 3000), (400_000, 1500), (160_000, 100_000),
                                         (1_000_000, 40)])
def test_batches_of_many_rows(rows, graphs):
    g = torch.Generator(device=DEV).manual_seed(rows)
    end = rows - rows // 50
    cuts = torch.randint(0, end + 1, (graphs - 1,), device=DEV, generator=g).sort().values
    ends = torch.tensor([0, end], device=DEV)
    _check_wide(rows, 36, 4, torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32), rows)


@pytest.mark.parametrize("length", [64, 65, 100, 128, 256, 257])
def test_equal_graphs(length):
    n = 1600 * length
    _check_wide(n, 8, 2, torch.arange(0, n + 1, length, device=DEV), length)


@pytest.mark.parametrize("ptr", [None, [0, 300]])
def test_in_place(ptr):
    _run(300, 64, 4, ptr, "relu", inplace=True)


def test_large_mean_small_spread():
    """Values whose mean is 3,000 times their spread: nothing is subtracted from sums of squares."""
    _run(3000, 32, 2, [0, 50, 3000], seed=4, shift=3000.0)


def test_constant_and_special_values():
    x = np.full((200, 8), 2.5, np.float32)
    x[150:] = np.random.default_rng(0).standard_normal((50, 8))
    _run(200, 8, 2, [0, 150, 200], x=x.copy())
    _run(200, 8, 2, None, x=x.copy())
    dx = torch.from_numpy(x).to(DEV)
    dx[160, 1], dx[10, 6] = float("nan"), float("inf")
    out = torch.empty_like(dx)
    M.group_norm_forward_(dx, 2, None, None, out, graph_ptr=torch.tensor([0, 150, 200], dtype=torch.int32, device=DEV))
    bad = torch.isnan(out)
    assert bool(bad[:150, 4:].all()) and bool(bad[150:, :4].all())
    assert not bool(bad[:150, :4].any()) and not bool(bad[150:, 4:].any())


def test_unaligned_base():
    base = torch.randn(50 * 16 + 1, device=DEV)
    x = base[1:].view(50, 16)
    a, b = torch.empty(50, 16, device=DEV), torch.empty(50, 16, device=DEV)
    M.group_norm_forward_(x, 4, None, None, a)
    M.group_norm_forward_(x.clone(), 4, None, None, b)
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_whole_graph_of_many_rows():
    n, c, groups = 300_000, 64, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(n, c, device=DEV, generator=g) + 10
    out = torch.empty_like(x)
    M.group_norm_forward_(x, groups, None, None, out, graph_ptr=torch.tensor([0, n], device=DEV), activation="none")
    v = x.double().view(n, groups, -1)
    d = v - v.mean((0, 2), keepdim=True)
    sd = (d.square().mean((0, 2), keepdim=True) + EPS).sqrt()
    # one shift of the mean by 24 u * 16 (the largest value) over a spread of 1, as derived above
    bound = 24 * U * 16 * (1 + (d / sd).abs()) + 28 * U * (d / sd).abs()
    assert bool(((out.double().view(n, groups, -1) - d / sd).abs() <= bound).all())


def test_graph_replay_on_two_streams():
    n = 5000
    ptr = torch.tensor([0, 100, 4000, 5000], dtype=torch.int32, device=DEV)
    xs = [torch.randn(n, 64, device=DEV) for _ in range(2)]
    wants = [torch.empty_like(x) for x in xs]
    for x, o in zip(xs, wants):
        M.group_norm_forward_(x, 8, None, None, o, graph_ptr=ptr, activation="relu")
    outs, graphs = [torch.zeros_like(x) for x in xs], []
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            M.group_norm_forward_(x, 8, None, None, o, graph_ptr=ptr, activation="relu")
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))
