"""GPU parity of the 8-bit rows: quantiser and transform (run with -m gpu).

Every step of both is defined to the bit (an exact integer, then single fp32
roundings in a fixed order), so results are compared bit for bit with the numpy
form, whose integer sums and rounding decisions are made in 64 bits.
"""
import ctypes

import numpy as np
import pytest
import torch

from gnn_cuda_b200 import _native as N
from gnn_cuda_b200.GNN_cuda_common import int8_ops as I
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _status():
    status = ctypes.c_int(-1)
    N.check(N.lib().gnn_device_status(1, ctypes.byref(status)))
    return status.value


def _features(rows, cols, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, cols)).astype(np.float32) * np.exp(r.standard_normal((rows, 1))).astype(np.float32)
    if rows > 3:
        x[1] = 0
    return x


def _rows8(q):
    t = I.empty_rows(q.shape[0], q.shape[1], DEV)
    t.copy_(torch.from_numpy(q))
    return t


def _quantize(x):
    q, s = I.empty_rows(x.shape[0], x.shape[1], DEV), torch.empty(x.shape[0], device=DEV)
    I.quantize_rows_(torch.from_numpy(x).to(DEV), q, s)
    return q, s


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 3), (33, 128), (1000, 127), (257, 200), (70, 501), (64, 1024),
                                       (9, 1023), (7, 1025), (5, 1300), (6, 4096), (3, 5000), (4, 9001), (40000, 64)])
def test_quantize_rows(rows, cols):
    x = _features(rows, cols, rows + cols)
    q, s = _quantize(x)
    eq, es = O.quantize(x)
    assert O.same_bits(s.cpu().numpy(), es)
    assert np.array_equal(q.cpu().numpy(), eq)


def test_quantize_borders_and_odd_rows():
    """Ties, quotients one unit beside a tie, tiny, subnormal, huge, infinite and NaN rows."""
    rows = []
    for s in (1.0, 2.0 ** -140, 3.0e-39, 1.1754944e-38, 0.3333333, 1e-30, 2.0 ** 120):
        s = np.float32(s)
        base = (np.arange(-127, 128, dtype=np.float64) + 0.5) * np.float64(s)
        r = base.astype(np.float32)
        near = np.concatenate([r, np.nextafter(r, np.float32(np.inf)), np.nextafter(r, np.float32(-np.inf))])
        near = near[np.abs(near) <= np.float64(s) * 127]
        rows.append(np.concatenate([near, [np.float32(s) * np.float32(127)]]).astype(np.float32))
    width = max(len(r) for r in rows)
    x = np.stack([np.pad(r, (0, width - len(r))) for r in rows])
    extra = np.zeros((7, width), np.float32)
    extra[0, 5] = np.nan
    extra[1, :] = np.inf
    extra[2, 3] = -np.inf
    extra[3, :] = np.float32(1e-45)          # scale underflows to 0
    extra[4, :] = np.float32(180 * 1e-45)    # scale of one subnormal unit: past 127 steps, clamped
    extra[5, 0] = np.float32(3.4e38)
    extra[6, :3] = [np.float32(1.0), np.nan, np.inf]
    x = np.concatenate([x, extra])
    q, s = _quantize(x)
    eq, es = O.quantize(x)
    assert O.same_bits(s.cpu().numpy(), es)
    assert np.array_equal(q.cpu().numpy(), eq)


@pytest.mark.parametrize("k,n", [(1, 1), (128, 128), (501, 47), (33, 100), (300, 1)])
def test_quantize_weight(k, n):
    w = _features(k, n, 3)
    q, s = I.empty_rows(n, k, DEV), torch.empty(n, device=DEV)
    I.quantize_weight_(torch.from_numpy(w).to(DEV), q, s)
    eq, es = O.quantize(np.ascontiguousarray(w.T))
    assert O.same_bits(s.cpu().numpy(), es) and np.array_equal(q.cpu().numpy(), eq)


SHAPES = [(1, 1, 1), (1, 512, 512), (3, 16, 7), (130, 128, 128), (1000, 501, 47), (257, 130, 33), (515, 64, 256),
          (128 * 148 + 5, 128, 128), (300, 1000, 257), (64, 4096, 1000), (2, 1433, 7), (4, 130, 300), (8, 64, 64), (8, 5120, 40), (9, 40, 24), (16, 300, 40), (31, 1000, 65), (32, 1280, 300), (32, 1281, 20), (33, 64, 64), (129, 200, 640), (17, 2048, 96)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("relu", [False, True])
def test_linear_int8(m, k, n, relu):
    x, w = _features(m, k, m + k), _features(n, k, n)
    b = np.random.default_rng(9).standard_normal(n).astype(np.float32)
    q, sx = O.quantize(x)
    wq, sw = O.quantize(w)
    out = torch.full((m, n), float("nan"), device=DEV)
    args = (_rows8(wq), torch.from_numpy(sw).to(DEV))
    bias = torch.from_numpy(b).to(DEV)
    I.linear_int8_forward_(_rows8(q), torch.from_numpy(sx).to(DEV), *args, bias, out, relu)
    want = O.linear(q, sx, wq, sw, b, relu)
    assert O.same_bits(out.cpu().numpy(), want)
    # fp32 rows quantised on the way, without a bias
    out.fill_(float("nan"))
    I.linear_int8_forward_(torch.from_numpy(x).to(DEV), None, *args, None, out, relu)
    assert O.same_bits(out.cpu().numpy(), O.linear(q, sx, wq, sw, None, relu))
    # 8-bit output rows; bytes behind a row stay
    o8, os_ = torch.full((m, (n + 31) // 16 * 16), 77, dtype=torch.int8, device=DEV), torch.empty(m, device=DEV)
    I.linear_int8_forward_(_rows8(q), torch.from_numpy(sx).to(DEV), *args, bias, o8[:, :n], relu, out_scale=os_)
    eq, es = O.quantize(want)
    assert O.same_bits(os_.cpu().numpy(), es) and np.array_equal(o8[:, :n].cpu().numpy(), eq)
    assert bool((o8[:, n:] == 77).all())
    assert _status() == 0


@pytest.mark.parametrize("k", [128, 77])
def test_linear_int8_strides_and_extremes(k):
    """Unaligned strides and bases, -128, products at the edge of 32-bit sums' fp32 rounding."""
    r = np.random.default_rng(k)
    m, n = 141, 37
    q = r.integers(-128, 128, (m, k)).astype(np.int8)
    w = r.integers(-128, 128, (n, k)).astype(np.int8)
    q[0], w[0] = -128, -128
    q[1], w[1] = 127, -128
    sx, sw = r.random(m).astype(np.float32), r.random(n).astype(np.float32)
    want = O.linear(q, sx, w, sw, None, False)
    hold = torch.zeros(m, k + 5, dtype=torch.int8, device=DEV)
    hold[:, 3:3 + k] = torch.from_numpy(q).to(DEV)
    whold = torch.zeros(n, k + 1, dtype=torch.int8, device=DEV)
    whold[:, 1:] = torch.from_numpy(w).to(DEV)
    base = torch.zeros(m * n + 1, device=DEV)
    for x8 in (hold[:, 3:3 + k], torch.from_numpy(q).to(DEV)):
        out = base[1:].view(m, n)  # rows that start on 4-byte boundaries only
        out.zero_()
        I.linear_int8_forward_(x8, torch.from_numpy(sx).to(DEV), whold[:, 1:], torch.from_numpy(sw).to(DEV), None, out)
        assert O.same_bits(out.cpu().numpy(), want)
        o8, os_ = torch.zeros(m, n, dtype=torch.int8, device=DEV), torch.empty(m, device=DEV)
        I.linear_int8_forward_(x8, torch.from_numpy(sx).to(DEV), whold[:, 1:], torch.from_numpy(sw).to(DEV), None, o8,
                               out_scale=os_)
        eq, es = O.quantize(want)
        assert O.same_bits(os_.cpu().numpy(), es) and np.array_equal(o8.cpu().numpy(), eq)


def test_linear_int8_long_sums():
    """Sums past 2^24: exact in 32-bit integers, then one rounding."""
    k = 40000
    q = np.full((5, k), 127, np.int8)
    q[1:, ::3] = -127
    w = np.full((9, k), 127, np.int8)
    w[3:, 1::7] = 5
    one = lambda n: np.full(n, 0.5, np.float32)  # noqa: E731
    out = torch.empty(5, 9, device=DEV)
    I.linear_int8_forward_(_rows8(q), torch.from_numpy(one(5)).to(DEV), _rows8(w), torch.from_numpy(one(9)).to(DEV),
                           None, out)
    assert O.same_bits(out.cpu().numpy(), O.linear(q, one(5), w, one(9), None, False))


def test_nan_rows_poison_their_outputs_only():
    x, w = _features(300, 64, 1), _features(40, 64, 2)
    x[7, 3], x[200, 0] = np.nan, np.inf
    wq, sw = O.quantize(w)
    out = torch.empty(300, 40, device=DEV)
    I.linear_int8_forward_(torch.from_numpy(x).to(DEV), None, _rows8(wq), torch.from_numpy(sw).to(DEV), None, out, True)
    bad = torch.isnan(out).all(1).cpu()
    assert bad[7] and bad[200] and int(torch.isnan(out).any(1).sum()) == 2
    o8, os_ = I.empty_rows(300, 40, DEV), torch.empty(300, device=DEV)
    I.linear_int8_forward_(torch.from_numpy(x).to(DEV), None, _rows8(wq), torch.from_numpy(sw).to(DEV), None, o8, True,
                           out_scale=os_)
    assert torch.isnan(os_).nonzero().flatten().tolist() == [7, 200] and int(o8[7].abs().max()) == 0


def test_empty_and_streams_and_graphs():
    wq, sw = O.quantize(_features(96, 200, 5))
    args = (_rows8(wq), torch.from_numpy(sw).to(DEV), None)
    I.linear_int8_forward_(I.empty_rows(0, 200, DEV), torch.empty(0, device=DEV), *args, torch.empty(0, 96, device=DEV))
    I.quantize_rows_(torch.empty(0, 8, device=DEV), I.empty_rows(0, 8, DEV), torch.empty(0, device=DEV))
    xs = [torch.from_numpy(_features(3000, 200, 30 + i)).to(DEV) for i in range(2)]
    wants = [torch.empty(3000, 96, device=DEV) for _ in xs]
    for x, o in zip(xs, wants):
        I.linear_int8_forward_(x, None, *args, o)
    # two captured graphs replayed on two streams at once, each with its own scratch
    outs, graphs = [torch.zeros(3000, 96, device=DEV) for _ in xs], []
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            I.linear_int8_forward_(x, None, *args, o)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, wants):
        assert torch.equal(o, w)
    assert _status() == 0
