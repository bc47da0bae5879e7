"""GPU parity of the aggregation over 8-bit rows (run with -m gpu).

Bound, per element, against the 64-bit sum: a row of d entries is summed in fp32 in
some order, so the error is at most (d + 4) * 2^-24 * sum_e |w_e s_c q_c| for the
additions and the weight's roundings (first order; the 1.01 covers the rest).
"""
import numpy as np
import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import int8_ops as I
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _graph(n, degrees, seed):
    r = np.random.default_rng(seed)
    rp = np.concatenate([[0], np.cumsum(degrees)])
    col = r.integers(0, n, rp[-1]).astype(np.int32)
    return rp, col


def _degrees(kind, n, seed):
    r = np.random.default_rng(seed)
    if kind == "short":
        return r.integers(0, 9, n)
    if kind == "empty":
        return np.zeros(n, np.int64)
    if kind == "hub":  # one hub across many shares, long runs of empty rows around it
        d = np.zeros(n, np.int64)
        d[n // 2] = 70001
        d[-1] = 33
        return d
    if kind == "skewed":
        return np.minimum((r.pareto(1.1, n) * 4).astype(np.int64), 20000)
    return np.full(n, 64)  # every share boundary falls on or beside a row end


def _check(rp, col, f, agg, seed, index=np.int32, x8=None):
    n = len(rp) - 1
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, f)).astype(np.float32) * np.exp(r.standard_normal((n, 1))).astype(np.float32)
    q, s = O.quantize(x)
    dis = r.random(n).astype(np.float32) + np.float32(0.1)
    ew = r.standard_normal(len(col)).astype(np.float32)
    deg = np.diff(rp)
    row = np.repeat(np.arange(n), deg)
    w = s[col].astype(np.float64)
    if agg == "gcn":
        w = w * dis[row] * dis[col]
    elif agg == "weighted":
        w = w * ew
    elif agg == "mean":
        w = w / deg[row]
    import scipy.sparse as sp
    a = sp.csr_matrix((w, col, rp), shape=(n, n), copy=True)  # scipy merges duplicates in place
    want = a @ q.astype(np.float64)
    size = abs(a) @ np.abs(q.astype(np.float64))
    held = I.empty_rows(n, f, DEV) if x8 is None else x8
    held.copy_(torch.from_numpy(q))
    out = torch.full((n, f), float("nan"), device=DEV)
    kw = {"deg_inv_sqrt": torch.from_numpy(dis).to(DEV) if agg == "gcn" else None,
          "edge_weight": torch.from_numpy(ew).to(DEV) if agg == "weighted" else None}
    args = (torch.from_numpy(rp.astype(index)).to(DEV), torch.from_numpy(col).to(DEV), held,
            torch.from_numpy(s).to(DEV))
    I.spmm_int8_forward_(*args, out, aggregation=agg, **kw)
    got = out.cpu().numpy().astype(np.float64)
    bound = 1.01 * (deg[:, None] + 4) * 2.0 ** -24 * size
    assert np.all(np.abs(got - want) <= bound)
    again = torch.empty_like(out)
    I.spmm_int8_forward_(*args, again, aggregation=agg, **kw)
    assert torch.equal(again, out)


@pytest.mark.parametrize("agg", ["sum", "mean", "gcn", "weighted"])
@pytest.mark.parametrize("kind", ["short", "empty", "hub", "skewed", "even"])
def test_aggregations(agg, kind):
    n = 3001
    _check(*_graph(n, _degrees(kind, n, 3), 4), 100, agg, 5)


@pytest.mark.parametrize("f", [1, 7, 16, 17, 32, 33, 64, 96, 128, 129, 201, 256, 300, 512, 513, 1100])
def test_widths(f):
    n = 700
    _check(*_graph(n, _degrees("skewed", n, f), f), f, "gcn", f)


@pytest.mark.parametrize("n,deg", [(1, 0), (1, 1), (1, 1000), (2, 3), (64, 1), (5, 0)])
def test_small(n, deg):
    _check(*_graph(n, np.full(n, deg), 1), 40, "mean", 2, index=np.int64)


@pytest.mark.parametrize("f", [40, 48])
def test_unaligned_rows(f):
    n = 333
    rp, col = _graph(n, _degrees("short", n, 1), 2)
    hold = torch.empty(n * (f + 3) + 1, dtype=torch.int8, device=DEV)
    _check(rp, col, f, "sum", 7, x8=hold[1:].view(n, f + 3)[:, :f])
    # a padded stride without storage behind the last row's columns
    flat = torch.empty((n - 1) * 64 + f, dtype=torch.int8, device=DEV)
    _check(rp, col, f, "sum", 8, x8=flat.as_strided((n, f), (64, 1)))


def test_large_offsets():
    """Row offsets past 2^31 bytes: a 5,000,000 x 448 matrix, entries in its last rows."""
    n, f = 5_000_000, 448
    x = torch.zeros(n, f, dtype=torch.int8, device=DEV)
    x[-3:] = torch.randint(-127, 128, (3, f), device=DEV, dtype=torch.int8)
    s = torch.full((n,), 0.5, device=DEV)
    rp = torch.zeros(n + 1, dtype=torch.int64, device=DEV)
    rp[-1] = 3
    col = torch.tensor([n - 3, n - 2, n - 1], dtype=torch.int32, device=DEV)
    out = torch.ones(n, f, device=DEV)
    I.spmm_int8_forward_(rp, col, x, s, out)
    assert torch.equal(out[-1], x[-3:].float().sum(0) * 0.5)
    assert int(torch.count_nonzero(out[:-1])) == 0


def test_nan_scale_poisons_its_readers_only():
    rp = torch.tensor([0, 2, 3, 3], dtype=torch.int32, device=DEV)
    col = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    x = torch.ones(3, 32, dtype=torch.int8, device=DEV)
    s = torch.tensor([1.0, float("nan"), 2.0], device=DEV)
    out = torch.empty(3, 32, device=DEV)
    I.spmm_int8_forward_(rp, col, x, s, out)
    assert bool(torch.isnan(out[0]).all()) and bool((out[1] == 2).all()) and bool((out[2] == 0).all())
