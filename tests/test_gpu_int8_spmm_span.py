"""The aggregation over 8-bit rows takes its entries from row_ptr (run with -m gpu).

col_ind and edge_weight may be longer than what row_ptr spans, before its first entry and
behind its last; out is the middle of a filled buffer, whose rest must stay as it is.

Bound as in test_gpu_int8_spmm.py: (d + 4) * 2^-24 * sum_e |w_e s_c q_c| for a row of d
entries, 1.01 for the higher orders.
"""
import ctypes

import numpy as np
import pytest
import scipy.sparse as sp
import torch

from gnn_cuda_b200 import _native as N
from gnn_cuda_b200.GNN_cuda_common import int8_ops as I
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FILL = 12345.0
OUTSIDE = 39  # status: row_ptr spans entries outside col_ind


def _status():
    status = ctypes.c_int(-1)
    N.check(N.lib().gnn_device_status(1, ctypes.byref(status)))
    return status.value


def _run(degrees, f, agg, index, front=0, slack=0, seed=1):
    """The CSR of `degrees` with `front` foreign entries before it and `slack` behind it; entries
    that a negative slack cuts off do not count."""
    r = np.random.default_rng(seed)
    n = len(degrees)
    rp = front + np.concatenate([[0], np.cumsum(degrees)])
    size = rp[-1] + slack
    col = r.integers(0, n, size).astype(np.int32)
    ew = r.standard_normal(size).astype(np.float32)
    q, s = O.quantize(r.standard_normal((n, f)).astype(np.float32))
    dis = r.random(n).astype(np.float32) + np.float32(0.1)
    held = np.minimum(rp, size)  # rows over the entries that exist
    deg = np.diff(held)
    row = np.repeat(np.arange(n), deg)
    c = col[held[0]:held[-1]]
    w = s[c].astype(np.float64)
    if agg == "gcn":
        w = w * dis[row] * dis[c]
    elif agg == "weighted":
        w = w * ew[held[0]:held[-1]]
    elif agg == "mean":
        w = w / deg[row]
    a = sp.csr_matrix((w, c, held - held[0]), shape=(n, n), copy=True)
    want, size_ = a @ q.astype(np.float64), abs(a) @ np.abs(q.astype(np.float64))
    x = I.empty_rows(n, f, DEV)
    x.copy_(torch.from_numpy(q))
    around = torch.full((n + 8, f), FILL, device=DEV)
    out = around[4:4 + n]
    I.spmm_int8_forward_(torch.from_numpy(rp.astype(index)).to(DEV), torch.from_numpy(col).to(DEV), x,
                         torch.from_numpy(s).to(DEV), out, aggregation=agg,
                         deg_inv_sqrt=torch.from_numpy(dis).to(DEV) if agg == "gcn" else None,
                         edge_weight=torch.from_numpy(ew).to(DEV) if agg == "weighted" else None)
    err = np.abs(out.cpu().numpy().astype(np.float64) - want)
    assert np.all(err <= 1.01 * (deg[:, None] + 4) * 2.0 ** -24 * size_)
    assert bool((around[:4] == FILL).all()) and bool((around[4 + n:] == FILL).all())


def _degrees(n, seed=3):
    r = np.random.default_rng(seed)
    d = r.integers(0, 9, n)
    d[n // 3] = 900  # a row over several shares
    return d


@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("agg", ["sum", "mean", "gcn", "weighted"])
@pytest.mark.parametrize("front,slack", [(0, 0), (0, 1), (0, 1000), (5, 0), (5, 1), (700, 1000)])
def test_entries_outside_the_rows(agg, index, front, slack):
    _run(_degrees(501), 40, agg, index, front, slack)
    assert _status() == 0


@pytest.mark.parametrize("n,deg", [(1, 0), (1, 1), (40, 3), (64, 1)])
@pytest.mark.parametrize("f", [1, 128, 300])
def test_small_graphs_with_slack(n, deg, f):
    _run(np.full(n, deg), f, "mean", np.int32, 2, 1)
    _run(np.full(n, deg), f, "gcn", np.int64, 0, 33)
    assert _status() == 0


@pytest.mark.parametrize("index", [np.int32, np.int64])
@pytest.mark.parametrize("missing", [1, 33, 1500])
def test_fewer_entries_than_row_ptr_spans(index, missing):
    """The rows hold what there is, and the status word says so."""
    assert _status() == 0
    _run(_degrees(501), 40, "weighted", index, 0, -missing)
    assert _status() == OUTSIDE
    assert _status() == 0


def test_as_many_nodes_as_are_accepted():
    """2^31 - 1 nodes: the rows behind the last one are not looked up at negative places."""
    n, deg = (1 << 31) - 1, 5
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    rp = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    rp[-1] = deg
    col = torch.tensor([n - 1, 0, n - 2, n - 1, 7], dtype=torch.int32, device=DEV)
    x = torch.zeros(n, 1, dtype=torch.int8, device=DEV)
    x[-2:, 0] = torch.tensor([3, -100], dtype=torch.int8, device=DEV)
    x[0], x[7] = 11, 1
    s = torch.full((n,), 0.5, device=DEV)
    out = torch.ones(n, 1, device=DEV)
    I.spmm_int8_forward_(rp, col, x, s, out)
    assert float(out[-1]) == 0.5 * (-100 + 11 + 3 - 100 + 1)
    assert int(torch.count_nonzero(out[:-1])) == 0
    assert _status() == 0
    with pytest.raises(RuntimeError, match="2\\^31 - 1"):
        N.check(N.lib().gnn_spmm_int8_forward(rp.data_ptr(), N.GNN_INDEX_INT32, col.data_ptr(), N.GNN_WEIGHT_SUM, None,
                                              None, x.data_ptr(), 1, s.data_ptr(), out.data_ptr(), n + 1, deg, 1, None,
                                              0, None))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", ["alternate", "runs", "ends", "none"])
def test_rows_without_entries_whose_factor_is_infinite(kind, index):
    """deg_inv_sqrt = degree^-0.5 is infinite for isolated nodes, whose rows are 0, as in the fp32 aggregation."""
    from gnn_cuda_b200.GNN_cuda_common import gcn_ops
    n, f = 2003, 48
    r = np.random.default_rng(4)
    deg = {"alternate": np.arange(n) % 2 * 3, "runs": (np.arange(n) // 70 % 2) * r.integers(1, 9, n),
           "ends": np.where((np.arange(n) < 90) | (np.arange(n) > n - 40), 0, 2), "none": np.zeros(n, np.int64)}[kind]
    rp = torch.from_numpy(np.concatenate([[0], np.cumsum(deg)])).to(DEV, index)
    full = np.flatnonzero(deg) if deg.any() else np.zeros(1, np.int64)
    col = torch.from_numpy(r.choice(full, int(deg.sum())).astype(np.int32)).to(DEV)
    dis = torch.from_numpy(deg).to(DEV).float().pow(-0.5)
    x = torch.randint(-127, 128, (n, f), device=DEV).to(torch.int8)
    s = torch.rand(n, device=DEV)
    out, ref = torch.empty(n, f, device=DEV), torch.empty(n, f, device=DEV)
    I.spmm_int8_forward_(rp, col, x, s, out, aggregation="gcn", deg_inv_sqrt=dis)
    gcn_ops.spmm_gcn_forward_(rp, col, dis, x.float() * s[:, None], ref)
    empty = torch.from_numpy(deg == 0).to(DEV)
    assert int(torch.count_nonzero(out[empty])) == 0 and int(torch.count_nonzero(ref[empty])) == 0
    # both sides: 8 additions, the product by the scale and three of weights, each 2^-24 of at most 127 per entry
    assert float((out - ref).abs().max()) <= 2 * 12 * 2.0 ** -24 * 127 * 9
