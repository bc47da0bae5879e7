"""The 8-bit path at sizes where each block works through several tiles, chunks or windows
(run with -m gpu): reused accumulators and staging, column tiles that follow one another,
tabulated GCN scales, long shares. References are made on the GPU in 64 bits.
"""
import ctypes

import pytest
import torch

from gnn_cuda_b200 import _native as N
from gnn_cuda_b200.GNN_cuda_common import int8_ops as I

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _status():
    status = ctypes.c_int(-1)
    N.check(N.lib().gnn_device_status(1, ctypes.byref(status)))
    return status.value


def _rows8(rows, cols, g):
    t = I.empty_rows(rows, cols, DEV)
    t.copy_(torch.randint(-127, 128, (rows, cols), device=DEV, generator=g, dtype=torch.int8))
    return t


def _quantize(y):
    s = (y.abs().amax(1).double() / 127).float()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    return torch.round(y.double() / safe.double()[:, None]).clamp(-127, 127).to(torch.int8), s


# (blocks that share an SM, output columns)
WIDTHS = [(3, 20), (2, 60), (1, 100), (1, 250)]


def _check_linear(m, k, n, relu):
    g = torch.Generator(device=DEV).manual_seed(m + k + n)
    x, w = _rows8(m, k, g), _rows8(n, k, g)
    sx = torch.rand(m, device=DEV, generator=g) + 0.1
    sw = torch.rand(n, device=DEV, generator=g) + 0.1
    b = torch.randn(n, device=DEV, generator=g) * 100
    want = (x.double() @ w.double().t()).float()  # whole numbers below 2^53
    want.mul_(sx[:, None]).mul_(sw).add_(b)
    if relu:
        want = torch.where(want < 0, torch.zeros_like(want), want)
    out = torch.full((m, n), float("nan"), device=DEV)
    I.linear_int8_forward_(x, sx, w, sw, b, out, relu)
    assert torch.equal(out, want)
    o8, os_ = I.empty_rows(m, n, DEV), torch.empty(m, device=DEV)
    I.linear_int8_forward_(x, sx, w, sw, b, o8, relu, out_scale=os_)
    eq, es = _quantize(want)
    assert torch.equal(os_, es) and torch.equal(o8, eq)
    assert _status() == 0


@pytest.mark.parametrize("per_sm,n", WIDTHS)
def test_several_row_tiles_per_block(per_sm, n):
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    _check_linear(4 * per_sm * sms * 128 + 5, 64, n, True)


@pytest.mark.parametrize("n", [257, 700])
@pytest.mark.parametrize("k", [64, 1100])
def test_several_column_tiles_per_block(k, n):
    _check_linear(40_003, k, n, False)


def test_long_k_one_column_tile():
    _check_linear(4 * 148 * 128 + 77, 1100, 200, True)


@pytest.mark.parametrize("m,k", [(1, 2048), (1, 2049), (1, 4096), (1, 40_000), (2, 2047), (2, 4096), (4, 2049),
                                 (8, 1024)])
def test_few_long_rows(m, k):
    """fp32 rows beside the limits of the few-rows kernel: the bits of quantiser and 8-bit transform."""
    _check_linear(m, k, 300, False)
    g = torch.Generator(device=DEV).manual_seed(k)
    x, w = torch.randn(m, k, device=DEV, generator=g), _rows8(300, k, g)
    sw = torch.rand(300, device=DEV, generator=g) + 0.1
    q, s = I.empty_rows(m, k, DEV), torch.empty(m, device=DEV)
    I.quantize_rows_(x, q, s)
    eq, es = _quantize(x)
    assert torch.equal(q, eq) and torch.equal(s, es)
    want, out = torch.empty(m, 300, device=DEV), torch.empty(m, 300, device=DEV)
    I.linear_int8_forward_(q, s, w, sw, None, want)
    I.linear_int8_forward_(x, None, w, sw, None, out)
    assert torch.equal(out, want)


def _check_spmm(n, nnz, f, agg, index, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    # skewed degrees: hubs over many shares, rows without entries
    row = (torch.rand(nnz, device=DEV, generator=g, dtype=torch.float64) ** 3 * n).long().clamp_(max=n - 1)
    row = row.sort().values
    deg = torch.bincount(row, minlength=n)
    rp = torch.cat([deg.new_zeros(1), deg.cumsum(0)]).to(index)
    col = torch.randint(0, n, (nnz,), device=DEV, generator=g)
    x = _rows8(n, f, g)
    s = torch.rand(n, device=DEV, generator=g) + 0.1
    dis = torch.rand(n, device=DEV, generator=g) + 0.1
    ew = torch.randn(nnz, device=DEV, generator=g)
    w = s.double()[col]
    if agg == "gcn":
        w = w * dis.double()[row] * dis.double()[col]
    elif agg == "weighted":
        w = w * ew.double()
    elif agg == "mean":
        w = w / deg.double()[row]
    out = torch.full((n, f), float("nan"), device=DEV)
    I.spmm_int8_forward_(rp, col.to(torch.int32), x, s, out, aggregation=agg,
                         deg_inv_sqrt=dis if agg == "gcn" else None, edge_weight=ew if agg == "weighted" else None)
    for c0 in range(0, f, 64):
        terms = x[:, c0:c0 + 64][col].double() * w[:, None]
        zero = torch.zeros(n, terms.shape[1], dtype=torch.float64, device=DEV)
        want, size = zero.index_add(0, row, terms), zero.index_add(0, row, terms.abs())
        # d additions and four roundings of weights, first order; 1.01 for the rest
        bound = 1.01 * (deg[:, None] + 4) * 2.0 ** -24 * size
        assert bool(((out[:, c0:c0 + 64].double() - want).abs() <= bound).all())
    assert _status() == 0


@pytest.mark.parametrize("f", [40, 128, 201, 300])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_gcn_of_many_entries(f, index):
    _check_spmm(60_000, 1_300_000, f, "gcn", index, f)


@pytest.mark.parametrize("nnz", [(1 << 20) - 1, 1 << 20])
def test_gcn_beside_the_tabulated_scales(nnz):
    _check_spmm(50_000, nnz, 72, "gcn", torch.int32, 3)


@pytest.mark.parametrize("agg", ["sum", "mean", "weighted"])
@pytest.mark.parametrize("f", [201, 300, 530])
def test_long_shares(agg, f):
    _check_spmm(60_000, 1_300_000, f, agg, torch.int32, f)
