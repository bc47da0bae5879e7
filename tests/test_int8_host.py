"""Refusals of the 8-bit path that need no device: C entry points and Python checks."""
import pytest
import torch

from gnn_cuda_b200 import _native as N
from gnn_cuda_b200.GNN_cuda_common import int8_ops as I


def _linear(m, k, n, x=1 << 20, x_type=1, ldx=None, xs=1 << 20, w=1 << 20, out=1 << 20, out_type=0, ldo=None, os_=None):
    return N.lib().gnn_linear_int8_forward(x, x_type, k if ldx is None else ldx, xs, w, k, 1 << 20, None, out, out_type,
                                           n if ldo is None else ldo, os_, m, k, n, 0, None, 0, None)


def test_c_entry_refusals():
    assert _linear(4, 0, 4) == 1 and "k >= 1" in N.last_error()
    assert _linear(-1, 8, 4) == 1
    assert _linear(4, 8, 4, x_type=2) == 1 and "row types" in N.last_error()
    assert _linear(4, 131072, 4) == 3 and "131071" in N.last_error()
    assert _linear(4, 16, 4, ldx=8) == 1 and "strides" in N.last_error()
    assert _linear(4, 16, 4, xs=None) == 2 and "x_scale" in N.last_error()
    assert _linear(4, 16, 4, out_type=1) == 2 and "out_scale" in N.last_error()
    assert _linear(4, 16, 4, x=None) == 2
    assert _linear(0, 16, 4) == 0 and _linear(4, 16, 0) == 0
    L = N.lib()
    assert L.gnn_quantize_rows(None, 4, 3, 4, None, 4, None, None) == 2
    assert L.gnn_quantize_rows(1 << 20, 3, 3, 4, 1 << 20, 4, 1 << 20, None) == 1
    assert L.gnn_quantize_rows(None, 4, 0, 4, None, 4, None, None) == 0
    assert L.gnn_quantize_weight(None, 4, 3, None, 4, None, None) == 2
    assert L.gnn_quantize_weight(1 << 20, 8, 3, 1 << 20, 4, 1 << 20, None) == 1


def test_workspace_query():
    q = N.lib().gnn_linear_int8_workspace_bytes
    al, un = 1 << 20, (1 << 20) + 1
    assert q(al, 1, 128, al, 128, 0, 1000, 128, 64) == 0
    assert q(al, 1, 128, al, 128, 1, 1000, 128, 256) == 0
    assert q(al, 0, 100, al, 112, 0, 1000, 100, 64) >= 1000 * 112 + 4000       # fp32 rows: quantised copy and scales
    assert q(un, 1, 128, al, 128, 0, 1000, 128, 64) >= 1000 * 128              # unaligned rows: repacked
    assert q(al, 1, 128, al, 129, 0, 1000, 128, 64) >= 64 * 128
    assert q(al, 1, 128, al, 128, 1, 1000, 128, 257) >= 4 * 1000 * 257         # wide 8-bit rows: fp32 first
    assert q(al, 1, 128, al, 128, 0, 0, 128, 64) == 0


def test_python_refusals():
    x8, s = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        I.quantize_rows_(torch.zeros(4, 8), x8, s)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        I.quantize_weight_(torch.zeros(8, 4), x8, s)
    with pytest.raises(RuntimeError, match="out must be CUDA"):
        I.linear_int8_forward_(x8, s, x8, s, None, torch.zeros(4, 4))
    t = I.empty_rows(5, 21, "cpu")
    assert t.shape == (5, 21) and t.stride(0) == 32


def test_overlap_check():
    base = torch.empty(10, 32, dtype=torch.int8)

    def apart(a, b):
        I._check_apart(a, a.data_ptr(), a.stride(0), b, b.data_ptr(), b.stride(0))

    apart(base[:2], base[3:])
    apart(base[5:], base[:5, :7])
    apart(base[:0], base)
    for a, b in ((base, base[2:]), (base[2:], base), (base[3:6], base[5:])):
        with pytest.raises(RuntimeError, match="must not alias"):
            apart(a, b)


def test_spmm_c_refusals():
    L = N.lib()
    p = 1 << 20
    call = lambda n=4, e=4, f=8, ty=0, wt=0, dis=None, ew=None, x=p, ldx=8, ws=None, wsb=0: L.gnn_spmm_int8_forward(  # noqa: E731
        p, ty, p, wt, dis, ew, x, ldx, p, p, n, e, f, ws, wsb, None)
    assert call(n=-1) == 1 and call(ty=4) == 1 and call(wt=4) == 1 and call(wt=-1) == 1
    assert call(e=1 << 31) == 1 and "int64 row_ptr" in N.last_error()
    assert call(ldx=7) == 1
    assert call(wt=2) == 2 and call(wt=3) == 2 and call(x=None) == 2
    assert call() == 7 and "workspace" in N.last_error()
    assert call(n=0) == 0 and call(f=0) == 0
    assert L.gnn_spmm_int8_workspace_bytes(1000, 5000, 128) > 0


def test_spmm_python_refusals():
    rp, ci = torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="out must be CUDA"):
        I.spmm_int8_forward_(rp, ci, torch.zeros(4, 8, dtype=torch.int8), torch.ones(4), torch.zeros(4, 8))


@pytest.mark.parametrize("argv,match", [
    (["--features", "int8"], "needs a CUDA device and device placement"),
    (["--norm", "node"], "needs a CUDA device"),
    (["--norm", "graph", "--norm_groups", "3"], "must divide the hidden dimension"),
])
def test_driver_refusals(argv, match):
    from gnn_cuda_b200.GNN_cuda_common import gcn_inference
    with pytest.raises(ValueError, match=match):
        gcn_inference.run_gcn_inference(framework_label="pyg", select_device=torch.device, load_graph_features=None,
                                        load_kind="pyg", argv=["--device", "cpu", "--memory_mode", "device", *argv])
