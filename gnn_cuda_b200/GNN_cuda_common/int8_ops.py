"""The 8-bit inference path: features and weights held in signed 8-bit integers
with one fp32 scale per row (per node, per output channel).

The reference holds every feature in fp32; these calls stand beside
``linear_forward_`` and the ``spmm_*_forward_`` family for users whose features
should take a quarter of the memory and of the gather traffic. An 8-bit matrix is
a tensor ``q`` of ``torch.int8`` and a tensor ``scale`` of float32, element
``(i, j)`` standing for ``q[i, j] * scale[i]``:

    q, s = empty_rows(n, f, device), torch.empty(n, device=device)
    quantize_rows_(features, q, s)                         # once, or per step
    wq, ws = empty_rows(out_dim, f, device), torch.empty(out_dim, device=device)
    quantize_weight_(weight, wq, ws)                       # once, weight [f, out_dim]
    linear_int8_forward_(q, s, wq, ws, bias, out, relu=True)

Checks raise RuntimeError; calls run on the current stream of the output's device,
write preallocated outputs and never synchronise. Scratch memory is taken from
PyTorch's caching allocator per call, so calls on several streams and captured
graphs never share it.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .native_ops import _check, _index_type, _stream


def empty_rows(rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised [rows, cols] int8 storage whose rows start on 16-byte boundaries,
    the layout every call here reads without repacking."""
    return torch.empty(int(rows), (int(cols) + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :int(cols)]


def _on_device(name: str, t: torch.Tensor, device: torch.device) -> None:
    _check(t.is_cuda, f"{name} must be CUDA")
    _check(t.device == device, f"{name} must be on the device of out")


def _check_rows8(name: str, t: torch.Tensor) -> None:
    _check(t.dtype == torch.int8, f"{name} must be int8")
    _check(t.dim() == 2, f"{name} must be rank-2")
    _check(t.size(1) <= 1 or t.stride(1) == 1, f"{name} must have contiguous rows")
    _check(t.size(0) <= 1 or t.stride(0) >= t.size(1), f"{name} must not have overlapping rows")


def _check_f32(name: str, t: torch.Tensor, dim: int, device: torch.device) -> None:
    _on_device(name, t, device)
    _check(t.dtype == torch.float32, f"{name} must be float32")
    _check(t.dim() == dim, f"{name} must be rank-{dim}")
    _check(t.is_contiguous(), f"{name} must be contiguous")


def _ld(t: torch.Tensor) -> int:
    """Elements from row to row (a tensor of one row may report any stride)."""
    return int(t.stride(0)) if t.size(0) > 1 else max(int(t.stride(0)), int(t.size(1)))


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors of contiguous rows meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    end = lambda t: t.data_ptr() + ((t.size(0) - 1) * t.stride(0) + (t.size(1) if t.dim() > 1 else 1)) * t.element_size()  # noqa: E731
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


class _Device:
    """torch.cuda.device without its cost where the device is current already."""

    def __init__(self, device: torch.device):
        self.index = device.index
        self.old = -1

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.index:
            self.old = now
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.old >= 0:
            torch.cuda.set_device(self.old)


def quantize_rows_(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """scale[i] = max|x[i]| / 127; q[i] = x[i] / scale[i] to the nearest integer, ties to
    even, on the exact quotient. Zero rows: scale 0, q 0. Rows with a NaN or an
    infinity: scale NaN, q 0 (what is computed from them is NaN)."""
    _on_device("q", q, q.device)
    _check_rows8("q", q)
    _check_f32("x", x, 2, q.device)
    _check_f32("scale", scale, 1, q.device)
    _check(tuple(x.shape) == tuple(q.shape), "x and q must have the same shape")
    _check(scale.numel() == x.size(0), "scale length must equal the number of rows")
    with _Device(q.device):
        N.call("gnn_quantize_rows", x.data_ptr(), x.size(1), x.size(0), x.size(1), q.data_ptr(), _ld(q),
               scale.data_ptr(), _stream(q.device))


def quantize_weight_(weight: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """weight [in, out] (the layout of linear_forward_) as q [out, in] with one scale per output channel."""
    _on_device("q", q, q.device)
    _check_rows8("q", q)
    _check_f32("weight", weight, 2, q.device)
    _check_f32("scale", scale, 1, q.device)
    _check(weight.size(0) == q.size(1) and weight.size(1) == q.size(0), "q must be [out, in] for weight [in, out]")
    _check(scale.numel() == q.size(0), "scale length must equal the number of output channels")
    with _Device(q.device):
        N.call("gnn_quantize_weight", weight.data_ptr(), weight.size(0), weight.size(1), q.data_ptr(), _ld(q),
               scale.data_ptr(), _stream(q.device))


def linear_int8_forward_(x: torch.Tensor, x_scale: torch.Tensor | None, weight: torch.Tensor,
                         weight_scale: torch.Tensor, bias: torch.Tensor | None, out: torch.Tensor,
                         relu: bool = False, out_scale: torch.Tensor | None = None) -> None:
    """out = relu?(x · weightᵀ * scales + bias) on the 8-bit tensor cores.

    x: int8 [m, k] with x_scale [m], or float32 [m, k] with x_scale None (its rows are
    quantised on the way). weight: int8 [n, k] with weight_scale [n]
    (``quantize_weight_``). out: float32 [m, n], or int8 [m, n] with out_scale [m]
    (quantised as ``quantize_rows_`` would quantise the float32 result)."""
    dev = out.device
    _check(out.is_cuda, "out must be CUDA")
    _on_device("x", x, dev)
    _on_device("weight", weight, dev)
    _check_rows8("weight", weight)
    _check_f32("weight_scale", weight_scale, 1, dev)
    if x.dtype == torch.int8:
        _check_rows8("x", x)
        _check(x_scale is not None, "x_scale is needed for int8 x")
        _check_f32("x_scale", x_scale, 1, dev)
        _check(x_scale.numel() == x.size(0), "x_scale length must equal the number of rows")
        x_type = N.GNN_ROWS_INT8
    else:
        _check(x.dtype == torch.float32, "x must be int8 or float32")
        _check_f32("x", x, 2, dev)
        _check(x_scale is None, "x_scale must be None for float32 x")
        x_type = N.GNN_ROWS_FP32
    m, k, n = x.size(0), x.size(1), weight.size(0)
    _check(k == weight.size(1), "Inner GEMM dimensions must match")
    _check(k >= 1, "x must have at least one column")
    _check(weight_scale.numel() == n, "weight_scale length must equal the number of output channels")
    _check(out.dim() == 2 and out.size(0) == m and out.size(1) == n, "Output shape must match x @ weight")
    if out.dtype == torch.int8:
        _check_rows8("out", out)
        _check(out_scale is not None, "out_scale is needed for int8 out")
        _check_f32("out_scale", out_scale, 1, dev)
        _check(out_scale.numel() == m, "out_scale length must equal the number of rows")
        out_type = N.GNN_ROWS_INT8
    else:
        _check(out.dtype == torch.float32, "out must be int8 or float32")
        _check(out.is_contiguous(), "out must be contiguous")
        _check(out_scale is None, "out_scale must be None for float32 out")
        out_type = N.GNN_ROWS_FP32
    if bias is not None and bias.numel() != 0:
        _check_f32("bias", bias, 1, dev)
        _check(bias.numel() == n, "bias length must equal output feature dimension")
        bias_ptr = bias.data_ptr()
    else:
        bias_ptr = None
    _check(not _overlap(out, x), "out must not alias x")
    L = N.lib()
    xp, ldx, wp, ldw = x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight)
    with _Device(dev):
        wsb = L.gnn_linear_int8_workspace_bytes(xp, x_type, ldx, wp, ldw, out_type, m, k, n)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        N.check(L.gnn_linear_int8_forward(
            xp, x_type, ldx, None if x_scale is None else x_scale.data_ptr(), wp, ldw, weight_scale.data_ptr(), bias_ptr,
            out.data_ptr(), out_type, _ld(out), None if out_scale is None else out_scale.data_ptr(), m, k, n,
            1 if relu else 0, None if ws is None else ws.data_ptr(), wsb, _stream(dev)), "gnn_linear_int8_forward")


_WEIGHTING = {"sum": N.GNN_WEIGHT_SUM, "mean": N.GNN_WEIGHT_MEAN, "gcn": N.GNN_WEIGHT_GCN,
              "weighted": N.GNN_WEIGHT_EDGE}


def spmm_int8_forward_(row_ptr: torch.Tensor, col_ind: torch.Tensor, x: torch.Tensor, x_scale: torch.Tensor,
                       out: torch.Tensor, aggregation: str = "sum", deg_inv_sqrt: torch.Tensor | None = None,
                       edge_weight: torch.Tensor | None = None) -> None:
    """out[r] = f_r * sum_e w_e * x_scale[c] * x[c] over the entries e = (r, c) of a CSR, in float32.

    aggregation: "sum"; "mean" (divided by the degree); "gcn" (deg_inv_sqrt[r] *
    deg_inv_sqrt[c]); "weighted" (edge_weight[e]) — the weightings of
    ``spmm_sum_forward_``, ``spmm_mean_forward_``, ``spmm_gcn_forward_`` and
    ``spmm_pyg_gcn_forward_``. x: int8 [num_nodes, f] with x_scale [num_nodes]; out:
    float32 [num_nodes, f]. Rows are summed in another order than the float32
    aggregations, the same one in every call."""
    dev = out.device
    _check(out.is_cuda, "out must be CUDA")
    _check(aggregation in _WEIGHTING, "aggregation must be sum, mean, gcn or weighted")
    for name, t in (("row_ptr", row_ptr), ("col_ind", col_ind), ("x", x)):
        _on_device(name, t, dev)
    for name, t in (("row_ptr", row_ptr), ("col_ind", col_ind)):
        _check(t.is_contiguous(), f"{name} must be contiguous")
        _check(t.dim() == 1, f"{name} must be rank-1")
    _check(row_ptr.dtype in (torch.int32, torch.int64), "row_ptr must be int32")
    _check(col_ind.dtype == torch.int32, "col_ind must be int32")
    _check_rows8("x", x)
    _check_f32("x_scale", x_scale, 1, dev)
    _check_f32("out", out, 2, dev)
    _check(tuple(x.shape) == tuple(out.shape), "x and out must have the same shape")
    n, f, nnz = x.size(0), x.size(1), col_ind.numel()
    _check(x_scale.numel() == n, "x_scale length must equal num_nodes")
    _check(row_ptr.numel() == n + 1, "row_ptr length must be num_nodes + 1")
    dis_ptr = ew_ptr = None
    if aggregation == "gcn":
        _check(deg_inv_sqrt is not None, "deg_inv_sqrt is needed for gcn")
        _check_f32("deg_inv_sqrt", deg_inv_sqrt, 1, dev)
        _check(deg_inv_sqrt.numel() == n, "deg_inv_sqrt length must equal num_nodes")
        dis_ptr = deg_inv_sqrt.data_ptr()
    else:
        _check(deg_inv_sqrt is None, "deg_inv_sqrt is only for gcn")
    if aggregation == "weighted":
        _check(edge_weight is not None, "edge_weight is needed for weighted")
        _check_f32("edge_weight", edge_weight, 1, dev)
        _check(edge_weight.numel() == nnz, "col_ind and edge_weight lengths must match")
        ew_ptr = edge_weight.data_ptr()
    else:
        _check(edge_weight is None, "edge_weight is only for weighted")
    _check(not _overlap(out, x), "out must not alias x")
    L = N.lib()
    with _Device(dev):
        wsb = L.gnn_spmm_int8_workspace_bytes(n, nnz, f)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        N.check(L.gnn_spmm_int8_forward(
            row_ptr.data_ptr(), _index_type(row_ptr), col_ind.data_ptr(), _WEIGHTING[aggregation], dis_ptr, ew_ptr,
            x.data_ptr(), _ld(x), x_scale.data_ptr(), out.data_ptr(), n, nnz, f, ws.data_ptr(), wsb, _stream(dev)),
            "gnn_spmm_int8_forward")
