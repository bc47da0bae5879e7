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

import functools

import torch

from .. import _native as N
from .native_ops import _check, _index_type


def empty_rows(rows: int, cols: int, device) -> torch.Tensor:
    """Uninitialised [rows, cols] int8 storage whose rows start on 16-byte boundaries,
    the layout every call here reads without repacking."""
    return torch.empty(int(rows), (int(cols) + 15) // 16 * 16, dtype=torch.int8, device=device)[:, :int(cols)]


# The checks below are written for what they cost: small calls are bound by the host.
# _current_stream and _current_device are torch.cuda.current_stream(d).cuda_stream and
# torch.cuda.current_device() without the objects around them.
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_I8, _F32 = torch.int8, torch.float32


def _device_of(out: torch.Tensor, name: str = "out") -> int:
    """The output's device index; it is made current by _on() around the call."""
    index = out.get_device()
    if index < 0 or not out.is_cuda:
        _check(False, f"{name} must be CUDA")
    return index


def _same_device(name: str, t: torch.Tensor, index: int) -> None:
    if t.get_device() != index or not t.is_cuda:
        _check(t.is_cuda, f"{name} must be CUDA")
        _check(False, f"{name} must be on the device of out")


def _check_rows8(name: str, t: torch.Tensor, index: int) -> int:
    """Checks an int8 matrix of contiguous rows; returns the elements from row to row."""
    _same_device(name, t, index)
    if t.dtype is not _I8:
        _check(False, f"{name} must be int8")
    if t.dim() != 2:
        _check(False, f"{name} must be rank-2")
    rows, cols = t.shape
    ld, step = t.stride()
    if cols > 1 and step != 1:
        _check(False, f"{name} must have contiguous rows")
    if rows > 1:
        if ld < cols:
            _check(False, f"{name} must not have overlapping rows")
        return ld
    return ld if ld > cols else cols  # a tensor of one row may report any stride


def _check_f32(name: str, t: torch.Tensor, dim: int, index: int) -> None:
    _same_device(name, t, index)
    if t.dtype is not _F32:
        _check(False, f"{name} must be float32")
    if t.dim() != dim:
        _check(False, f"{name} must be rank-{dim}")
    if not t.is_contiguous():
        _check(False, f"{name} must be contiguous")


def _check_vector(name: str, t: torch.Tensor, length: int, index: int, what: str) -> None:
    _check_f32(name, t, 1, index)
    if t.shape[0] != length:
        _check(False, f"{name} length must equal {what}")


def _check_apart(out: torch.Tensor, out_ptr: int, out_ld: int, x: torch.Tensor, x_ptr: int, x_ld: int,
                 what: str = "out must not alias x") -> None:
    """Refuses an output whose address range meets that of x (matrices of contiguous rows)."""
    if out_ptr <= x_ptr:
        m, n = out.shape
        first, last = x_ptr, out_ptr + ((m - 1) * out_ld + n) * out.element_size()
    else:
        m, n = x.shape
        first, last = out_ptr, x_ptr + ((m - 1) * x_ld + n) * x.element_size()
    if first < last and out.numel() and x.numel():
        _check(False, what)


class _On:
    """torch.cuda.device(index), at the cost of one query where it is current already."""

    __slots__ = ("index", "old")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        now = _current_device() if _current_device else torch.cuda.current_device()
        self.old = now
        if now != self.index:
            torch.cuda.set_device(self.index)
        return _current_stream(self.index) if _current_stream else torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.old != self.index:
            torch.cuda.set_device(self.old)


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor | None:
    """Uninitialised bytes on the device of `like`, from the allocator's pool of the current stream."""
    return like.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _launch(index: int, call):
    """call(stream) with the device made current."""
    if _current_device is not None and _current_stream is not None and _current_device() == index:
        return call(_current_stream(index))
    with _On(index) as stream:
        return call(stream)


def quantize_rows_(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """scale[i] = max|x[i]| / 127; q[i] = x[i] / scale[i] to the nearest integer, ties to
    even, on the exact quotient. Zero rows: scale 0, q 0. Rows with a NaN or an
    infinity: scale NaN, q 0 (what is computed from them is NaN)."""
    index = _device_of(q, "q")
    ldq = _check_rows8("q", q, index)
    _check_f32("x", x, 2, index)
    rows, cols = x.shape
    _check(x.shape == q.shape, "x and q must have the same shape")
    _check_vector("scale", scale, rows, index, "the number of rows")
    _check_apart(q, q.data_ptr(), ldq, x, x.data_ptr(), cols, "q must not alias x")
    with _On(index) as stream:
        N.check(N.lib().gnn_quantize_rows(x.data_ptr(), cols, rows, cols, q.data_ptr(), ldq, scale.data_ptr(), stream),
                "gnn_quantize_rows")


def quantize_weight_(weight: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """weight [in, out] (the layout of linear_forward_) as q [out, in] with one scale per output channel."""
    index = _device_of(q, "q")
    ldq = _check_rows8("q", q, index)
    _check_f32("weight", weight, 2, index)
    k, n = weight.shape
    _check(k == q.shape[1] and n == q.shape[0], "q must be [out, in] for weight [in, out]")
    _check_vector("scale", scale, n, index, "the number of output channels")
    _check_apart(q, q.data_ptr(), ldq, weight, weight.data_ptr(), n, "q must not alias weight")
    with _On(index) as stream:
        N.check(N.lib().gnn_quantize_weight(weight.data_ptr(), k, n, q.data_ptr(), ldq, scale.data_ptr(), stream),
                "gnn_quantize_weight")


def linear_int8_forward_(x: torch.Tensor, x_scale: torch.Tensor | None, weight: torch.Tensor,
                         weight_scale: torch.Tensor, bias: torch.Tensor | None, out: torch.Tensor,
                         relu: bool = False, out_scale: torch.Tensor | None = None) -> None:
    """out = relu?(x · weightᵀ * scales + bias) on the 8-bit tensor cores.

    x: int8 [m, k] with x_scale [m], or float32 [m, k] with x_scale None (its rows are
    quantised on the way). weight: int8 [n, k] with weight_scale [n]
    (``quantize_weight_``). out: float32 [m, n], or int8 [m, n] with out_scale [m]
    (quantised as ``quantize_rows_`` would quantise the float32 result)."""
    m, k, n, ldx, ldw, ldo = (_linear_sizes_quick(x, x_scale, weight, weight_scale, bias, out, out_scale)
                              or _linear_sizes(x, x_scale, weight, weight_scale, bias, out, out_scale))
    xp, wp, op = x.data_ptr(), weight.data_ptr(), out.data_ptr()
    x_type = N.GNN_ROWS_FP32 if x_scale is None else N.GNN_ROWS_INT8
    out_type = N.GNN_ROWS_FP32 if out_scale is None else N.GNN_ROWS_INT8
    lib = N.lib()
    args = (xp, x_type, ldx, None if x_scale is None else x_scale.data_ptr(), wp, ldw, weight_scale.data_ptr(),
            None if bias is None or bias.numel() == 0 else bias.data_ptr(), op, out_type, ldo,
            None if out_scale is None else out_scale.data_ptr(), m, k, n, 1 if relu else 0)

    def call(stream):
        # Most calls on 8-bit rows need no scratch: the entry point says where one does, before it launches
        # anything. fp32 rows need it but for the fewest (and then not for an 8-bit output).
        rc = N.GNN_ERR_WORKSPACE
        if x_scale is not None or (m <= 16 and out_scale is None):
            rc = lib.gnn_linear_int8_forward(*args, None, 0, stream)
        if rc == N.GNN_ERR_WORKSPACE:
            wsb = lib.gnn_linear_int8_workspace_bytes(xp, x_type, ldx, wp, ldw, out_type, m, k, n)
            ws = _scratch(wsb, out)
            rc = lib.gnn_linear_int8_forward(*args, None if ws is None else ws.data_ptr(), wsb, stream)
        return rc

    rc = _launch(out.get_device(), call)
    if rc:
        N.check(rc, "gnn_linear_int8_forward")


def _vector_ok(t: torch.Tensor, length: int, index: int) -> bool:
    return (t.dtype is _F32 and t.get_device() == index and t.shape == (length,)
            and (length < 2 or t.stride(0) == 1))


def _linear_sizes_quick(x, x_scale, weight, weight_scale, bias, out, out_scale):
    """The sizes of a call with fp32 output that passes every check of _linear_sizes, found in fewer steps;
    None where that is not plain."""
    index = out.get_device()
    if out_scale is not None or out.dtype is not _F32 or not out.is_contiguous() or not out.is_cuda:
        return None
    if x.dim() != 2 or weight.dim() != 2 or out.dim() != 2 or weight.dtype is not _I8:
        return None
    (m, k), (n, kw), (mo, no) = x.shape, weight.shape, out.shape
    (ldx, sx), (ldw, sw) = x.stride(), weight.stride()
    if (k != kw or m != mo or n != no or sx != 1 or sw != 1 or ldx < k or ldw < k or k < 1
            or x.get_device() != index or weight.get_device() != index):
        return None
    if x.dtype is _I8:
        if x_scale is None or not _vector_ok(x_scale, m, index):
            return None
    elif x.dtype is not _F32 or x_scale is not None or (ldx != k and m > 1):
        return None
    if not _vector_ok(weight_scale, n, index) or not (bias is None or _vector_ok(bias, n, index)):
        return None
    xp, op = x.data_ptr(), out.data_ptr()
    if not (op + 4 * m * n <= xp or xp + m * ldx * x.element_size() <= op):
        return None
    return m, k, n, ldx, ldw, n


def _linear_sizes(x, x_scale, weight, weight_scale, bias, out, out_scale) -> tuple[int, int, int, int, int, int]:
    """The checks of linear_int8_forward_: (m, k, n, ldx, ldw, ldo)."""
    index = _device_of(out)
    ldw = _check_rows8("weight", weight, index)
    n, k = weight.shape
    _check_vector("weight_scale", weight_scale, n, index, "the number of output channels")
    if x.dtype is _I8:
        ldx = _check_rows8("x", x, index)
        _check(x_scale is not None, "x_scale is needed for int8 x")
        _check_vector("x_scale", x_scale, x.shape[0], index, "the number of rows")
    else:
        _check(x.dtype is _F32, "x must be int8 or float32")
        _check_f32("x", x, 2, index)
        _check(x_scale is None, "x_scale must be None for float32 x")
        ldx = x.shape[1]
    m = x.shape[0]
    _check(k == x.shape[1], "Inner GEMM dimensions must match")
    _check(k >= 1, "x must have at least one column")
    _check(out.dim() == 2 and out.shape[0] == m and out.shape[1] == n, "Output shape must match x @ weight")
    if out.dtype is _I8:
        ldo = _check_rows8("out", out, index)
        _check(out_scale is not None, "out_scale is needed for int8 out")
        _check_vector("out_scale", out_scale, m, index, "the number of rows")
    else:
        _check(out.dtype is _F32, "out must be int8 or float32")
        _check(out.is_contiguous(), "out must be contiguous")
        _check(out_scale is None, "out_scale must be None for float32 out")
        ldo = n
    if bias is not None and bias.numel() != 0:
        _check_vector("bias", bias, n, index, "output feature dimension")
    _check_apart(out, out.data_ptr(), ldo, x, x.data_ptr(), ldx)
    return m, k, n, ldx, ldw, ldo


@functools.lru_cache(maxsize=1024)
def _spmm_workspace(index: int, n: int, nnz: int, f: int) -> int:
    """A size by sizes: asked once for each (the device is current)."""
    return N.lib().gnn_spmm_int8_workspace_bytes(n, nnz, f)


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
    index = _device_of(out)
    weighting = _WEIGHTING.get(aggregation)
    _check(weighting is not None, "aggregation must be sum, mean, gcn or weighted")
    for name, t in (("row_ptr", row_ptr), ("col_ind", col_ind)):
        _same_device(name, t, index)
        if not t.is_contiguous():
            _check(False, f"{name} must be contiguous")
        if t.dim() != 1:
            _check(False, f"{name} must be rank-1")
    row_type = _index_type(row_ptr)
    _check(col_ind.dtype is torch.int32, "col_ind must be int32")
    ldx = _check_rows8("x", x, index)
    _check_f32("out", out, 2, index)
    _check(x.shape == out.shape, "x and out must have the same shape")
    n, f = out.shape
    nnz = col_ind.shape[0]
    if not _vector_ok(x_scale, n, index):
        _check_vector("x_scale", x_scale, n, index, "num_nodes")
    _check(row_ptr.shape[0] == n + 1, "row_ptr length must be num_nodes + 1")
    dis_ptr = ew_ptr = None
    if aggregation == "gcn":
        _check(deg_inv_sqrt is not None, "deg_inv_sqrt is needed for gcn")
        if not _vector_ok(deg_inv_sqrt, n, index):
            _check_vector("deg_inv_sqrt", deg_inv_sqrt, n, index, "num_nodes")
        dis_ptr = deg_inv_sqrt.data_ptr()
    else:
        _check(deg_inv_sqrt is None, "deg_inv_sqrt is only for gcn")
    if aggregation == "weighted":
        _check(edge_weight is not None, "edge_weight is needed for weighted")
        _check_vector("edge_weight", edge_weight, nnz, index, "the number of entries")
        ew_ptr = edge_weight.data_ptr()
    else:
        _check(edge_weight is None, "edge_weight is only for weighted")
    xp, op = x.data_ptr(), out.data_ptr()
    _check_apart(out, op, f, x, xp, ldx)
    args = (row_ptr.data_ptr(), row_type, col_ind.data_ptr(), weighting, dis_ptr, ew_ptr, xp, ldx, x_scale.data_ptr(),
            op, n, nnz, f)

    def call(stream):
        wsb = _spmm_workspace(index, n, nnz, f)
        ws = _scratch(wsb, out)
        return N.lib().gnn_spmm_int8_forward(*args, None if ws is None else ws.data_ptr(), wsb, stream)

    rc = _launch(index, call)
    if rc:
        N.check(rc, "gnn_spmm_int8_forward")
