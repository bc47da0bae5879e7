"""Normalisation between layers: group norm with its activation in one call.

Stands beside ``bias_relu_forward_`` and ``relu_inplace_``, the epilogues of the
reference's layers, which has no normalisation. Node features are [num_nodes,
channels] float32, channels last. Without ``graph_ptr`` every node is normalised on
its own (``torch.nn.GroupNorm`` on [N, C]); with it, over the nodes of each graph of a
batch: ``groups=1`` is a layer norm over a whole graph, ``groups=channels`` an
instance norm, in between a group norm whose spatial axis is the graph's nodes.
"""
from __future__ import annotations

import functools

import torch

from .. import _native as N
from .int8_ops import _check_apart, _check_f32, _check_vector, _device_of, _launch, _same_device, _scratch, _vector_ok
from .native_ops import _check

ACTIVATIONS = {"none": N.GNN_ACT_NONE, "relu": N.GNN_ACT_RELU, "silu": N.GNN_ACT_SILU, "gelu": N.GNN_ACT_GELU}


def group_norm_forward_(x: torch.Tensor, groups: int, weight: torch.Tensor | None, bias: torch.Tensor | None,
                        out: torch.Tensor, graph_ptr: torch.Tensor | None = None, eps: float = 1e-5,
                        activation: str = "none") -> None:
    """out = act((x - mean) / sqrt(var + eps) * weight + bias), biased variance.

    graph_ptr: int32 or int64 [num_graphs + 1] ascending row offsets; rows before the
    first and behind the last are left as they are in out. activation: none, relu,
    silu or gelu (erf). weight / bias: [channels] or None. out may be x itself."""
    index = _device_of(out)
    _check_f32("out", out, 2, index)
    _check_f32("x", x, 2, index)
    if x.shape != out.shape:
        _check(False, "x and out must have the same shape")
    n, c = x.shape
    groups = int(groups)
    if groups < 1 or c % groups:
        _check(False, "groups must be >= 1 and divide the number of channels")
    w_ptr = b_ptr = None
    if weight is not None:
        if not _vector_ok(weight, c, index):
            _check_vector("weight", weight, c, index, "the number of channels")
        w_ptr = weight.data_ptr()
    if bias is not None:
        if not _vector_ok(bias, c, index):
            _check_vector("bias", bias, c, index, "the number of channels")
        b_ptr = bias.data_ptr()
    act = ACTIVATIONS.get(activation)
    _check(act is not None, "activation must be none, relu, silu or gelu")
    eps = float(eps)
    _check(eps >= 0.0, "eps must be >= 0")
    xp, op = x.data_ptr(), out.data_ptr()
    if xp != op:
        _check_apart(out, op, c, x, xp, c)
    ptr, ptr_type, graphs = None, N.GNN_INDEX_INT32, 0
    if graph_ptr is not None:
        _same_device("graph_ptr", graph_ptr, index)
        if graph_ptr.dtype is torch.int64:
            ptr_type = N.GNN_INDEX_INT64
        elif graph_ptr.dtype is not torch.int32:
            _check(False, "graph_ptr must be int32 or int64")
        if graph_ptr.dim() != 1 or not graph_ptr.is_contiguous():
            _check(False, "graph_ptr must be rank-1 and contiguous")
        graphs = graph_ptr.shape[0] - 1
        if graphs < 0:
            _check(False, "graph_ptr must hold num_graphs + 1 offsets")
        ptr = graph_ptr.data_ptr()
    def call(stream):
        wsb = 0 if ptr is None else _workspace(index, n, graphs, groups)
        ws = _scratch(wsb, out)
        return N.lib().gnn_group_norm_forward(xp, ptr, ptr_type, graphs, w_ptr, b_ptr, op, n, c, groups, eps, act,
                                              None if ws is None else ws.data_ptr(), wsb, stream)

    rc = _launch(index, call)
    if rc:
        N.check(rc, "gnn_group_norm_forward")


@functools.lru_cache(maxsize=1024)
def _workspace(index: int, n: int, graphs: int, groups: int) -> int:
    """A size by sizes: asked once for each (the device is current)."""
    return N.lib().gnn_group_norm_workspace_bytes(n, graphs, groups)
