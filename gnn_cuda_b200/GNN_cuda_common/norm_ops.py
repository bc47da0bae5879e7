"""Normalisation between layers: group norm with its activation in one call.

Stands beside ``bias_relu_forward_`` and ``relu_inplace_``, the epilogues of the
reference's layers, which has no normalisation. Node features are [num_nodes,
channels] float32, channels last. Without ``graph_ptr`` every node is normalised on
its own (``torch.nn.GroupNorm`` on [N, C]); with it, over the nodes of each graph of a
batch: ``groups=1`` is a layer norm over a whole graph, ``groups=channels`` an
instance norm, in between a group norm whose spatial axis is the graph's nodes.
"""
from __future__ import annotations

import torch

from .. import _native as N
from .int8_ops import _check_f32, _Device, _on_device, _overlap
from .native_ops import _check, _index_type, _stream

ACTIVATIONS = {"none": N.GNN_ACT_NONE, "relu": N.GNN_ACT_RELU, "silu": N.GNN_ACT_SILU, "gelu": N.GNN_ACT_GELU}


def group_norm_forward_(x: torch.Tensor, groups: int, weight: torch.Tensor | None, bias: torch.Tensor | None,
                        out: torch.Tensor, graph_ptr: torch.Tensor | None = None, eps: float = 1e-5,
                        activation: str = "none") -> None:
    """out = act((x - mean) / sqrt(var + eps) * weight + bias), biased variance.

    graph_ptr: int32 or int64 [num_graphs + 1] ascending row offsets; rows before the
    first and behind the last are left as they are in out. activation: none, relu,
    silu or gelu (erf). weight / bias: [channels] or None. out may be x itself."""
    dev = out.device
    _check_f32("out", out, 2, dev)
    _check_f32("x", x, 2, dev)
    _check(tuple(x.shape) == tuple(out.shape), "x and out must have the same shape")
    n, c = x.size(0), x.size(1)
    groups = int(groups)
    _check(groups >= 1 and c % groups == 0, "groups must be >= 1 and divide the number of channels")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_f32(name, t, 1, dev)
            _check(t.numel() == c, f"{name} length must equal the number of channels")
    _check(activation in ACTIVATIONS, "activation must be none, relu, silu or gelu")
    _check(float(eps) >= 0.0, "eps must be >= 0")
    _check(x.data_ptr() == out.data_ptr() or not _overlap(out, x), "out must be x itself or not overlap it")
    ptr, ptr_type, graphs = None, N.GNN_INDEX_INT32, 0
    if graph_ptr is not None:
        _on_device("graph_ptr", graph_ptr, dev)
        _check(graph_ptr.dtype in (torch.int32, torch.int64), "graph_ptr must be int32 or int64")
        _check(graph_ptr.dim() == 1 and graph_ptr.is_contiguous(), "graph_ptr must be rank-1 and contiguous")
        _check(graph_ptr.numel() >= 1, "graph_ptr must hold num_graphs + 1 offsets")
        ptr, ptr_type, graphs = graph_ptr.data_ptr(), _index_type(graph_ptr), graph_ptr.numel() - 1
    L = N.lib()
    with _Device(dev):
        wsb = L.gnn_group_norm_workspace_bytes(n, graphs, groups) if ptr is not None else 0
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        N.check(L.gnn_group_norm_forward(
            x.data_ptr(), ptr, ptr_type, graphs, None if weight is None else weight.data_ptr(),
            None if bias is None else bias.data_ptr(), out.data_ptr(), n, c, groups, float(eps), ACTIVATIONS[activation],
            None if ws is None else ws.data_ptr(), wsb, _stream(dev)), "gnn_group_norm_forward")
