"""Refusals of the group normalisation that need no device."""
import pytest
import torch

from gnn_cuda_b200 import _native as N
from gnn_cuda_b200.GNN_cuda_common import norm_ops as M


def test_c_refusals():
    L = N.lib()
    p = 1 << 20
    call = lambda n=200, c=8, g=2, eps=1e-5, act=0, x=p, ptr=None, ty=0, graphs=1, ws=None, wsb=0: L.gnn_group_norm_forward(  # noqa: E731
        x, ptr, ty, graphs, None, None, p, n, c, g, eps, act, ws, wsb, None)
    assert call(n=-1) == 1 and call(g=0) == 1 and call(g=3) == 1
    assert "divide" in N.last_error()
    assert call(act=4) == 1 and call(act=-1) == 1 and call(eps=-1.0) == 1 and call(eps=float("nan")) == 1
    assert call(ptr=p, ty=7) == 1
    assert call(c=1025, g=1) == 3 and "1024" in N.last_error()
    assert call(x=None) == 2
    assert call(ptr=p) == 7
    assert call(n=0) == 0 and call(c=0) == 0 and call(ptr=p, graphs=0) == 0
    assert L.gnn_group_norm_workspace_bytes(64, 1, 8) == 0
    assert L.gnn_group_norm_workspace_bytes(65, 1, 8) > 0


def test_python_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="out must be CUDA"):
        M.group_norm_forward_(x, 2, None, None, torch.zeros(4, 8))
