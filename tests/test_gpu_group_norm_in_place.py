"""Group norm written over its input: the bits of a call with an output of its own (run
with -m gpu)."""
import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import norm_ops as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _check(x, groups, ptr, activation="silu"):
    w, b = torch.rand(x.shape[1], device=DEV) + 0.5, torch.randn(x.shape[1], device=DEV)
    want = x.clone()  # rows of no graph stay as they are
    M.group_norm_forward_(x, groups, w, b, want, graph_ptr=ptr, activation=activation)
    M.group_norm_forward_(x, groups, w, b, x, graph_ptr=ptr, activation=activation)
    assert torch.equal(x, want)


@pytest.mark.parametrize("c,groups", [(36, 4), (64, 4), (100, 10), (256, 1), (999, 27)])
@pytest.mark.parametrize("low,high,graphs", [(1, 64, 2000), (1, 300, 2000), (65, 200, 2000), (1, 3000, 60)])
def test_batches(c, groups, low, high, graphs):
    """Short graphs that run on into the next window, whole ones read a second time, split ones."""
    lengths = torch.randint(low, high + 1, (graphs,), device=DEV)
    ptr = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]) + 3
    _check(torch.randn(int(ptr[-1]) + 70, c, device=DEV), groups, ptr)


@pytest.mark.parametrize("n,c,groups", [(50_001, 27, 3), (30_000, 32, 32), (7_000, 300, 100), (20_000, 256, 16),
                                        (9, 5, 1)])
def test_nodes(n, c, groups):
    _check(torch.randn(n, c, device=DEV), groups, None)
