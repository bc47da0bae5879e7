"""Calls of the 8-bit quantiser that are refused before anything runs (run with -m gpu)."""
import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import int8_ops as I

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_quantising_into_the_input():
    """Rows would be overwritten while others are still to be read."""
    x = torch.randn(50, 32, device=DEV)
    kept = x.clone()
    inside = x.view(torch.int8)
    with pytest.raises(RuntimeError, match="q must not alias x"):
        I.quantize_rows_(x, inside[:, :32], torch.empty(50, device=DEV))
    with pytest.raises(RuntimeError, match="q must not alias x"):
        I.quantize_rows_(x[:25], inside[20:45, 64:96], torch.empty(25, device=DEV))
    with pytest.raises(RuntimeError, match="q must not alias weight"):
        I.quantize_weight_(x, inside[:32, :50], torch.empty(32, device=DEV))
    assert torch.equal(x, kept)
    # beside it is fine
    q, s = inside[25:, :32], torch.empty(25, device=DEV)
    I.quantize_rows_(x[:25], q, s)
    assert torch.equal(x[:25], kept[:25])
    want, ws = I.empty_rows(25, 32, DEV), torch.empty(25, device=DEV)
    I.quantize_rows_(kept[:25], want, ws)
    assert torch.equal(q, want) and torch.equal(s, ws)
