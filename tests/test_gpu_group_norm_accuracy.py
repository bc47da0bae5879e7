"""How exact the group norm is where a coarse step would show (run with -m gpu).

u = 2^-24 throughout; references in 64 bits.
"""
import pytest
import torch

from gnn_cuda_b200.GNN_cuda_common import norm_ops as M

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
EPS = 1e-5


def _activated(y, act):
    """act(y): weight 0 leaves the bias as the activation's argument."""
    c = y.numel()
    x = torch.randn(3, c, device=DEV)
    out = torch.empty_like(x)
    M.group_norm_forward_(x, c // 64, torch.zeros(c, device=DEV), y, out, activation=act)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    return out[0].double()


def test_gelu_relative_error():
    """y Phi(y) = max(y, 0) - z Phi(-z), z = |y|. The fit of Phi(-z) exp(z^2 / 2) is off by 1.4e-7 of itself; its two
    polynomials, their quotient, the exponential (two units) and the products are below 20 roundings; the exponent
    z^2 / 2 carries three. For y > 0 two more roundings of the result come on top, and Phi(-z) is below it."""
    y = torch.linspace(-8, 8, 4096, device=DEV)
    d = y.double()
    want = d * 0.5 * torch.special.erfc(-d / 2 ** 0.5)
    rel = 1.4e-7 + (20 + 1.5 * d * d) * U
    tail = d.abs() * 0.5 * torch.special.erfc(d.abs() / 2 ** 0.5)
    bound = rel * tail + torch.where(d > 0, 2 * U * want, torch.zeros_like(d))
    assert bool(((_activated(y, "gelu") - want).abs() <= bound).all())


def test_gelu_special_values():
    inf = float("inf")
    y = torch.tensor([0.0, -0.0, 30.0, -30.0, inf, float("nan"), 1e30, -1e30] * 64, device=DEV)
    got = torch.empty(2, y.numel(), device=DEV)
    M.group_norm_forward_(torch.randn(2, y.numel(), device=DEV), 8, torch.zeros(y.numel(), device=DEV), y, got,
                          activation="gelu")
    row = got[0, :8].tolist()
    assert row[0] == 0 and row[1] == 0 and row[2] == 30 and row[3] == 0 and row[4] == inf
    assert row[5] != row[5] and row[6] == torch.tensor(1e30).item() and row[7] == 0


def test_silu_relative_error():
    """The exponential's argument, |y| log2 e, is rounded twice; two units each for it and the quotient, two sums."""
    y = torch.linspace(-80, 40, 4096, device=DEV)
    d = y.double()
    want = d / (1 + torch.exp(-d))
    assert bool(((_activated(y, "silu") - want).abs() <= (2 * d.abs() + 12) * U * want.abs()).all())


# narrow nodes (few channels), then a warp per row: pieces of 16, 8 and 4 bytes, one and several column tiles
@pytest.mark.parametrize("c,groups", [(16, 8), (27, 9), (12, 3), (63, 21), (192, 96), (300, 100), (256, 64), (512, 128),
                                      (1024, 512), (262, 131), (1050, 350), (201, 67), (2050, 1025), (4100, 1025)])
def test_groups_of_few_near_values(c, groups):
    """Values 3 + 0.001 t: differences from the group's first value are exact (they are within a factor of two), so
    every step is rounded in proportion to their largest, D: cg sums, a product, two subtractions."""
    n = 3000
    x = 3 + 1e-3 * torch.randn(n, c, device=DEV)
    out = torch.empty_like(x)
    M.group_norm_forward_(x, groups, None, None, out)
    v = x.double().view(n, groups, -1)
    cg = c // groups
    d = v - v.mean(2, keepdim=True)
    sd = (d.square().mean(2, keepdim=True) + EPS).sqrt()
    z = d / sd
    big = (v - v[:, :, :1]).abs().amax(2, keepdim=True)
    bound = (cg + 6) * U * big / sd * (1 + z.abs()) + 12 * U * z.abs()
    assert bool(((out.double().view(n, groups, -1) - z).abs() <= bound).all())


@pytest.mark.parametrize("c,groups", [(32, 8), (100, 25), (128, 16), (64, 16)])
def test_equal_values_far_from_zero(c, groups):
    """Graphs whose features are equal within a group, whole numbers up to 4,095: with counts that are powers of two
    every sum is exact, so the deviation is 0 and the output is the bias, in graphs short and long, whole and split."""
    lengths = torch.tensor([1, 2, 4, 8, 16, 32, 64] * 40 + [128, 256, 1024, 4096] + [1] * 30, device=DEV)
    ptr = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    per = torch.randint(1000, 4096, (len(lengths), groups), device=DEV).float()
    x = per.repeat_interleave(lengths, 0).repeat_interleave(c // groups, 1)
    w, b = torch.rand(c, device=DEV) + 0.5, torch.randn(c, device=DEV)
    out = torch.empty_like(x)
    M.group_norm_forward_(x, groups, w, b, out, graph_ptr=ptr)
    assert torch.equal(out, b.expand_as(out))
