"""GPU tests of MeshNet's layers on the network-side operators, and of those operators inside PyTorch."""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_layers_under_autocast(dtype):
    """the calls of a fused net under torch.autocast are the calls with every tensor cast; gradients come back in the leaves' types; float64 is
    refused inside as outside"""
    from umr_amd import functional as UF, model as M
    torch.manual_seed(0)
    net = M.fuse_linears(nn.Sequential(nn.Linear(40, 50), nn.LeakyReLU(0.2), nn.Linear(50, 30))).to(DEV)
    x = torch.randn(20, 40, device=DEV, requires_grad=True)
    w = torch.randn(3, 30, 10, device=DEV, requires_grad=True)
    r = torch.randn(20, 3, 30, device=DEV, dtype=dtype)
    leaves = [x, w] + list(net.parameters())
    with torch.autocast("cuda", dtype=dtype):
        h = net(x)
        y = UF.heads_linear_act(h[:, None, :10].expand(20, 3, 10), w, residual=r, activation="silu")
    c = lambda t: t.to(dtype)
    h2 = UF.linear_act(UF.linear_act(c(x), c(net[0].weight), c(net[0].bias), activation="leaky_relu", slope=0.2), c(net[2].weight), c(net[2].bias))
    y2 = UF.heads_linear_act(h2[:, None, :10].expand(20, 3, 10), c(w), residual=r, activation="silu")
    assert h.dtype == y.dtype == dtype and torch.equal(h, h2) and torch.equal(y, y2)
    g = torch.randn_like(y)
    for a, b, leaf in zip(torch.autograd.grad(y, leaves, g), torch.autograd.grad(y2, leaves, g), leaves):
        assert a.dtype == leaf.dtype and torch.equal(a, b)
    for cast in (False, True):
        with torch.autocast("cuda", dtype=dtype, enabled=cast), pytest.raises(RuntimeError, match="float32, bfloat16|weight is"):
            UF.linear_act(x.double(), net[0].weight.double())


def test_fused_net_with_an_activation_that_is_changed_in_place():
    from umr_amd import model as M
    torch.manual_seed(1)
    net = nn.Sequential(nn.Linear(5, 6), nn.LeakyReLU(0.2), nn.ReLU(inplace=True)).to(DEV)
    x = torch.randn(7, 5, device=DEV)
    want = net(x)
    M.fuse_linears(net)
    y = net(x)
    # sums of 5 products and a bias, and two roundings: at most 9 u of their magnitudes on either side
    mag = x.abs() @ net[0].weight.detach().abs().t() + net[0].bias.detach().abs()
    assert bool(((y - want).detach().abs() <= 2 * 9 * 2.0 ** -24 * mag).all())
    y.square().sum().backward()
    assert bool(torch.isfinite(net[0].weight.grad).all()) and float(net[0].weight.grad.abs().sum()) > 0
