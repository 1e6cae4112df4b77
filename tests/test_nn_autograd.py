"""CPU tests of what surrounds the network-side operators in PyTorch (csrc/torch_nn.cpp), on tensors without a device."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from umr_amd import functional as UF


def _m(*s, dtype=torch.float32, grad=False):
    return torch.empty(*s, dtype=dtype, device="meta", requires_grad=grad)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual", "scores"])
def test_forward_mode_is_refused_and_not_dropped(which, grad):
    """a tangent that reaches an operator raises, with and without requires_grad and inside torch.func.jvp"""
    if which == "scores":
        given = dict(scores=_m(5, 3, grad=grad))
        call = lambda t: UF.balance_loss(t["scores"], _m(5, 1, dtype=torch.int64))[0]
    else:
        given = dict(x=_m(5, 3, grad=grad), weight=_m(4, 3, grad=grad), bias=_m(4, grad=grad), residual=_m(5, 4, grad=grad))
        call = lambda t: UF.linear_act(t["x"], t["weight"], t["bias"], residual=t["residual"], activation="tanh")
    with fwAD.dual_level():
        dual = dict(given, **{which: fwAD.make_dual(given[which], torch.ones_like(given[which]))})
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            call(dual)
        call(given)                                                          # no tangent among its inputs: as everywhere
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: call(dict(given, **{which: v})), (given[which].detach(),), (torch.ones_like(given[which].detach()),))


@pytest.mark.parametrize("which", ["linear", "balance"])
def test_forward_mode_over_a_gradient_is_refused(which):
    x, w, z = _m(5, 3, grad=True), _m(4, 3), _m(5, 3, grad=True)
    leaf, out = (x, UF.linear_act(x, w, activation="tanh")) if which == "linear" else (z, UF.balance_loss(z, _m(5, 1, dtype=torch.int64))[0])
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(out, leaf, fwAD.make_dual(torch.ones_like(out).detach(), torch.ones_like(out).detach()))


def test_autocast_is_registered_for_the_layer():
    """(what it does: tests/test_gpu_nn_layers.py)"""
    UF._nn_ops()
    assert torch._C._dispatch_has_kernel_for_dispatch_key("umr::linear_act", "AutocastCUDA")
