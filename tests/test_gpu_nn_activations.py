"""GPU tests of the activations' values and derivatives where they are tiny, and at NaN."""
import pytest
import torch

import host_nn as H
import nn_activation_checks as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _lib():
    from umr_amd import _lib
    return _lib.lib()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ["gelu", "tanh", "silu"])
def test_tails_keep_their_digits(act, dtype):
    A.check_tails(_lib(), act, dtype, device=DEV)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", [a for a in H.ACT if a != "none"])
def test_derivatives_let_nan_through_as_torch_does(act, dtype):
    F = torch.nn.functional
    z = torch.tensor([1.0, float("nan"), -2.0, 0.0], dtype=dtype)
    y, slope = A.run(_lib(), act, z.float(), dtype, DEV, slope=0.25)
    leaf = z.float().requires_grad_(True)
    ref = {"relu": F.relu, "leaky_relu": lambda v: F.leaky_relu(v, 0.25), "tanh": torch.tanh, "gelu": F.gelu, "silu": F.silu}[act](leaf)
    want, = torch.autograd.grad(ref, leaf, torch.ones(4))
    assert torch.equal(slope.cpu().isnan(), want.isnan()) and bool(y[1].isnan()) and int(y.isnan().sum()) == 1
    assert float((slope.cpu().float() - want).nan_to_num().abs().max()) <= torch.finfo(dtype).eps
