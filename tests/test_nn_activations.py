"""CPU tests of the activations' values and derivatives where they are tiny, and at NaN (csrc/linear_kernels.h on the wave64 emulator)."""
import pytest
import torch

import host_nn as H
import nn_activation_checks as A

TYPES = [torch.float32, torch.bfloat16, torch.float16]
pytestmark = pytest.mark.skipif(not H.available(), reason="clang++ of the ROCm toolchain not present")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gelu_keeps_its_digits_in_the_negative_tail(dtype):
    A.check_tails(H.lib(), "gelu", dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ["tanh", "silu"])
def test_tanh_and_silu_keep_their_digits_where_they_saturate(act, dtype):
    A.check_tails(H.lib(), act, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", list(H.ACT))
def test_derivatives_let_nan_through_as_torch_does(act, dtype):
    """a NaN pre-activation: the gradient is what torch's own function passes on (relu: the incoming gradient, leaky relu: the slope's
    share, the smooth ones: NaN); infinities beside it: no other element changes"""
    if act == "none":
        return
    F = torch.nn.functional
    z = torch.tensor([1.0, float("nan"), -2.0, 0.0], dtype=dtype)
    y, slope = A.run(H.lib(), act, z.float(), dtype, "cpu", slope=0.25)
    leaf = z.float().requires_grad_(True)
    ref = {"relu": F.relu, "leaky_relu": lambda v: F.leaky_relu(v, 0.25), "tanh": torch.tanh, "gelu": F.gelu, "silu": F.silu}[act](leaf)
    want, = torch.autograd.grad(ref, leaf, torch.ones(4))
    assert torch.equal(slope.isnan(), want.isnan()) and bool(y[1].isnan()) and int(y.isnan().sum()) == 1
    tol = torch.finfo(dtype).eps
    assert float((slope.float() - want).nan_to_num().abs().max()) <= tol
