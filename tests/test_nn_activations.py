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
