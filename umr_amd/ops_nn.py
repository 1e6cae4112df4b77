"""The network-side operators as registered PyTorch operators: loads libumr_torch.so (csrc/torch_nn.cpp), which defines
torch.ops.umr.linear_act, torch.ops.umr.balance_loss and their backward operators with device and meta kernels and their autograd.
umr_amd.functional's linear_act / heads_linear_act / balance_loss are the calls a user makes."""
import ctypes
import os

import torch

from . import _lib

LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libumr_torch.so")
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "tanh": 3, "gelu": 4, "silu": 5}      # UMR_ACT_* (include/umr_nn.h)
MAX_CHOICES = 1024                                                                          # UMR_BALANCE_MAX_CHOICES

if not os.path.exists(LIB_PATH):
    raise RuntimeError("umr_amd: %s is missing -- build it with `python -m umr_amd.build`. There is no CPU fallback." % LIB_PATH)
torch.ops.load_library(LIB_PATH)


def build_id():
    """Hash of the sources libumr_torch.so was compiled from (umr_amd.build.source_hash)."""
    fn = ctypes.CDLL(LIB_PATH).umr_torch_build_id
    fn.restype = ctypes.c_char_p
    return fn().decode()
