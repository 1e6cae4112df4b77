"""The activations and their derivatives by themselves, shared by the CPU and the GPU tests: a layer without inputs (K = 0), whose
pre-activations are its biases, and the act' pass on the same numbers.  Errors are bounded relative to the value (to its parts, where two
of them cancel), also where the value is tiny.  u = 2^-24; nn_checks.close adds the rounding to the type."""
import math

import torch

import host_nn as H
import nn_checks as C

# 16-bit kernels: the fit of the normal distribution's tail is off by 1e-5 of it at most (its own 7e-6, and fp32 evaluation)
TAIL = 1e-5


def values(act, z, slope=0.0):
    """(act(z), act'(z), the magnitudes that act' is the sum of) in float64; z float64 on the CPU"""
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        pdf = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, cdf + z.abs() * pdf
    if act == "tanh":
        e = torch.exp(-2 * z.abs())
        return torch.tanh(z), 4 * e / (1 + e) ** 2, 4 * e / (1 + e) ** 2
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * torch.sigmoid(-z)), s * (1 + z.abs() * torch.sigmoid(-z))


def run(L, act, z, dtype, device, slope=0.0, stream=None):
    """(y, act'(z) through gy = 1) of the library for the numbers z (float32)"""
    n = z.numel()
    b = z.to(device=device, dtype=dtype).reshape(1, n)
    x, w = torch.zeros(1, 1, 0, device=device, dtype=dtype), torch.zeros(1, n, 0, device=device, dtype=dtype)
    y, kept = H.linear_forward(L, x, w, b, None, act, slope, True, stream)
    dz, _, _ = H.linear_grad_act(L, torch.ones(1, 1, n, device=device, dtype=dtype), kept.contiguous(), act, slope, stream=stream)
    return y.flatten(), dz.flatten()


def check_tails(L, act, dtype, device="cpu", stream=None):
    """|z| up to 12: Phi(-12) = 2e-33.  An argument that is off by u of itself moves exp(-z^2 / 2) and erfc(|z| / sqrt 2) by up to z^2 u of
    themselves (two such roundings), exp(-2 |z|) and exp(-z) by 2 |z| u; 16 u for the functions and products"""
    z = torch.cat([torch.linspace(-12, 12, 4097), torch.linspace(-1e-3, 1e-3, 65)]).to(dtype).float()
    y, slope = run(L, act, z, dtype, device, stream=stream)
    z64 = z.double()
    want, dwant, dmag = values(act, z64)
    rel = (16 + (2 * z64 * z64 if act == "gelu" else 4 * z64.abs())) * C.U
    if act == "gelu" and dtype != torch.float32:
        rel = rel + TAIL
    C.close(slope.cpu(), dwant, rel * dmag, act + "'")
    C.close(y.cpu(), want, rel * want.abs(), act)
