"""Checks of the network-side operators against their definition in 64 bits, shared by tests/test_nn_operators.py (the kernels on the
wave64 emulator) and tests/test_gpu_nn_operators.py.

Tolerances, element by element.  u = 2^-24 is half a step of fp32, e = finfo(type).eps / 2 half a step of the type.
  * a sum of n products in fp32, in any order, fused or not, is off by at most (n + 2) u times the sum of the magnitudes (each term
    passes through at most n + 1 roundings; products of 16-bit values are exact)
  * one rounding to the type adds e |value| (and the type's smallest step where it underflows)
  * act has |act'| <= 1.13 (gelu 1.129, silu 1.0998, the others <= 1), so an error of z reaches y at most 1.13 times as large; its own
    evaluation (erff, expf, tanhf, a division: 1 - 4 steps each, on values of at most |z| + 1) is given 16 u (|z| + 1)
  * act' = a sum of at most two products of such values, |act''| <= 0.8: 32 u (|z| + 1)"""
import torch

import host_nn as H

U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol, what):
    """got: the operator's output; want and tol in float64.  Adds the output's own rounding."""
    t = got.dtype
    bound = tol + half_step(t) * (want.abs() + tol) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), "%s: %d of %d elements off, worst %.3g (allowed there %.3g)" % (
        what, int(bad.sum()), bad.numel(), float((got.double() - want).abs()[bad].max()), float(bound[bad].max()))


def act64(z, act, slope):
    F = torch.nn.functional
    return {"none": lambda v: v, "relu": F.relu, "leaky_relu": lambda v: F.leaky_relu(v, slope), "tanh": torch.tanh, "gelu": F.gelu,
            "silu": F.silu}[act](z)


def act_slope64(z, act, slope):
    if act in ("relu", "leaky_relu"):
        return torch.where(z > 0, 1.0, 0.0 if act == "relu" else slope)
    v = z.clone().requires_grad_(True)
    return torch.autograd.grad(act64(v, act, slope).sum(), v)[0]


def product(eq, a, b):
    """einsum in float64 and the same of the magnitudes"""
    a, b = a.double(), b.double()
    return torch.einsum(eq, a, b), torch.einsum(eq, a.abs(), b.abs())


def inputs(M, G, N, K, dtype, device, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + M + 7 * N + 13 * K + G)
    rnd = lambda *s: torch.randn(*s, generator=g)
    x = H.Guarded((M, G, K), dtype, device, pad)
    w = H.Guarded((G, N, K), dtype, device, pad)
    r = H.Guarded((M, G, N), dtype, device, pad)
    gy = H.Guarded((M, G, N), dtype, device, pad)
    for t, v in ((x, rnd(M, G, K)), (w, rnd(G, N, K)), (r, rnd(M, G, N)), (gy, rnd(M, G, N))):
        t.t.copy_(v)
    return x.t, w.t, rnd(G, N).to(device=device, dtype=dtype), r.t, gy.t


def check_linear(L, M, G, N, K, dtype, act, device="cpu", pad=0, bias=True, residual=True, stream=None, parts=("forward", "act", "input", "weight")):
    """Every entry point on one shape; what lies between and around the rows is NaN and stays as it was."""
    x, w, b, r, gy = inputs(M, G, N, K, dtype, device, pad)
    slope = 0.2 if act == "leaky_relu" else 0.0
    if not bias:
        b = None
    if not residual:
        r = None
    z64, mag = product("mgk,gnk->mgn", x, w)
    if b is not None:
        z64, mag = z64 + b.double(), mag + b.double().abs()
    ztol = (K + 2) * U * mag
    zk = z64
    if "forward" in parts:
        y, z = H.linear_forward(L, x, w, b, r, act, slope, True, stream)
        close(z, z64, ztol, "z")
        ytol = 1.13 * ztol + 16 * U * (z64.abs() + 1)
        y64 = act64(z64, act, slope)
        if r is not None:
            y64, ytol = y64 + r.double(), ytol + U * (y64.abs() + r.double().abs())
        close(y, y64, ytol, "y")
        y2, none = H.linear_forward(L, x, w, b, r, act, slope, False, stream)
        assert none is None and torch.equal(y, y2)                       # z asked for or not, run after run: the same bits
        zk = z
    dz = gy
    if "act" in parts:
        zk = (zk if zk.dtype != torch.float64 else zk.to(dtype if act in ("relu", "leaky_relu") else torch.float32)).contiguous()
        got, db, dr = H.linear_grad_act(L, gy, None if act == "none" else zk, act, slope, stream=stream)
        g64 = gy.double()
        d64 = g64 * act_slope64(zk.double(), act, slope)
        dtol = 32 * U * g64.abs() * (zk.double().abs() + 1) if act != "none" else torch.zeros_like(g64)
        if act == "none":
            assert got is None
        else:
            close(got, d64, dtol, "dz")
            dz = got
        close(db, d64.sum(0), (M + 2) * U * d64.abs().sum(0) + dtol.sum(0), "db")
        close(dr, g64.sum(0), (M + 2) * U * g64.abs().sum(0), "dr")
    if "input" in parts:
        want, mag = product("mgn,gnk->mgk", dz, w)
        close(H.linear_grad_input(L, dz, w, stream), want, (N + 2) * U * mag, "dx")
    if "weight" in parts:
        want, mag = product("mgn,mgk->gnk", dz, x)
        close(H.linear_grad_weight(L, dz, x, stream), want, (M + 2) * U * mag, "dw")


def balance64(z, inds, mask):
    """loss (None without a valid row), counts, d loss / d z, and p of every row, from the definition"""
    E, k = z.shape[1], inds.shape[1]
    keep = ~(z == -float("inf")).all(1)
    if mask is not None:
        keep = keep & mask
    chosen = inds[keep].reshape(-1)
    counts = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
    leaf = z[keep].double().requires_grad_(True)
    dz = torch.zeros(z.shape, dtype=torch.float64, device=z.device)
    p = torch.zeros_like(dz)
    if not bool(keep.any()):
        return torch.zeros((), dtype=torch.float64, device=z.device), counts, dz, p
    soft = torch.softmax(leaf, 1)
    loss = E * torch.dot(counts.double() / (int(keep.sum()) * k), soft.mean(0))
    dz[keep] = torch.autograd.grad(loss, leaf)[0]
    p[keep] = soft.detach()
    return loss.detach(), counts, dz, p


def balance_inputs(T, E, k, dtype, device, mask, seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + T + 31 * E + k)
    z = (2 * torch.randn(T, E, generator=g)).to(dtype)
    inds = torch.randint(0, E, (T, k), generator=g)
    m = None
    if mask in ("choices", "both") and T:
        z[torch.rand(T, E, generator=g) < 0.15] = -float("inf")
        z[torch.rand(T, generator=g) < 0.1] = -float("inf")
        z[torch.rand(T, generator=g) < 0.05] = torch.finfo(dtype).min
        inds[torch.rand(T, k, generator=g) < 0.1] = -1
        inds[torch.rand(T, k, generator=g) < 0.05] = E
    if mask in ("rows", "both"):
        m = torch.rand(T, generator=g) < 0.8
        z[~m] = float("nan")
    if mask == "nothing":
        m = torch.zeros(T, dtype=torch.bool)
    return z.to(device), inds.to(device), (None if m is None else m.to(device))


def check_balance(L, T, E, k, dtype, mask, device="cpu", stream=None):
    """p is off by at most (E + 8 + |z - max| of what counts) u of itself: 40 + E steps cover |z - max| <= 32 (beyond it p is below
    e^-32 of the largest); the sum over T rows adds T + 2 steps.  The gradient is scale p (f - sum f p), off by the steps of p and E + 8
    of the bracket's magnitudes max |f - mean| <= max f."""
    z, inds, m = balance_inputs(T, E, k, dtype, device, mask)
    loss, counts, coef = H.balance_forward(L, z, inds, m, stream)
    want, c64, d64, p = balance64(z, inds, m)
    assert torch.equal(counts, c64)
    close(loss, want.reshape(1), ((T + E + 48) * U * want.abs()).reshape(1), "loss")
    again = H.balance_forward(L, z, inds, m, stream)
    assert torch.equal(loss, again[0]) and torch.equal(coef, again[2])
    up = 64.0
    dz = H.balance_backward(L, z, m, coef, torch.tensor([up], device=device), stream)
    valid = p.sum(1) > 0
    n = max(int(valid.sum()), 1)
    f = c64.double() / (n * k)
    spread = (f - f.mean()).abs().max()
    close(dz, up * d64, up * (E / n) * p * spread * (2 * E + 96) * U, "dz")
    assert bool((dz[~valid] == 0).all())
