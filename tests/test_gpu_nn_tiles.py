"""GPU tests of the widest tiles of the network-side products (csrc/linear_kernels.h): shapes whose plan takes them, asserted by
tests/test_nn_tiles.py on the host."""
import pytest
import torch

import nn_checks as C
import nn_tiles as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _lib():
    from umr_amd import _lib
    return _lib.lib()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", R.WIDE, ids=str)
def test_widest_tiles_against_64_bits(shape, dtype):
    direction, M, G, N, K = shape
    act = "gelu" if direction == "forward" else "none"
    C.check_linear(_lib(), M, G, N, K, dtype, act, device=DEV, pad=1, parts=(direction,))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_widest_tiles_hand_over_rows_that_lie_far_apart(dtype):
    """rows of 2^22 elements in memory: the same product through the next smaller tile; x far, then the weight"""
    from umr_amd import functional as UF
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(4000, 523, device=DEV, generator=g).to(dtype)
    w = torch.randn(4090, 523, device=DEV, generator=g).to(dtype)
    far = torch.empty(4090, 1 << 22, device=DEV, dtype=dtype)
    tol = (523 + 2) * C.U * (x.double().abs() @ w.double().abs().t())
    want = x.double() @ w.double().t()
    fx, fw = far[:4000, 7:530], far[:, 1000:1523]
    fx.copy_(x)
    C.close(UF.linear_act(fx, w), want, tol, "far rows of x")
    fw.copy_(w)
    C.close(UF.linear_act(x, fw), want, tol, "far rows of the weight")


def test_more_heads_than_a_launch_holds():
    """65535 heads of 257 tiles, 2^32 threads and more: forward with z, dx and dw of some heads against the same heads alone, in 64 bits"""
    from umr_amd import functional as UF
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 160 GB")
    M, G, N, K = 16448, 65535, 8, 8
    t, U, e = torch.bfloat16, C.U, C.half_step(torch.bfloat16)
    torch.manual_seed(6)
    x = torch.empty(M, G, K, device=DEV, dtype=t).normal_().requires_grad_(True)
    w = torch.empty(G, N, K, device=DEV, dtype=t).normal_().requires_grad_(True)
    y = UF.heads_linear_act(x, w, activation="silu")
    gy = torch.empty(M, G, N, device=DEV, dtype=t).normal_()
    dx, dw = torch.autograd.grad(y, [x, w], gy)
    for g in (0, 1, 32767, 65279, 65280, G - 2, G - 1):
        xg, wg, gg = (v.detach().double() for v in (x[:, g], w[g], gy[:, g]))
        z, zmag = xg @ wg.t(), xg.abs() @ wg.abs().t()
        ztol = (K + 2) * U * zmag
        C.close(y[:, g].detach(), C.act64(z, "silu", 0.0), 1.13 * ztol + 16 * U * (z.abs() + 1), "y")
        dz = gg * C.act_slope64(z, "silu", 0.0)
        dtol = gg.abs() * (0.8 * ztol + 32 * U * (z.abs() + 1)) + e * dz.abs()
        mag = dz.abs() + dtol
        C.close(dx[:, g], dz @ wg, (dtol + (N + 2) * U * mag) @ wg.abs(), "dx")
        C.close(dw[g], dz.t() @ xg, (dtol + (M + 2) * U * mag).t() @ xg.abs(), "dw")
