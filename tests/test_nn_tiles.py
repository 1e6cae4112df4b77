"""CPU tests of the tiled products (csrc/linear_kernels.h) on the wave64 emulator, tile by tile at sizes that the plan would give to a
smaller one: overlap in both directions, a contraction of several steps with a cut last one, rows far apart in memory."""
import pytest
import torch

import host_nn as H
import nn_checks as C
import nn_tiles as R

TYPES = [torch.float32, torch.bfloat16, torch.float16]
pytestmark = pytest.mark.skipif(not H.available(), reason="clang++ of the ROCm toolchain not present")
TILES = [(t, d) for d in TYPES for t in (64, 128, 256) if t <= R.widest(d)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", R.WIDE, ids=str)
def test_the_plan_takes_the_widest_tiles_where_they_are_tested(shape, dtype):
    assert R.route(R.lib(), *shape, dtype) == (R.widest(dtype), 1)


@pytest.mark.parametrize("tile,dtype", TILES, ids=str)
@pytest.mark.parametrize("direction", list(R.KIND))
def test_every_tile_against_64_bits(direction, tile, dtype):
    """three steps of the contraction and a cut one; for the smaller tiles also matrices smaller than a tile"""
    L = R.lib()
    a, b, c = (tile + 37, tile + 9, 3 * (32 if dtype == torch.float32 else 64) + 13)
    for G, a, b, c in [(2, a, b, c)] + ([(1, 5, 70, 3), (1, tile + 1, 3, c)] if tile < 256 else []):
        M, N, K = {"forward": (a, b, c), "input": (a, c, b), "weight": (c, a, b)}[direction]
        x, w, bias, r, gy = C.inputs(M, G, N, K, dtype, "cpu", pad=3)
        if direction == "forward":
            y, z = R.run_tile(L, direction, tile, x, w, None, bias, r, "gelu", want_z=True)
            z64, mag = C.product("mgk,gnk->mgn", x, w)
            z64, mag = z64 + bias.double(), mag + bias.double().abs()
            ztol = (K + 2) * C.U * mag
            C.close(z, z64, ztol, "z")
            y64 = C.act64(z64, "gelu", 0.0) + r.double()
            C.close(y, y64, 1.13 * ztol + 16 * C.U * (z64.abs() + 1) + C.U * (y64.abs() + r.double().abs()), "y")
        elif direction == "input":
            want, mag = C.product("mgn,gnk->mgk", gy, w)
            C.close(R.run_tile(L, direction, tile, None, w, gy)[0], want, (N + 2) * C.U * mag, "dx")
        else:
            want, mag = C.product("mgn,mgk->gnk", gy, x)
            C.close(R.run_tile(L, direction, tile, x, None, gy)[0], want, (M + 2) * C.U * mag, "dw")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_far_apart_take_another_path_to_the_same_bits(dtype):
    """rows of 2^22 elements in memory: the widest 16-bit tile hands over to the next one, the others load by 64-bit offsets; a 128 tile of
    the same rows side by side gives the bits"""
    L = R.lib()
    M, N, K = 259, 258, 70
    gen = torch.Generator().manual_seed(0)
    far = torch.empty(M, (1 << 22) + 1, dtype=dtype)                         # (pages that are never touched take no memory)
    near = torch.randn(M, 1, K, generator=gen).to(dtype)
    x = far[:, None, 3:3 + K]
    x.copy_(near)
    w, gy = torch.randn(1, N, K, generator=gen).to(dtype), torch.randn(M, 1, N, generator=gen).to(dtype)
    for tile in (64, 128, 256) if dtype != torch.float32 else (64, 128):
        assert torch.equal(R.run_tile(L, "forward", tile, x, w, None)[0], R.run_tile(L, "forward", 128, near, w, None)[0])
        assert torch.equal(R.run_tile(L, "weight", tile, x, None, gy)[0], R.run_tile(L, "weight", 128, near, None, gy)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("direction", list(R.KIND))
def test_more_heads_than_a_launch_holds(direction, dtype):
    """a launch's threads are counted in 32 bits, so many heads take several launches (here: of 2 and of 3 heads of 2 x 1 tiles, then of all);
    a head alone that is more than a launch is refused"""
    L = R.lib()
    M, G, N, K = {"forward": (70, 7, 20, 9), "input": (70, 7, 9, 20), "weight": (9, 7, 70, 20)}[direction]
    x, w, bias, r, gy = C.inputs(M, G, N, K, dtype, "cpu", pad=1)
    args = {"forward": (x, w, None, bias, r), "input": (None, w, gy), "weight": (x, None, gy)}[direction]
    for act in (("relu", "gelu") if direction == "forward" else ("none",)):
        kw = dict(act=act, want_z=direction == "forward")
        want = R.run_tile(L, direction, 64, *args, **kw)
        for most in (4, 7, 1000):
            got = R.run_tile(L, direction, 64, *args, most=most, **kw)
            assert torch.equal(got[0], want[0]) and (want[1] is None or torch.equal(got[1], want[1]))
        assert R.run_tile(L, direction, 64, *args, most=1, **kw) == -1
