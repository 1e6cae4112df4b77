"""TEST INFRASTRUCTURE: the products whose plan takes the widest tiles (tests/test_gpu_nn_tiles.py runs them, tests/test_nn_tiles.py asserts
the plan), and host_kernel/nn_routes.h on the wave64 emulator."""
import ctypes
import os
import subprocess

import torch

import host_nn as H

SO = os.path.join(H.SRC_DIR, "libumr_nn_routes.so")
KIND = {"forward": 0, "input": 1, "weight": 2}
_P, _L, _I, _F = ctypes.c_void_p, ctypes.c_long, ctypes.c_int, ctypes.c_float

# (direction, M, G, N, K): tiles that overlap in both directions, a contraction of several steps whose last one is cut; one and several heads
WIDE = [("forward", 4000, 1, 4090, 523), ("input", 4000, 1, 517, 4090), ("weight", 541, 1, 4000, 4090),
        ("forward", 1230, 10, 1241, 577), ("input", 1230, 10, 515, 1241), ("weight", 1031, 10, 1230, 1241)]


def widest(dtype):
    return 128 if dtype == torch.float32 else 256


def lib():
    csrc = os.path.join(H.ROOT, "umr_amd", "csrc")
    deps = [os.path.join(H.SRC_DIR, f) for f in ("nn_tu.cpp", "nn_routes.h", "wave_emu.h")] + \
           [os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith((".hip", ".h"))] + \
           [os.path.join(H.ROOT, "include", f) for f in ("umr_hip.h", "umr_nn.h")]
    if not os.path.exists(SO) or os.path.getmtime(SO) < max(os.path.getmtime(d) for d in deps):
        tmp = SO + ".%d" % os.getpid()
        subprocess.check_call([H.CLANG, "-O1", "-g", "-std=c++17", "-fPIC", "-shared", "-ffp-contract=off", "-mf16c", "-Wno-unused-function", "-Wno-unknown-attributes",
                               "-Wno-ignored-attributes", "-Wno-unknown-pragmas", "-Wno-pass-failed", "-Wno-psabi", '-DUMR_TU="nn_routes.h"',
                               os.path.join(H.SRC_DIR, "nn_tu.cpp"), "-o", tmp])
        os.replace(tmp, SO)
    L = ctypes.CDLL(SO)
    L.nn_route.argtypes = [_I, _L, _L, _L, _I, _I, ctypes.POINTER(_I)]
    L.nn_run_tile.argtypes = [_I, _I, _I, _P, _L, _L, _P, _L, _L, _P, _P, _L, _L, _P, _P, _L, _L, _L, _I, _I, _F, _L]
    return L


def route(L, direction, M, G, N, K, dtype):
    """(0 few rows / 1 outer products / the edge of the tile, parts of the contraction) of a layer's product"""
    nq, np, nc = {"forward": (M, N, K), "input": (M, K, N), "weight": (N, K, M)}[direction]
    parts = _I()
    return L.nn_route(KIND[direction], nq, np, nc, G, H.DTYPE[dtype], ctypes.byref(parts)), parts.value


def run_tile(L, direction, tile, x, w, gy, bias=None, res=None, act="none", slope=0.0, want_z=False, most=0):
    """x [M,G,K], w [G,N,K], gy [M,G,N] of which the direction's two are read -> (output, z or None); margins checked"""
    (M, G, K), N = (x if x is not None else gy).shape, (w if w is not None else gy).shape[1 if w is not None else 2]
    K = (x if x is not None else w).shape[2]
    rows = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))
    heads = lambda t: (t.data_ptr(), t.stride(1), t.stride(0))
    t = x if x is not None else w
    if direction == "forward":
        P, Q, nq, np, nc, shape = heads(w), rows(x), M, N, K, (M, G, N)
    elif direction == "input":
        P, Q, nq, np, nc, shape = heads(w), rows(gy), M, K, N, (M, G, K)
    else:
        P, Q, nq, np, nc, shape = rows(x), rows(gy), N, K, M, (G, N, K)
    out = H.Guarded(shape, t.dtype, "cpu")
    z = H.Guarded(shape, t.dtype if act in ("relu", "leaky_relu") else torch.float32, "cpu") if want_z else None
    rc = L.nn_run_tile(KIND[direction], tile, H.DTYPE[t.dtype], *P, *Q, None if bias is None else bias.data_ptr(),
                       *((None, 0, 0) if res is None else rows(res)), out.t.data_ptr(), z.t.data_ptr() if z else None, nq, np, nc, G, H.ACT[act], slope, most)
    if rc:
        return rc
    assert out.untouched_outside() and (z is None or z.untouched_outside())
    return out.t, (z.t if z else None)
