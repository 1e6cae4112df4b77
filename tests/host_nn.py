"""TEST INFRASTRUCTURE: umr_amd/csrc/linear.hip and balance.hip compiled for x86-64 on the wave64 emulator (host_kernel/nn_tu.cpp)
into libumr_nn_host.so, the C ABI of include/umr_nn.h on host pointers, and calls of that ABI on torch tensors of either side.
Never used by the product."""
import ctypes
import os
import subprocess

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CLANG = "/opt/rocm/lib/llvm/bin/clang++"
SRC_DIR = os.path.join(HERE, "host_kernel")
SO = os.path.join(SRC_DIR, "libumr_nn_host.so")
TUS = ["linear", "linear_f32", "linear_bf16", "linear_f16", "balance"]
DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACT = {"none": 0, "relu": 1, "leaky_relu": 2, "tanh": 3, "gelu": 4, "silu": 5}


def available():
    return os.path.exists(CLANG)


def build(extra_flags=(), out=SO):
    csrc = os.path.join(ROOT, "umr_amd", "csrc")
    deps = [os.path.join(SRC_DIR, f) for f in ("nn_tu.cpp", "wave_emu.h")] + \
           [os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith((".hip", ".h"))] + \
           [os.path.join(ROOT, "include", f) for f in ("umr_hip.h", "umr_nn.h")]
    if not extra_flags and os.path.exists(out) and os.path.getmtime(out) >= max(os.path.getmtime(d) for d in deps):
        return out
    os.makedirs(out + ".objs", exist_ok=True)
    objs = []
    procs = []
    for tu in TUS:
        obj = os.path.join(out + ".objs", tu + ".o")
        procs.append(subprocess.Popen([CLANG, "-O1", "-g", "-std=c++17", "-fPIC", "-ffp-contract=off", "-mf16c", "-Wno-unused-function",
                                       "-Wno-unknown-attributes", "-Wno-ignored-attributes", "-Wno-unknown-pragmas", "-Wno-pass-failed", "-Wno-psabi"] + list(extra_flags) +
                                      ['-DUMR_TU="../../umr_amd/csrc/%s.hip"' % tu, "-c", os.path.join(SRC_DIR, "nn_tu.cpp"), "-o", obj]))
        objs.append(obj)
    for p in procs:
        assert p.wait() == 0
    subprocess.check_call([CLANG, "-shared"] + list(extra_flags) + ["-o", out] + objs)
    return out


_LIB = {}


def lib(path=None):
    path = path or build()
    if path not in _LIB:
        from umr_amd._lib import SIGNATURES_NN
        L = ctypes.CDLL(path)
        for name, (argtypes, restype) in SIGNATURES_NN.items():
            getattr(L, name).argtypes, getattr(L, name).restype = argtypes, restype
        _LIB[path] = L
    return _LIB[path]


class Guarded:
    """A tensor in the middle of a larger buffer whose margins are checked afterwards; rows may be `pad` elements longer."""

    def __init__(self, shape, dtype, device, pad=0, fill=float("nan")):
        self.shape, self.pad = tuple(shape), pad
        full = self.shape[:-1] + (self.shape[-1] + pad,)
        n = 1
        for s in full:
            n *= s
        whole = fill if dtype.is_floating_point else -77
        self.buf = torch.full((n + 64,), whole, dtype=dtype, device=device)
        self.mark = self.buf.clone()
        self.t = self.buf[32:32 + n].view(full)[..., :self.shape[-1]]

    def untouched_outside(self):
        m, b = self.mark.clone(), self.buf.clone()
        n = b.numel() - 64
        for v in (m, b):
            v[32:32 + n].view(self.shape[:-1] + (self.shape[-1] + self.pad,))[..., :self.shape[-1]] = 0
        return torch.equal(torch.nan_to_num(m.double(), nan=-1.0), torch.nan_to_num(b.double(), nan=-1.0))


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """(row, head) strides of [M, G, .]; ([G, N, .]: pass w=True order swapped by the caller)"""
    return (0, 0) if t is None else (t.stride(0), t.stride(1))


def _ws(n, device):
    return torch.full((n + 16,), 255, dtype=torch.uint8, device=device), n


def linear_forward(L, x, w, b, r, act, slope, want_z, stream=None):
    """x [M,G,K], w [G,N,K], b [G,N], r [M,G,N] -> (y, z or None), the buffers' margins checked"""
    M, G, K = x.shape
    N = w.shape[1]
    dt = DTYPE[x.dtype]
    y = Guarded((M, G, N), x.dtype, x.device)
    z = Guarded((M, G, N), x.dtype if act in ("relu", "leaky_relu") else torch.float32, x.device) if want_z else None
    ws, n = _ws(L.umr_linear_forward_workspace_bytes(M, N, K, G, dt), x.device)
    rc = L.umr_linear_forward(_p(x), x.stride(0), x.stride(1), _p(w), w.stride(1), w.stride(0), _p(b), _p(r), *_rows(r), _p(y.t),
                              _p(z.t) if z else None, M, N, K, G, dt, ACT[act], slope, _p(ws), n, stream)
    assert rc == 0
    if x.is_cuda:
        torch.cuda.synchronize()
    assert bool((ws[n:] == 255).all()) and y.untouched_outside() and (z is None or z.untouched_outside())
    return y.t, (z.t if z else None)


def linear_grad_act(L, gy, z, act, slope, want_db=True, want_dr=True, stream=None):
    M, G, N = gy.shape
    dt = DTYPE[gy.dtype]
    dz = Guarded((M, G, N), gy.dtype, gy.device) if act != "none" else None
    db = Guarded((G, N), gy.dtype, gy.device) if want_db else None
    dr = Guarded((G, N), gy.dtype, gy.device) if want_dr else None
    ws, n = _ws(L.umr_linear_grad_act_workspace_bytes(M, N, G), gy.device)
    opt = lambda v: _p(v.t) if v else None
    rc = L.umr_linear_grad_act(_p(gy), *_rows(gy), _p(z), opt(dz), opt(db), opt(dr), M, N, G, dt, ACT[act], slope, _p(ws), n, stream)
    assert rc == 0
    if gy.is_cuda:
        torch.cuda.synchronize()
    assert bool((ws[n:] == 255).all()) and all(v is None or v.untouched_outside() for v in (dz, db, dr))
    return tuple(v.t if v else None for v in (dz, db, dr))


def linear_grad_input(L, dz, w, stream=None):
    M, G, N = dz.shape
    K = w.shape[2]
    dt = DTYPE[dz.dtype]
    dx = Guarded((M, G, K), dz.dtype, dz.device)
    ws, n = _ws(L.umr_linear_grad_input_workspace_bytes(M, N, K, G, dt), dz.device)
    rc = L.umr_linear_grad_input(_p(dz), *_rows(dz), _p(w), w.stride(1), w.stride(0), _p(dx.t), M, N, K, G, dt, _p(ws), n, stream)
    assert rc == 0
    if dz.is_cuda:
        torch.cuda.synchronize()
    assert bool((ws[n:] == 255).all()) and dx.untouched_outside()
    return dx.t


def linear_grad_weight(L, dz, x, stream=None):
    M, G, N = dz.shape
    K = x.shape[2]
    dt = DTYPE[dz.dtype]
    dw = Guarded((G, N, K), dz.dtype, dz.device)
    ws, n = _ws(L.umr_linear_grad_weight_workspace_bytes(M, N, K, G, dt), dz.device)
    rc = L.umr_linear_grad_weight(_p(dz), *_rows(dz), _p(x), *_rows(x), _p(dw.t), M, N, K, G, dt, _p(ws), n, stream)
    assert rc == 0
    if dz.is_cuda:
        torch.cuda.synchronize()
    assert bool((ws[n:] == 255).all()) and dw.untouched_outside()
    return dw.t


def balance_forward(L, z, inds, mask, stream=None):
    T, E = z.shape
    k = inds.shape[1]
    dt = DTYPE[z.dtype]
    loss, coef = Guarded((1,), torch.float32, z.device), Guarded((E + 1,), torch.float32, z.device)
    counts = Guarded((E,), torch.int64, z.device)
    ws, n = _ws(L.umr_balance_workspace_bytes(T, E), z.device)
    rc = L.umr_balance_forward(_p(z), _p(inds), _p(mask), _p(loss.t), _p(counts.t), _p(coef.t), T, E, k, dt, _p(ws), n, stream)
    assert rc == 0
    if z.is_cuda:
        torch.cuda.synchronize()
    assert bool((ws[n:] == 255).all()) and all(v.untouched_outside() for v in (loss, counts, coef))
    return loss.t, counts.t, coef.t


def balance_backward(L, z, mask, coef, grad, stream=None):
    T, E = z.shape
    dz = Guarded((T, E), z.dtype, z.device)
    rc = L.umr_balance_backward(_p(z), _p(mask), _p(coef), _p(grad), _p(dz.t), T, E, DTYPE[z.dtype], stream)
    assert rc == 0
    if z.is_cuda:
        torch.cuda.synchronize()
    assert dz.untouched_outside()
    return dz.t
