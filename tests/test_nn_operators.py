"""CPU tests of the network-side operators (include/umr_nn.h): every kernel of csrc/linear.hip and csrc/balance.hip on the wave64
emulator against its definition in 64 bits, and what each interface refuses.  tests/test_gpu_nn_operators.py has the GPU side."""
import ctypes
import os
import re

import pytest
import torch

import host_nn as H
import nn_checks as C

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = [torch.float32, torch.bfloat16, torch.float16]
needs_clang = pytest.mark.skipif(not H.available(), reason="clang++ of the ROCm toolchain not present")


def test_every_declared_symbol_is_exported_and_in_the_prototype_table():
    from umr_amd import _lib, build, ops_nn
    build.build(verbose=False)
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "umr_nn.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(umr_[a-z0-9_]+)\s*\(", text))
    assert declared == set(_lib.SIGNATURES_NN) and len(declared) == 11
    handle = ctypes.CDLL(_lib.LIB_PATH)
    for name in declared:
        assert hasattr(handle, name), name
    assert ops_nn.build_id() == build.source_hash() == _lib.build_id()
    assert ops_nn.MAX_CHOICES == int(re.search(r"UMR_BALANCE_MAX_CHOICES (\d+)", text).group(1))
    for name, v in ops_nn.ACTIVATIONS.items():
        assert int(re.search(r"UMR_ACT_%s (\d+)" % name.upper(), text).group(1)) == v


# few rows / tiles, a part of a tile, one element, nothing to sum, odd rows in memory, split contractions, several heads
LINEAR = [(1, 1, 1, 1, 0), (1, 1, 200, 200, 0), (3, 2, 37, 5, 1), (16, 1, 64, 700, 0), (17, 1, 33, 130, 3), (40, 2, 20, 600, 0),
          (65, 1, 70, 100, 0), (130, 2, 129, 40, 1), (70, 1, 3, 1000, 0), (300, 1, 5, 9, 2), (5, 1, 7, 0, 0)]


@needs_clang
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,G,N,K,pad", LINEAR)
def test_linear_against_64_bits(M, G, N, K, pad, dtype):
    C.check_linear(H.lib(), M, G, N, K, dtype, "gelu", pad=pad)


@needs_clang
@pytest.mark.parametrize("act", list(H.ACT))
@pytest.mark.parametrize("bias,residual", [(True, True), (False, True), (True, False), (False, False)])
def test_linear_activations_bias_and_residual(act, bias, residual):
    C.check_linear(H.lib(), 6, 2, 21, 19, torch.float32, act, bias=bias, residual=residual)
    C.check_linear(H.lib(), 66, 1, 21, 19, torch.bfloat16, act, bias=bias, residual=residual)


@needs_clang
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_linear_broadcast_operands_and_no_rows(dtype):
    """strides of 0 (one row for all, one head's weights for all, a gradient that is one number) read like their copies; no rows or
    no columns: the sums are 0 and nothing else is written"""
    L = H.lib()
    x, w, b, r, _ = C.inputs(9, 3, 10, 12, dtype, "cpu")
    x1, w1, r1 = x[:1].expand(9, 3, 12), w[:1].expand(3, 10, 12), r[:1].expand(9, 3, 10)
    y, z = H.linear_forward(L, x1, w1, b, r1, "silu", 0.0, True)
    yc, zc = H.linear_forward(L, x1.contiguous(), w1.contiguous(), b, r1.contiguous(), "silu", 0.0, True)
    assert torch.equal(y, yc) and torch.equal(z, zc)
    one = torch.ones(1, 1, 1, dtype=dtype).expand(9, 3, 10)
    copy = torch.ones(9, 3, 10, dtype=dtype)
    for a, c in zip(H.linear_grad_act(L, one[..., :1], z[..., :1].contiguous(), "silu", 0.0), H.linear_grad_act(L, copy[..., :1].contiguous(), z[..., :1].contiguous(), "silu", 0.0)):
        assert torch.equal(a, c)
    empty = torch.zeros(0, 3, 10, dtype=dtype)
    dz, db, dr = H.linear_grad_act(L, empty, torch.zeros(0, 3, 10), "silu", 0.0)
    assert bool((db == 0).all()) and bool((dr == 0).all())
    assert bool((H.linear_grad_weight(L, empty, torch.zeros(0, 3, 12, dtype=dtype)) == 0).all())
    assert bool((H.linear_grad_input(L, torch.zeros(4, 3, 0, dtype=dtype), torch.zeros(3, 0, 12, dtype=dtype)) == 0).all())


@needs_clang
def test_linear_lets_infinities_and_nan_through_but_only_where_they_belong():
    """a row with a NaN or an infinity poisons its own results and no neighbour's, also where a tile's edge repeats rows"""
    L = H.lib()
    for M, act in ((5, "none"), (5, "relu"), (70, "none"), (70, "gelu")):
        x, w, b, r, _ = C.inputs(M, 1, 33, 20, torch.float32, "cpu")
        clean, _ = H.linear_forward(L, x, w, b, None, act, 0.0, False)
        bad = x.clone()
        bad[M - 1, 0, 3], bad[M - 2, 0, 19] = float("nan"), float("inf")
        y, _ = H.linear_forward(L, bad, w, b, None, act, 0.0, False)
        assert torch.equal(y[:M - 2], clean[:M - 2]) and bool(y[M - 1].isnan().all())
        want = C.act64(torch.einsum("mgk,gnk->mgn", bad[M - 2:M - 1].double(), w.double()) + b.double(), act, 0.0)
        assert torch.equal(torch.nan_to_num(y[M - 2:M - 1].double(), nan=7.0), torch.nan_to_num(want, nan=7.0))


@needs_clang
@pytest.mark.parametrize("act", ["tanh", "gelu", "silu"])
def test_linear_gradient_against_differences(act):
    """the gradient in x, w and b of sum(y * g) against the central difference of the 64-bit formula along a direction d: its error is
    h^2 / 6 times the third derivative along d, bounded here by 4 (|act'''| <= 4) times sum |g| |dz/dh|^3"""
    L = H.lib()
    x, w, b, r, gy = C.inputs(4, 2, 6, 5, torch.float32, "cpu")
    y, z = H.linear_forward(L, x, w, b, r, act, 0.0, True)
    dz, db, dr = H.linear_grad_act(L, gy, z.contiguous(), act, 0.0)
    grads = dict(x=H.linear_grad_input(L, dz, w), w=H.linear_grad_weight(L, dz, x), b=db, r=gy)
    at = dict(x=x.double(), w=w.double(), b=b.double(), r=r.double())
    h = 1e-4

    def value(v):
        return ((C.act64(torch.einsum("mgk,gnk->mgn", v["x"], v["w"]) + v["b"], act, 0.0) + v["r"]) * gy.double()).sum()
    gen = torch.Generator().manual_seed(3)
    for name in at:
        d = torch.randn(at[name].shape, generator=gen).double()
        plus, minus = (value(dict(at, **{name: at[name] + s * h * d})) for s in (1, -1))
        slope = (plus - minus) / (2 * h)
        got = (grads[name].double() * d).sum()
        dzdh = {"x": lambda: torch.einsum("mgk,gnk->mgn", d, at["w"]), "w": lambda: torch.einsum("mgk,gnk->mgn", at["x"], d),
                "b": lambda: d.expand(4, 2, 6), "r": lambda: torch.zeros(4, 2, 6)}[name]()
        tol = h * h / 6 * 4 * (gy.double().abs() * dzdh.abs() ** 3).sum() + 100 * C.U * (grads[name].double().abs() * d.abs()).sum() + 1e-9
        assert abs(float(got - slope)) <= float(tol), (name, float(got), float(slope))


BALANCE = [(1, 1, 1, "none"), (1, 5, 2, "none"), (16, 8, 1, "none"), (100, 61, 2, "both"), (333, 128, 3, "rows"), (50, 300, 1, "choices"),
           (9, 1024, 5, "both"), (700, 3, 2, "both"), (40, 16, 4, "nothing"), (0, 7, 1, "none"), (2000, 33, 1, "both")]


@needs_clang
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k,mask", BALANCE)
def test_balance_against_64_bits(T, E, k, mask, dtype):
    C.check_balance(H.lib(), T, E, k, dtype, mask)


@needs_clang
def test_balance_values_that_are_known():
    L = H.lib()
    z, even = torch.zeros(12, 4), torch.arange(12).reshape(12, 1) % 4
    loss, counts, coef = H.balance_forward(L, z, even, None)
    assert float(loss) == 1.0 and counts.tolist() == [3, 3, 3, 3] and bool((coef[:4] == 0).all())
    loss, counts, _ = H.balance_forward(L, torch.tensor([[50.0, 0.0], [50.0, 0.0]]), torch.zeros(2, 3, dtype=torch.int64), None)
    assert float(loss) == 2.0 and counts.tolist() == [6, 0]                  # everything on one of two, an index three times in a row
    for bad in (float("nan"), float("inf")):
        z = torch.zeros(3, 4)
        z[1, 2] = bad
        loss, _, coef = H.balance_forward(L, z, even[:3], None)
        dz = H.balance_backward(L, z, None, coef, torch.ones(1))
        assert bool(loss.isnan()) and bool(dz[1].isnan().all()) and bool(dz[[0, 2]].isfinite().all())
        loss, counts, coef = H.balance_forward(L, z, even[:3], torch.tensor([True, False, True]))
        assert bool(loss.isfinite()) and counts.tolist() == [1, 0, 1, 0]


def test_c_abi_refusals():
    """UMR_ERR_ARG before anything is enqueued"""
    from umr_amd import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(16)

    def forward(M=4, N=4, K=4, G=1, dtype=0, act=0, slope=0.0, x=p, w=p, y=p, strides=(4, 4), ws=None, n=0):
        return L.umr_linear_forward(x, strides[0], strides[1], w, 4, 16, None, None, 0, 0, y, None, M, N, K, G, dtype, act, slope, ws, n, None)
    for kw in (dict(M=-1), dict(N=-1), dict(K=-1), dict(G=0), dict(G=65536), dict(dtype=3), dict(dtype=-1), dict(act=6), dict(act=-1),
               dict(act=2, slope=-0.1), dict(act=2, slope=float("nan")), dict(x=None), dict(w=None), dict(y=None), dict(strides=(-1, 0)),
               dict(M=2 ** 27), dict(N=2 ** 31), dict(M=2 ** 26, G=60000, N=2 ** 20)):
        assert forward(**kw) == -1, kw
    assert forward(M=0) == 0 and forward(N=0) == 0                          # nothing to do, nothing enqueued
    need = L.umr_linear_forward_workspace_bytes(16, 8, 8192, 1, 0)
    assert need > 0 and forward(M=16, N=8, K=8192) == -1                    # no workspace
    assert forward(M=16, N=8, K=8192, ws=p, n=need - 1) == -1               # too small a one
    assert L.umr_linear_grad_input(None, 4, 4, p, 4, 16, p, 4, 4, 4, 1, 0, None, 0, None) == -1
    assert L.umr_linear_grad_weight(p, 4, 4, p, 4, 4, None, 4, 4, 4, 1, 0, None, 0, None) == -1
    assert L.umr_linear_grad_act(p, 4, 4, p, None, p, None, 4, 4, 1, 0, 4, 0.0, None, 0, None) == -1     # an activation without dz
    assert L.umr_linear_grad_act(p, 4, 4, None, p, p, None, 4, 4, 1, 0, 4, 0.0, None, 0, None) == -1     # ... without z
    assert L.umr_linear_grad_act(p, 4, 4, p, p, p, None, 4, 4, 1, 0, 0, 0.0, None, 0, None) == -1        # dz without an activation
    assert L.umr_linear_grad_act(p, 4, 4, None, None, p, None, 100000, 4, 1, 0, 0, 0.0, None, 0, None) == -1

    def balance(z=p, inds=p, T=4, E=4, k=1, dtype=0, ws=None, n=0, loss=p):
        return L.umr_balance_forward(z, inds, None, loss, p, p, T, E, k, dtype, ws, n, None)
    for kw in (dict(z=None), dict(inds=None), dict(T=-1), dict(E=0), dict(E=1025), dict(k=0), dict(dtype=5), dict(loss=None),
               dict(T=100000, E=64), dict(T=2 ** 30, k=4, ws=p, n=1 << 40)):
        assert balance(**kw) == -1, kw
    assert L.umr_balance_backward(p, None, None, p, p, 4, 4, 0, None) == -1
    assert L.umr_balance_backward(p, None, p, None, p, 4, 4, 0, None) == -1
    assert L.umr_balance_backward(p, None, p, p, None, 4, 4, 0, None) == -1


def test_operator_refusals():
    from umr_amd import functional as UF
    m = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="meta")
    with pytest.raises(RuntimeError, match="no CPU path"):
        UF.linear_act(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="no CPU path"):
        UF.balance_loss(torch.zeros(2, 3), torch.zeros(2, 1, dtype=torch.int64))
    for args, kw, text in (
            ((m(2, 3), m(4, 5)), {}, "does not fit weight"), ((m(2, 3), m(4)), {}, "weight must be"),
            ((m(2, 3), m(2, 4, 3)), {}, "weight must be"), ((m(2, 3, dtype=torch.float64), m(4, 3, dtype=torch.float64)), {}, "float32, bfloat16"),
            ((m(2, 3), m(4, 3, dtype=torch.bfloat16)), {}, "weight is"), ((m(2, 3), m(4, 3), m(3)), {}, "bias"),
            ((m(2, 3), m(4, 3), m(4, dtype=torch.float16)), {}, "bias is"), ((m(2, 3), m(4, 3)), dict(residual=m(3, 4)), "residual must be"),
            ((m(2, 3), m(4, 3)), dict(residual=m(2, 4, dtype=torch.float16)), "residual is"),
            ((m(2, 3), m(4, 3)), dict(residual=m(1, 4)), "residual must be"),
            ((m(2, 3), m(4, 3)), dict(activation="leaky_relu", slope=-1.0), "slope")):
        with pytest.raises(RuntimeError, match=text):
            UF.linear_act(*args, **kw)
    with pytest.raises(ValueError, match="activation must be one of"):
        UF.linear_act(m(2, 3), m(4, 3), activation="swish")
    with pytest.raises(RuntimeError, match="does not fit weight"):
        UF.heads_linear_act(m(2, 3, 3), m(2, 4, 3))
    with pytest.raises(RuntimeError, match="weight must be"):
        UF.heads_linear_act(m(2, 3), m(4, 3))
    i = lambda *s: m(*s, dtype=torch.int64)
    for args, text in (((m(4), i(4, 1)), "scores must be"), ((m(4, 1025), i(4, 1)), "scores must be"), ((m(4, 3), i(5, 1)), "inds must be"),
                       ((m(4, 3), i(4, 0)), "inds must be"), ((m(4, 3), m(4, 1)), "inds must be"), ((m(4, 3), i(4, 1), m(4)), "mask must be"),
                       ((m(4, 3), i(4, 1), m(3, dtype=torch.bool)), "mask must be"), ((m(4, 3, dtype=torch.float64), i(4, 1)), "float32, bfloat16")):
        with pytest.raises(RuntimeError, match=text):
            UF.balance_loss(*args)


def test_operators_have_shapes_without_a_device():
    """meta tensors through both operators and their backward: shapes, types, and no second derivative"""
    from umr_amd import functional as UF
    m = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="meta", requires_grad=True)
    x, w, b, r = m(2, 5, 3, 6), m(3, 4, 6), m(3, 4), m(3, 4)
    y = UF.heads_linear_act(x, w, b, residual=r, activation="gelu")
    assert y.shape == (2, 5, 3, 4) and y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y.sum(), [x, w, b, r])
    assert [g.shape for g in grads] == [t.shape for t in (x, w, b, r)]
    y = UF.linear_act(m(6), m(4, 6))
    assert y.shape == (4,)
    z = m(7, 5)
    loss, counts = UF.balance_loss(z, torch.empty(7, 2, dtype=torch.int64, device="meta"))
    assert loss.shape == () and loss.dtype == torch.float32 and counts.shape == (5,) and counts.dtype == torch.int64 and not counts.requires_grad
    assert torch.autograd.grad(loss, z)[0].shape == z.shape
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(UF.linear_act(m(2, 6), w[0], activation="tanh").sum(), w, create_graph=True)


# ---------------------------------------------------------------------------------------------- MeshNet's layers (host tensors: plain torch)
def _tiny_net(seed=0, **kw):
    from umr_amd import model as M
    torch.manual_seed(seed)
    opts = M.default_opts(multiple_cam_hypo=True, subdivide=1, **kw)
    return M, M.MeshNet((64, 64), opts, nz_feat=opts.nz_feat)


def test_fused_layers_keep_the_state_dict_and_the_values():
    import copy
    M, net = _tiny_net()
    fused = M.fuse_linears(copy.deepcopy(net))
    assert list(fused.state_dict()) == list(net.state_dict())
    assert not any(type(m) is torch.nn.Linear for m in fused.modules()) and sum(isinstance(m, M.Linear) for m in fused.modules()) == \
        sum(type(m) is torch.nn.Linear for m in net.modules())
    # a LeakyReLU right behind a layer moved into it: the hypotheses' shared stack, the two latent heads; one behind a batch norm stayed
    assert [l[0].activation for l in fused.cam_predictor.fc] == ["leaky_relu"] * 2 and fused.cam_predictor.fc[0][0].slope == pytest.approx(0.1)
    assert fused.encoder.mean_fc[0].activation == "leaky_relu" and fused.encoder.enc_fc[0][0].activation == "none"
    assert type(fused.encoder.enc_fc[0][2]) is torch.nn.LeakyReLU and type(fused.encoder.mean_fc[1]) is torch.nn.Identity
    assert M.MeshNet((64, 64), M.default_opts(subdivide=1, fused_fc=True)).shape_predictor.pred_layer.__class__ is M.Linear
    x = torch.randn(2, 3, 64, 64)
    torch.manual_seed(5)
    a = net(x)
    torch.manual_seed(5)
    b = fused(x)
    assert list(a) == list(b) and all(torch.equal(a[k], b[k]) for k in a)
    assert torch.equal(torch.softmax(a["cam_logits"], 1), a["cam_probs"])


def test_folded_net_equals_the_net_in_eval_mode():
    M, net = _tiny_net(1)
    for k in range(3):                                                   # running statistics that are not the initial ones
        net(torch.randn(4, 3, 64, 64))
    net = net.double().eval()
    folded = M.fold_for_inference(net)
    assert not any(isinstance(m, torch.nn.BatchNorm1d) for m in folded.modules()) and not any(p.requires_grad for p in folded.parameters())
    assert isinstance(folded.cam_predictor.camera_predictor, M.FoldedCameras) and not isinstance(net.cam_predictor.camera_predictor, M.FoldedCameras)
    again = M.fold_for_inference(M.fuse_linears(net))                    # of a net whose layers were fused already
    x = torch.randn(2, 3, 64, 64).double()
    outs = []
    for m in (net, folded, again):
        torch.manual_seed(5)
        outs.append(m(x))
    for k in outs[0]:
        for o in outs[1:]:       # in 64 bits: the same numbers in another order of operations (scale_bias and 1e-12 of the cameras are fp32 constants' sums)
            assert float((outs[0][k].double() - o[k].double()).abs().max()) <= 1e-9 * max(1.0, float(outs[0][k].double().abs().max())), k

