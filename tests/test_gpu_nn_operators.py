"""GPU tests of the network-side operators (include/umr_nn.h): the kernels at sizes that take every route through them, and
umr_amd.functional's linear_act / heads_linear_act / balance_loss as a user calls them."""
import pytest
import torch

import host_nn as H
import nn_checks as C

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _lib():
    from umr_amd import _lib
    return _lib.lib()


# few rows (one, two, four row blocks; split and not; odd rows in memory), tiles of 64 and 128 (edges in each direction, split), heads
LINEAR = [(1, 1, 200, 200, 0), (1, 1, 1, 1, 0), (16, 1, 200, 4096, 0), (5, 3, 1011, 350, 3), (31, 1, 515, 2047, 1), (64, 2, 130, 700, 8),
          (65, 1, 129, 65, 1), (777, 1, 301, 515, 13), (1000, 1, 1011, 350, 0), (2500, 1, 2049, 130, 0), (130, 9, 200, 200, 0),
          (70, 1, 5, 20000, 0), (20000, 1, 7, 3, 0), (300, 1, 7, 0, 0)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,G,N,K,pad", LINEAR)
def test_linear_against_64_bits(M, G, N, K, pad, dtype):
    C.check_linear(_lib(), M, G, N, K, dtype, "silu", device=DEV, pad=pad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_linear_largest_tiles_against_64_bits(dtype):
    """enough 16-bit results for the 256 x 256 tiles, with tiles that overlap in both directions and a cut last step, in each product"""
    C.check_linear(_lib(), 4100, 1, 4099, 203, dtype, "gelu", device=DEV, pad=1, parts=("forward",))
    C.check_linear(_lib(), 4100, 1, 77, 4099, dtype, "none", device=DEV, parts=("input",))
    C.check_linear(_lib(), 77, 1, 4100, 4099, dtype, "none", device=DEV, parts=("weight",))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_linear_largest_tiles_long_contraction_against_64_bits(dtype):
    """as above, over contractions of at least 512, with a cut last step"""
    C.check_linear(_lib(), 4100, 1, 4099, 523, dtype, "gelu", device=DEV, pad=1, parts=("forward",))
    C.check_linear(_lib(), 4100, 1, 517, 4099, dtype, "none", device=DEV, parts=("input",))
    C.check_linear(_lib(), 541, 1, 4100, 4099, dtype, "none", device=DEV, parts=("weight",))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("M,G,N,K", [(1, 1, 64, 64), (16, 2, 65, 131), (17, 1, 4100, 2049), (31, 1, 2899, 2901), (32, 3, 1500, 2000), (33, 1, 2049, 4099),
                                     (64, 1, 2899, 2901)])
def test_linear_weight_gradient_of_few_rows_against_64_bits(M, G, N, K, dtype):
    """outer products: up to 16 rows of any result, up to 64 of a large one, and what goes to the tiles next to them"""
    C.check_linear(_lib(), M, G, N, K, dtype, "none", device=DEV, parts=("weight",))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", list(H.ACT))
def test_linear_activations(act, dtype):
    C.check_linear(_lib(), 33, 2, 70, 64, dtype, act, device=DEV)
    C.check_linear(_lib(), 200, 1, 70, 64, dtype, act, device=DEV, bias=False, residual=False)


BALANCE = [(1, 1, 1, "none"), (16, 8, 1, "none"), (5001, 61, 2, "both"), (70000, 128, 8, "rows"), (3000, 1000, 3, "choices"), (40000, 3, 2, "both"),
           (640, 16, 4, "nothing"), (0, 7, 1, "none"), (9000, 257, 1, "both"), (1025, 513, 2, "rows")]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k,mask", BALANCE)
def test_balance_against_64_bits(T, E, k, mask, dtype):
    C.check_balance(_lib(), T, E, k, dtype, mask, device=DEV)


def _layer64(x, w, b, r, act, slope, gy):
    """z, the sum of the magnitudes that enter it, y and dz in 64 bits"""
    x, w, b, r, gy = (t.detach().double() for t in (x, w, b, r, gy))
    z = torch.einsum("mgk,gnk->mgn", x, w) + b
    zmag = torch.einsum("mgk,gnk->mgn", x.abs(), w.abs()) + b.abs()
    y = C.act64(z, act, slope) + r
    dz = gy * C.act_slope64(z, act, slope)
    return z, zmag, y, dz


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ["none", "tanh", "gelu", "silu"])
@pytest.mark.parametrize("M,G,N,K", [(1, 4, 200, 200), (16, 8, 200, 200), (100, 3, 65, 130), (3, 1, 9, 4)])
def test_layers_and_their_gradients(M, G, N, K, act, dtype):
    """heads_linear_act on strided inputs, every gradient through autograd, full and one-row residual; linear_act on the heads that share
    their input"""
    from umr_amd import functional as UF
    x, w, b, r, gy = C.inputs(M, G, N, K, dtype, DEV, pad=3)
    z, zmag, y64, dz64 = _layer64(x, w, b, r, act, 0.0, gy)
    U, e = C.U, C.half_step(dtype)
    ztol = (K + 2) * U * zmag
    ytol = 1.13 * ztol + 16 * U * (z.abs() + 1) + U * (y64.abs() + 2 * r.double().abs())
    # dz: |act''| <= 0.8 on the error of z, the evaluation of act', one rounding to the type (none without an activation)
    dtol = torch.zeros_like(z) if act == "none" else gy.double().abs() * (0.8 * ztol + 32 * U * (z.abs() + 1)) + e * dz64.abs()
    x64, w64 = x.double(), w.double()
    dmag = dz64.abs() + dtol
    want = dict(x=(torch.einsum("mgn,gnk->mgk", dz64, w64), torch.einsum("mgn,gnk->mgk", dtol + (N + 2) * U * dmag, w64.abs())),
                w=(torch.einsum("mgn,mgk->gnk", dz64, x64), torch.einsum("mgn,mgk->gnk", dtol + (M + 2) * U * dmag, x64.abs())),
                b=(dz64.sum(0), (dtol + (M + 2) * U * dmag).sum(0)))
    for one_row in (False, True):
        leaves = dict(x=x, w=w, b=b, r=(r[0] if one_row else r))
        leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
        y = UF.heads_linear_act(leaves["x"], leaves["w"], leaves["b"], residual=leaves["r"], activation=act)
        res = r[:1].expand_as(r).double() if one_row else r.double()
        C.close(y.detach(), y64 - r.double() + res, ytol + U * res.abs(), "y")
        grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))
        for name in want:
            C.close(grads[name], *want[name], name)
        if one_row:
            C.close(grads["r"], gy.double().sum(0), (M + 2) * U * gy.double().abs().sum(0), "r")
        else:
            assert torch.equal(grads["r"], gy)
    # heads that share their input are one layer
    shared = x[:, 0]
    y = UF.linear_act(shared, w.flatten(0, 1), b.flatten(), activation=act).unflatten(-1, (G, N))
    per = UF.heads_linear_act(shared.unsqueeze(1).expand(M, G, K), w, b, activation=act)
    tol = 2 * (1.13 * (K + 2) * U * (torch.einsum("mk,gnk->mgn", shared.double().abs(), w64.abs()) + b.double().abs()) + 16 * U * (z.abs().amax() + 1))
    C.close(y, per.double(), tol + e * per.double().abs(), "shared input")


def test_leading_dimensions_strides_and_one_row():
    from umr_amd import functional as UF
    g = torch.Generator(device=DEV).manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    x, w, b = rnd(4, 5, 6, 24), rnd(10, 24), rnd(10)
    flat = UF.linear_act(x.reshape(-1, 24), w, b, activation="relu")
    assert torch.equal(UF.linear_act(x, w, b, activation="relu").reshape(-1, 10), flat)
    for view in (x.transpose(0, 1), x[:, ::2], x.permute(2, 0, 1, 3), x[..., None, :].expand(4, 5, 6, 3, 24)):
        assert torch.equal(UF.linear_act(view, w, b, activation="relu"), UF.linear_act(view.contiguous(), w, b, activation="relu"))
    wt = rnd(24, 10).t()                                                    # weight whose columns lie together
    assert torch.equal(UF.linear_act(x, wt), UF.linear_act(x, wt.contiguous()))
    xt = rnd(24, 30).t()
    assert torch.equal(UF.linear_act(xt, w), UF.linear_act(xt.contiguous(), w))
    one = UF.linear_act(x[0, 0, 0], w, b, residual=b)                       # a vector in, a vector out
    assert one.shape == (10,) and torch.equal(one, UF.linear_act(x[0, 0, :1], w, b, residual=b)[0])
    assert UF.linear_act(x[:0], w, b).shape == (0, 5, 6, 10)
    # the gradient of a broadcast: one number for all outputs; no rows: zeros
    wl, xl = w.clone().requires_grad_(True), x.clone().requires_grad_(True)
    gs = torch.autograd.grad(UF.linear_act(xl, wl, activation="tanh").sum(), [xl, wl])
    ge = torch.autograd.grad(UF.linear_act(xl, wl, activation="tanh"), [xl, wl], torch.ones(4, 5, 6, 10, device=DEV))
    assert all(torch.equal(a, c) for a, c in zip(gs, ge))
    y = UF.linear_act(xl[:0], wl, activation="gelu")
    gx, gw = torch.autograd.grad(y.sum(), [xl, wl])
    assert bool((gx == 0).all()) and bool((gw == 0).all())
    # an input that needs no gradient gets none, and the others are the same bits
    only = torch.autograd.grad(UF.linear_act(x, wl, activation="tanh"), [wl], torch.ones(4, 5, 6, 10, device=DEV))[0]
    assert torch.equal(only, ge[1])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(UF.linear_act(xl, wl, activation="tanh").sum(), wl, create_graph=True)


def test_kinked_activations_keep_only_a_sign():
    """relu and leaky relu: without a residual the output serves the backward call, with one a copy of z does; 0 counts as negative"""
    from umr_amd import functional as UF
    x = torch.tensor([[-2.0], [0.0], [3.0]], device=DEV, requires_grad=True)
    w, r = torch.ones(1, 1, device=DEV), torch.full((3, 1), 5.0, device=DEV)
    for act, want in (("relu", [0.0, 0.0, 1.0]), ("leaky_relu", [0.25, 0.25, 1.0])):
        for res in (None, r):
            y = UF.linear_act(x, w, residual=res, activation=act, slope=0.25)
            assert torch.autograd.grad(y.sum(), x)[0].flatten().tolist() == want
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y = UF.linear_act(x, w, activation="relu")
        y.add_(1)
        y.sum().backward()


def test_offsets_beyond_32_bits():
    """outputs, weights and rows more than 2^31 elements in: the far ends against the same rows computed alone"""
    from umr_amd import functional as UF
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(70001, 24, device=DEV, generator=g).bfloat16()
    w = torch.randn(33000, 24, device=DEV, generator=g).bfloat16()
    y = UF.linear_act(x, w, activation="leaky_relu", slope=0.1)              # 2.3e9 outputs
    tail = UF.linear_act(x[-3:].clone(), w[-40:].clone(), activation="leaky_relu", slope=0.1)
    C.close(y[-3:, -40:].contiguous(), tail.double(), 52 * C.U * (x[-3:].double().abs() @ w[-40:].double().abs().t()) + 2.0 ** -8 * tail.double().abs(), "far outputs")
    gy = torch.zeros_like(y)
    gy[-1, -5:] = 1
    xl = x.clone().requires_grad_(True)
    gx, = torch.autograd.grad(UF.linear_act(xl, w), xl, gy)                  # reads the far end of a 2.3e9 gradient
    want = w[-5:].double().sum(0)
    C.close(gx[-1], want, 40000 * C.U * w[-5:].double().abs().sum(0), "dx of the last row")
    assert bool((gx[:-1] == 0).all())
    del y, gy, gx
    big = torch.zeros(3, 1 << 30, device=DEV, dtype=torch.bfloat16)          # rows 2^30 apart: the third is 2^31 elements in
    rows = big[:, :40]
    rows.copy_(torch.randn(3, 40, device=DEV, generator=g))
    w = torch.randn(7, 40, device=DEV, generator=g).bfloat16()
    assert torch.equal(UF.linear_act(rows, w), UF.linear_act(rows.contiguous(), w))
    assert torch.equal(UF.linear_act(w, rows), UF.linear_act(w, rows.contiguous()))
    del big, rows
    T = (1 << 31) // 64 + 5
    z = torch.zeros(T, 64, device=DEV, dtype=torch.bfloat16)
    z[-1, 3] = 40
    inds = torch.zeros(T, 1, device=DEV, dtype=torch.int64)
    inds[-1] = 3
    loss, counts = UF.balance_loss(z.requires_grad_(True), inds)
    assert counts[0] == T - 1 and counts[3] == 1
    assert abs(float(loss.detach()) - 1.0) < 1e-4
    dz, = torch.autograd.grad(loss, z, torch.tensor(float(T), device=DEV))
    assert float(dz[-1].abs().sum()) < 1e-6 and bool((dz[-2] == dz[0]).all()) and float(dz[0, 0]) > 0


def test_rows_far_apart_in_many_row_products():
    """rows of 2^22 elements and more in memory, more than 64 of them: the tiled kernels' 64-bit loads, for each operand of each product
    and each type; the same bits as from contiguous copies"""
    from umr_amd import functional as UF
    g = torch.Generator(device=DEV).manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.zeros(70, (1 << 22) + 3, device=DEV, dtype=dtype)
        for K in (40, 3, 131):
            x = big[:, 5:5 + K]
            x.copy_(torch.randn(70, K, device=DEV, generator=g))
            near = x.contiguous()
            w = torch.randn(90, K, device=DEV, generator=g).to(dtype)
            gy = torch.randn(70, 90, device=DEV, generator=g).to(dtype)
            gy2 = torch.randn(90, 70, device=DEV, generator=g).to(dtype)
            far_gy = big[:, 1000:1090]
            far_gy.copy_(gy)
            for a, b in ((x, near),):
                la, lb, wl = a.detach().requires_grad_(True), b.detach().requires_grad_(True), w.clone().requires_grad_(True)
                ya, yb = UF.linear_act(la, wl), UF.linear_act(lb, wl)            # x far: the fast Q operand, in dw the slow P one
                assert torch.equal(ya, yb)
                for u, v in zip(torch.autograd.grad(ya, [la, wl], far_gy), torch.autograd.grad(yb, [lb, wl], gy)):   # dz far: fast and slow Q
                    assert torch.equal(u, v)
                ya, yb = UF.linear_act(wl, la), UF.linear_act(wl, lb)            # the weight far: the fast P operand, in dx the slow one
                assert torch.equal(ya, yb)
                for u, v in zip(torch.autograd.grad(ya, [wl, la], gy2), torch.autograd.grad(yb, [wl, lb], gy2)):
                    assert torch.equal(u, v)


@pytest.mark.parametrize("want", ["x", "w", "b", "r", "xb", "wr", "br", "xwr"])
@pytest.mark.parametrize("bias", [True, False])
def test_gradients_of_some_inputs_only(want, bias):
    """any subset of the inputs may want a gradient, with and without a bias: each gets what it gets when all do, nothing else does"""
    from umr_amd import functional as UF
    x, w, b, r, gy = C.inputs(20, 2, 9, 7, torch.float32, DEV)
    for res in (r, r[0]):
        every = {k: v.detach().clone().requires_grad_(True) for k, v in dict(x=x, w=w, b=b, r=res).items()}
        call = lambda t: UF.heads_linear_act(t["x"], t["w"], t["b"] if bias else None, residual=t["r"], activation="gelu")
        names = [n for n in "xwbr" if bias or n != "b"]
        full = dict(zip(names, torch.autograd.grad(call(every), [every[n] for n in names], gy)))
        some = {k: v.detach().clone().requires_grad_(k in want) for k, v in every.items()}
        picked = [n for n in want if n in names]
        if not picked:
            assert not call(some).requires_grad
            continue
        call(some).backward(gy)
        for n in "xwbr":
            assert (some[n].grad is not None) == (n in picked), n
            if n in picked:
                assert torch.equal(some[n].grad, full[n]), n


def _capture(fn):
    """fn's first runs on a side stream, then captured"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_streams_and_graphs():
    """forward and backward of the operators on another stream, and captured: two graphs replayed in turn with eager work between them,
    every replay against the eager result on that replay's inputs"""
    from umr_amd import functional as UF

    def make(M, N, K, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(M, K, device=DEV, generator=g).requires_grad_(True)
        w = (torch.randn(N, K, device=DEV, generator=g) / 30).requires_grad_(True)
        b = torch.randn(N, device=DEV, generator=g).requires_grad_(True)
        r = torch.randn(N, device=DEV, generator=g).requires_grad_(True)
        inds = torch.randint(0, N, (M, 2), device=DEV, generator=g)

        def step():
            y = UF.linear_act(x, w, b, residual=r, activation="gelu")
            loss, counts = UF.balance_loss(y, inds)
            return [loss.detach(), counts, y.detach()] + list(torch.autograd.grad(loss + (y * y).mean(), [x, w, b, r]))
        return x, step
    cases = [make(16, 200, 4096, 1), make(700, 60, 900, 2)]                # split contractions and many-row sums: every workspace
    graphs = [_capture(step) for _, step in cases]
    gen = torch.Generator(device=DEV).manual_seed(9)
    for turn in range(4):
        for (x, step), (graph, out) in zip(cases, graphs):
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, device=DEV, generator=gen))
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = step()
            torch.cuda.current_stream().wait_stream(side)
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(eager, out):
                assert torch.equal(a, c), turn
    again = [step() for _, step in cases]
    for (x, step), first in zip(cases, again):
        assert all(torch.equal(a, c) for a, c in zip(first, step()))


def test_registered_operators_pass_opcheck():
    import umr_amd.ops_nn  # noqa: F401
    from torch.library import opcheck
    x, w, b, r, gy = C.inputs(5, 2, 6, 7, torch.float32, DEV)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
    utils = ("test_schema", "test_autograd_registration", "test_faketensor")
    opcheck(torch.ops.umr.linear_act, (*leaves, 4, 0.0), test_utils=utils)
    opcheck(torch.ops.umr.linear_act_backward, (gy.clone(), x, w, gy.clone(), 4, 0.0, True, True, True, True), test_utils=utils)
    z, inds, m = C.balance_inputs(9, 5, 2, torch.float32, DEV, "both")
    opcheck(torch.ops.umr.balance_loss, (z.requires_grad_(True), inds, m), test_utils=utils)


def test_a_routers_operators_together():
    """As they are used: a layer that every head shares, a layer of each head's own, one score a head, the softmax's choice, the balance
    loss over the heads; loss, counts and every gradient against the same in 64 bits, fp32 and 16 bits"""
    from umr_amd import functional as UF
    B, G, D = 64, 8, 200
    for dtype in (torch.float32, torch.bfloat16):
        gen = torch.Generator(device=DEV).manual_seed(4)
        rnd = lambda *s: torch.randn(*s, device=DEV, generator=gen)
        leaves = [t.to(dtype).requires_grad_(True) for t in (rnd(B, D), rnd(G * D, D) / D ** 0.5, 0.1 * rnd(G * D), rnd(G, 1, D) / D ** 0.5, 0.1 * rnd(G, 1))]
        x, w1, b1, w2, b2 = leaves
        hidden = UF.linear_act(x, w1, b1, activation="silu").unflatten(-1, (G, D))
        scores = UF.heads_linear_act(hidden, w2, b2)[..., 0]
        inds = torch.randint(0, G, (B, 1), device=DEV, generator=gen)
        loss, counts = UF.balance_loss(scores, inds)
        grads = torch.autograd.grad(loss, leaves, torch.tensor(float(B), device=DEV))
        d = [t.detach().double().requires_grad_(True) for t in leaves]
        h = torch.nn.functional.silu(d[0] @ d[1].t() + d[2]).unflatten(-1, (G, D))
        s = torch.einsum("bgd,gd->bg", h, d[3][:, 0]) + d[4][:, 0]
        c64 = torch.bincount(inds[:, 0], minlength=G)
        l64 = G * torch.dot(c64.double() / B, torch.softmax(s, 1).mean(0))
        g64 = torch.autograd.grad(l64, d, torch.tensor(float(B), device=DEV).double())
        assert torch.equal(counts, c64)
        # hidden, scores, d scores, d hidden and the gradients are each rounded to the type once; each rounding enters a gradient with
        # a factor of at most 2 in the 2-norm (softmax, silu and the products of unit variance here do not enlarge it), fp32 sums of
        # up to 1600 terms add 1600 u
        tol = 10 * C.half_step(dtype) + 1600 * C.U
        assert abs(float(loss.detach()) - float(l64.detach())) <= tol * float(l64.detach())
        for a, c in zip(grads, g64):
            assert float((a.double() - c).norm()) <= tol * float(c.norm())


# ---------------------------------------------------------------------------------------------- the framework's own paths
def _through(layers, x, err):
    """(value, bound) of linear layers [(weight, bias, slope or None)] in 64 bits: a layer adds (K + 3) u of its magnitudes (sum, bias,
    rounding) and passes the incoming error through |W|; a LeakyReLU does not enlarge it"""
    for w, b, slope in layers:
        w, b = w.double(), b.double()
        mag = x.abs() @ w.abs().t() + b.abs()
        x, err = x @ w.t() + b, err @ w.abs().t() + (w.shape[1] + 3) * C.U * mag
        if slope is not None:
            x = torch.nn.functional.leaky_relu(x, slope)
            err = err + C.U * x.abs()
    return x, err


def test_fused_and_folded_camera_predictor_against_64_bits():
    """MultiCamPredictor in eval mode, its layers fused and its cameras folded into three products, against the unfused module in
    64 bits: shared stack, then per camera three layers; the folded weights are each rounded once (u of their own magnitude)"""
    from umr_amd import model as M
    torch.manual_seed(3)
    net = M.MultiCamPredictor(200, 8).to(DEV)
    for m in net.modules():
        if isinstance(m, torch.nn.Linear):
            m.weight.data.normal_(0, 0.08)
        if isinstance(m, torch.nn.BatchNorm1d):
            m.running_mean.normal_(0, 0.3), m.running_var.uniform_(0.5, 2.0), m.weight.data.uniform_(0.5, 1.5), m.bias.data.normal_(0, 0.1)
    net.eval()
    folded = M.fold_for_inference(net)
    feat = torch.randn(16, 200, device=DEV)
    torch.manual_seed(0)
    cam, inds, probs, cams, quats, logits = folded(feat, with_logits=True)
    zero = torch.zeros(16, 200, device=DEV, dtype=torch.float64)
    f, ferr = _through([(l[0].weight, l[0].bias, 0.1) for l in net.fc], feat.double(), zero)
    got = M.fuse_linears(net).fc(feat)
    assert bool(((got.double() - f).abs() <= ferr).all())
    fc = folded.camera_predictor
    for k, c in enumerate(net.camera_predictor):
        h, err = f, ferr
        with torch.no_grad():
            for l in c.fc_layer:
                s = l[1].weight.double() / torch.sqrt(l[1].running_var.double() + l[1].eps)
                w, b = l[0].weight.double() * s[:, None], (l[0].bias.double() - l[1].running_mean.double()) * s + l[1].bias.double()
                err = err + C.U * h.abs()                                    # (the folded weight's rounding)
                h, err = _through([(w, b, 0.2)], h, err)
            last = [(p.weight, p.bias) for p in (c.quat_predictor.pred_layer, c.prob_predictor, c.scale_predictor.pred_layer, c.trans_predictor.pred_layer)]
            o, err = _through([(torch.cat([w for w, _ in last]), torch.cat([b for _, b in last]), None)], h, err)
        assert bool(((logits[:, k].double() - o[:, 4]).abs() <= err[:, 4]).all())
        assert bool(((cams[:, k, 1:3].double() - o[:, 6:8]).abs() <= err[:, 6:8]).all())
        scale = torch.relu(c.scale_lr * o[:, 5] + c.scale_bias) + 1e-12
        assert bool(((cams[:, k, 0].double() - scale).abs() <= err[:, 5] + 4 * C.U * scale.abs()).all())
        q, n = o[:, :4], o[:, :4].norm(dim=1, keepdim=True)
        # q / |q|: an error e of q moves it by at most 2 |e| / |q|; 8 roundings
        assert bool(((quats[:, k].double() - q / n).abs() <= 2 * err[:, :4].norm(dim=1, keepdim=True) / n + 8 * C.U).all())
    assert torch.equal(probs, torch.softmax(logits, 1)) and inds.shape == (16, 1)
    assert fc.w2.shape == (8, 200, 200)


def test_hypothesis_balance_loss_of_a_camera_predictor():
    """loss_utils.hypothesis_balance_loss on what MeshNet gives it, gradients into every camera's layers"""
    from umr_amd import loss_utils as LU, model as M
    torch.manual_seed(3)
    net = M.fuse_linears(M.MultiCamPredictor(200, 8)).to(DEV)
    feat = torch.randn(16, 200, device=DEV)
    out = net(feat, with_logits=True)
    loss, counts = LU.hypothesis_balance_loss(out[5], out[1])
    want, c64, d64, _ = C.balance64(out[5].detach(), out[1], None)
    assert torch.equal(counts, c64) and int(counts.sum()) == 16
    C.close(loss.detach(), want, 100 * C.U * want.abs(), "loss")
    loss.backward()
    for c in net.camera_predictor:
        g = c.prob_predictor.weight.grad
        assert g is not None and bool(torch.isfinite(g).all()) and float(g.abs().sum()) > 0


def _training_step(workload):
    import argparse
    from umr_amd import model as M
    from umr_amd.synthetic import make_s1_inputs
    dev = torch.device(DEV)
    args = argparse.Namespace(graph=1, batch=4, image_size=64 if workload == "s1" else 256, subdivide=2 if workload == "s1" else 3, epoch=0,
                              share_mask_render=1, data_seed=100, fused_fc=1, balance_wt=0.5)
    torch.manual_seed(77)
    if workload == "s2":
        return M, dev, M.build_training_step_s2(args, dev, 1)
    tv, faces, _, _ = make_s1_inputs(4, 64, 2, seed=100, device=dev)
    return M, dev, M.build_training_step(tv, faces, args, dev, 1)


@pytest.mark.parametrize("workload", ["s1", "s2"])
def test_training_step_with_fused_layers_and_the_balance_term(workload):
    """the training steps with --fused-fc (and, for train_s2, the balance term): finite losses and gradients, and every layer's weights
    move"""
    M, dev, step = _training_step(workload)
    net = step.model["net"]
    assert sum(isinstance(m, M.Linear) for m in net.modules()) > 10
    before = {n: p.detach().clone() for n, p in net.named_parameters() if p.requires_grad}
    losses = [step() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(l)) for l in losses)
    for n, p in net.named_parameters():
        if p.requires_grad:
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
            # (train_s1's single camera multiplies its probability head by 0: its gradient is 0)
            if n.endswith("weight") and not (workload == "s1" and "prob_predictor" in n):
                assert not torch.equal(p, before[n]), n


@pytest.mark.parametrize("workload", ["s1", "s2"])
def test_training_step_with_fused_layers_replays_from_a_hip_graph(workload):
    """the same step captured whole: a replay and an eager step from one saved state leave the same loss, moments and parameters, at the
    bounds the step has without the fused layers"""
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if root not in sys.path:
        sys.path.insert(0, root)
    from tests.test_gpu_round5 import replay_equals_eager
    _, dev, step = _training_step(workload)
    replay_equals_eager(step, dev, workload + " fused", bn_eval=True)
