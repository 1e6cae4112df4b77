"""What is measured of the network-side operators, and their plain forms.

  linear_act        y = act(x W^T + b) + r        the fully connected layers of MeshNet (model.fc / fc_stack, the predictors)
  heads_linear_act  the same for G heads at once: x [.., G, K], W [G, N, K]      the K camera predictors of MultiCamPredictor
  balance_loss      E sum_e f_e P_e over E choices, with the count of every choice     the camera hypotheses of a train_s2 step

`own` False: elementary torch operations in 32 bits, rounded once at the end.  `own` True: the calls a user makes of
umr_amd.functional, gradients through torch.autograd."""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = ("none", "relu", "leaky_relu", "tanh", "gelu", "silu")


def _linear(name, rows, n, k, dtype="fp32", heads=0, act="none", slope=0.0, bias=True, residual="none", pad=0, train=False):
    """rows x k times (n x k)^T; heads > 0: that many of them.  residual: none / full / row (one row for all).  pad: how many
    elements the rows of x are longer than k in memory."""
    c = dict(op="linear", rows=rows, n=n, k=k, dtype=dtype, heads=heads, act=act, slope=slope, bias=bias, residual=residual, pad=pad, train=train)
    return dict(c, name=name) if name else c


def _balance(name, rows, experts, top, dtype="fp32", mask="none", train=True):
    """mask: none / rows (a tenth of the rows is padding and holds NaN) / choices (some logits are -inf or the type's lowest
    value, some rows have nothing left) / both."""
    c = dict(op="balance", rows=rows, experts=experts, top=top, dtype=dtype, mask=mask, train=train)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one image through a layer of the camera head (nz_feat 200, LeakyReLU 0.1): latency is everything
        _linear("head_one_image", 1, 200, 200, act="leaky_relu", slope=0.1),
        # one image through the texture encoder's second layer, batch norm folded in: 268 MB of weights for one row
        _linear("texture_fc_one_image", 1, 8192, 8192, act="leaky_relu", slope=0.2),
        # the same layer in a training step at the batch of 16 (a batch norm follows, so no activation)
        _linear("texture_fc_train", 16, 8192, 8192, train=True),
        # the encoder's first layer in a training step: a long contraction onto few columns
        _linear("encoder_fc_train", 16, 200, 4096, train=True),
        # vertex offsets of the 10 000-pair evaluation (350 latents -> 337 vertices), added to the mean shape: one row for all
        _linear("vertices_10k", 10000, 1011, 350, residual="row"),
        # odd sizes, rows longer than the layer's input, smooth activation and residual, every gradient
        _linear("odd_fp16_train", 777, 1001, 515, dtype="fp16", act="silu", residual="full", pad=13, train=True),
        # a wide layer over many feature rows in 16 bits with the residual in its epilogue: the largest product
        _linear("wide_bf16_train", 8192, 4096, 4096, dtype="bf16", act="gelu", residual="full", train=True),
        # second layer of the 8 camera predictors in a training step
        _linear("camera_heads_train", 16, 200, 200, heads=8, act="leaky_relu", slope=0.2, train=True),
        # many heads over hundreds of rows each, 16 bits
        _linear("heads_bf16_train", 333, 512, 1024, dtype="bf16", heads=32, act="silu", train=True),
        # the 8 camera hypotheses of a train_s2 batch, one sampled for each image
        _balance("hypotheses_s2", 16, 8, 1),
        # a middle size with an odd number of choices, padded rows and forbidden choices
        _balance("choices_odd", 5001, 61, 2, mask="both"),
        # many rows, 8 of 128 choices each, 16 bits, padded rows
        _balance("choices_many_bf16", 1 << 19, 128, 8, dtype="bf16", mask="rows"),
    ]


_MOST_FLOPS = 6 * 8192 * 4096 * 4096
_MOST_BYTES = 8192 * 8192 * 4 * 2


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.3:
        experts = _log(rng, 2, 512)
        return _balance(None, _log(rng, 1, (1 << 19) * 128 // max(128, experts)), experts, rng.randint(1, min(8, experts)),
                        dtype=rng.choice(["fp32", "bf16", "fp16"]) if experts <= 64 else rng.choice(["bf16", "fp16"]),
                        mask=rng.choice(["none", "rows", "choices", "both"]), train=True)
    while True:
        heads = rng.choice([0, 0, 0, _log(rng, 2, 64)])
        rows, n, k = _log(rng, 1, 10000), _log(rng, 8, 8192), _log(rng, 8, 8192)
        if rng.random() < 0.4:
            rows = rng.randint(1, 64)
        # a kinked activation's gradient jumps where the pre-activation is 0: drawn with a gradient at the sizes of MeshNet's heads only
        few = rows * n * max(heads, 1) <= 20000
        train = rng.random() < 0.6
        act = rng.choice(ACTS if few or not train else ("none", "tanh", "gelu", "silu"))
        c = _linear(None, rows, n, k, dtype=rng.choice(["fp32", "bf16", "fp16"]), heads=heads, act=act,
                    slope=rng.choice([0.01, 0.1, 0.2]) if act == "leaky_relu" else 0.0, bias=rng.random() < 0.8,
                    residual=rng.choice(["none", "full", "row"]), pad=rng.choice([0, 0, 1, 8, 13]), train=train)
        w = work(c)
        limit = _MOST_FLOPS if c["dtype"] != "fp32" else _MOST_FLOPS // 16      # (the unit does 16 times fewer 32-bit products)
        if w["flops"] <= limit and w["bytes"] <= _MOST_BYTES:
            return c


def _inputs(case, seed):
    """The inputs as (float or integer) tensors, from the seed alone."""
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed % 1000003) + 17)
    t = TYPES[case["dtype"]]
    if case["op"] == "linear":
        G, M, N, K = max(case["heads"], 1), case["rows"], case["n"], case["k"]
        # features as they leave a LeakyReLU(0.2) layer; weights that keep the variance
        x = torch.nn.functional.leaky_relu(torch.randn(M, G, K + case["pad"], device=DEV, generator=g), 0.2).to(t)[..., :K]
        w = (torch.randn(G, N, K, device=DEV, generator=g) / math.sqrt(K)).to(t)
        b = (0.1 * torch.randn(G, N, device=DEV, generator=g)).to(t) if case["bias"] else None
        r = None
        if case["residual"] != "none":
            r = torch.randn(*([M] if case["residual"] == "full" else []), G, N, device=DEV, generator=g).to(t)
        gy = torch.randn(M, G, N, device=DEV, generator=g).to(t) if case["train"] else None
        if not case["heads"]:
            x, w, b, r, gy = x[:, 0], w[0], (None if b is None else b[0]), (None if r is None else r[..., 0, :]), (None if gy is None else gy[:, 0])
        return dict(x=x, w=w, b=b, r=r, gy=gy)
    T, E, k = case["rows"], case["experts"], case["top"]
    # scores with a preference that all rows share, so that the choices are used unevenly
    z = (torch.randn(T, E, device=DEV, generator=g) + torch.randn(E, device=DEV, generator=g)).to(t)
    inds = torch.rand(T, E, device=DEV, generator=g).add_(z.float().softmax(1)).topk(k, 1).indices
    mask = None
    if case["mask"] in ("choices", "both"):
        forbidden = torch.rand(T, E, device=DEV, generator=g) < 0.1
        forbidden |= (torch.rand(T, 1, device=DEV, generator=g) < 0.02)
        low = torch.where(torch.rand(T, 1, device=DEV, generator=g) < 0.5, -math.inf, torch.finfo(t).min).to(t)
        z = torch.where(forbidden, low, z)
    if case["mask"] in ("rows", "both"):
        mask = torch.rand(T, device=DEV, generator=g) >= 0.1
        z = torch.where(mask[:, None], z, torch.tensor(math.nan, dtype=t, device=DEV))
    # the gradient that reaches the loss: a loss scale, as 16-bit training has one (the mean over the rows is tiny without it)
    g = torch.tensor(float(1 << (T.bit_length() - 1)), device=DEV)
    return dict(z=z.contiguous(), inds=inds, mask=mask, g=g)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["train"]:
        for name in ("x", "w", "b", "r", "z"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_(True)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _act(z, act, slope):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, slope * z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act, slope):
    if act == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, slope)
    if act == "tanh":
        return 1 - torch.tanh(z) ** 2
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_linear(s):
    c, t = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    heads = c["heads"] > 0
    if heads:
        x = x.transpose(0, 1).contiguous()                               # [G, M, K]
    z = torch.matmul(x, w.transpose(-1, -2).contiguous() if heads else w.t())
    if s["b"] is not None:
        z = z + (s["b"].float()[:, None] if heads else s["b"].float())
    y = _act(z, c["act"], c["slope"])
    if heads:
        y = y.transpose(0, 1)
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(t).contiguous()
    if not c["train"]:
        return y
    gy = s["gy"].float()
    dz = (gy.transpose(0, 1).contiguous() if heads else gy) * _act_slope(z, c["act"], c["slope"])
    dx = torch.matmul(dz, w)
    dw = torch.matmul(dz.transpose(-1, -2).contiguous() if heads else dz.t(), x)
    out = dict(y=y, dx=(dx.transpose(0, 1) if heads else dx).to(t).contiguous(), dw=dw.to(t))
    if s["b"] is not None:
        out["db"] = dz.sum(-2).to(t)
    if s["r"] is not None:
        out["dr"] = s["gy"] if c["residual"] == "full" else gy.sum(0).to(t)
    return out


def _plain_balance(s):
    c, z, inds, mask = s["case"], s["z"].float(), s["inds"], s["mask"]
    E, k = c["experts"], c["top"]
    m = z.amax(1, keepdim=True)
    valid = m[:, 0] != -math.inf
    if mask is not None:
        valid = valid & mask
    p = torch.exp(z - m)
    p = torch.where(valid[:, None], p / p.sum(1, keepdim=True), 0.0)
    counts = torch.zeros(E, dtype=torch.int64, device=z.device).index_add_(0, inds.reshape(-1), valid.repeat_interleave(k).long())
    n = valid.sum().clamp_min(1).double()
    f = counts.double() / (n * k)
    loss = (E * (f * (p.sum(0, dtype=torch.float64) / n)).sum()).float()
    if not c["train"]:
        return dict(loss=loss, counts=counts)
    f32 = f.float()
    dz = s["g"] * (E / n).float() * p * (f32 - (p * f32).sum(1, keepdim=True))
    return dict(loss=loss, counts=counts, dz=dz.to(s["z"].dtype))


# ---------------------------------------------------------------------------------------------- the framework's operators
def _own_linear(s):
    from umr_amd import functional as UF
    c = s["case"]
    call = UF.heads_linear_act if c["heads"] else UF.linear_act
    y = call(s["x"], s["w"], s["b"], residual=s["r"], activation=c["act"], slope=c["slope"])
    if not c["train"]:
        return y
    names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["gy"])
    return dict(dict(("d" + n, g) for n, g in zip(names, grads)), y=y.detach())


def _own_balance(s):
    from umr_amd import functional as UF
    loss, counts = UF.balance_loss(s["z"], s["inds"], s["mask"])
    if not s["case"]["train"]:
        return dict(loss=loss, counts=counts)
    dz, = torch.autograd.grad(loss, [s["z"]], s["g"])
    return dict(loss=loss.detach(), counts=counts, dz=dz)


def run(state):
    if state["case"]["op"] == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    return _own_balance(state) if own else _plain_balance(state)


# ---------------------------------------------------------------------------------------------- floor and 64-bit values
def work(case):
    if case["op"] == "linear":
        e = 4 if case["dtype"] == "fp32" else 2
        G, M, N, K = max(case["heads"], 1), case["rows"], case["n"], case["k"]
        x, w, y, col = G * M * K * e, G * N * K * e, G * M * N * e, G * N * e
        b = col if case["bias"] else 0
        r = {"none": 0, "full": y, "row": col}[case["residual"]]
        if not case["train"]:
            return {"bytes": x + w + b + r + y, "flops": 2 * G * M * N * K}
        # reads x w b r gy, writes y dx dw db (dr of a full residual is gy itself)
        return {"bytes": 2 * (x + w + b + y) + r + (col if case["residual"] == "row" else 0), "flops": 6 * G * M * N * K}
    e = 4 if case["dtype"] == "fp32" else 2
    T, E, k = case["rows"], case["experts"], case["top"]
    data = T * E * e
    rest = T * k * 8 + (T if case["mask"] in ("rows", "both") else 0) + E * 8 + 4
    return {"bytes": data * (2 if case["train"] else 1) + rest, "flops": T * E * (9 if case["train"] else 4)}


def exact(case, seed):
    """From the definitions, in float64, the gradients by torch.autograd on them."""
    s = _inputs(case, seed)
    F = torch.nn.functional
    if case["op"] == "linear":
        leaf = {n: s[n].double().requires_grad_(case["train"]) for n in ("x", "w", "b", "r") if s[n] is not None}
        if case["heads"]:
            outs = [F.linear(leaf["x"][:, g], leaf["w"][g], leaf["b"][g] if "b" in leaf else None) for g in range(case["heads"])]
            y = torch.stack(outs, 1)
        else:
            y = F.linear(leaf["x"], leaf["w"], leaf.get("b"))
        y = {"none": lambda v: v, "relu": F.relu, "leaky_relu": lambda v: F.leaky_relu(v, case["slope"]), "tanh": torch.tanh,
             "gelu": F.gelu, "silu": F.silu}[case["act"]](y)
        if "r" in leaf:
            y = y + leaf["r"]
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, list(leaf.values()), s["gy"].double())
        return dict(dict(("d" + n, g) for n, g in zip(leaf, grads)), y=y.detach())
    E, k = case["experts"], case["top"]
    z = s["z"].double()
    keep = ~(z == -math.inf).all(1)
    if s["mask"] is not None:
        keep &= s["mask"]
    rows = keep.nonzero()[:, 0]
    picked = s["inds"][rows].reshape(-1)
    counts = torch.bincount(picked, minlength=E)
    leaf = z[rows].requires_grad_(True)
    if not len(rows):
        zero = torch.zeros((), dtype=torch.float64, device=z.device)
        return dict(loss=zero, counts=counts, dz=torch.zeros_like(z)) if case["train"] else dict(loss=zero, counts=counts)
    usage = torch.softmax(leaf, 1).mean(0)
    loss = E * torch.dot(counts.double() / picked.numel(), usage)
    if not case["train"]:
        return dict(loss=loss.detach(), counts=counts)
    dz = torch.zeros_like(z)
    dz[rows] = torch.autograd.grad(loss, leaf, s["g"].double())[0]
    return dict(loss=loss.detach(), counts=counts, dz=dz)
