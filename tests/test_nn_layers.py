"""CPU tests of umr_amd.model's rewriting of layers (fuse_linears, fold_for_inference): networks that hold more than plain nn.Linear
layers compute what they computed before.  Host tensors run plain torch, so values are compared bit for bit where the operations are
the same ones."""
import copy

import pytest
import torch
from torch import nn

from umr_amd import model as M


def _same(net, rewritten, x, exact=True):
    a, b = net(x), rewritten(x)
    if exact:
        assert torch.equal(a, b)
    else:       # folded in 64 bits: the same numbers in another order of operations
        assert float((a - b).abs().max()) <= 1e-12 * max(1.0, float(a.abs().max()))


class _Doubled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


@pytest.mark.parametrize("kind", ["subclass", "weight_norm", "spectral_norm"])
def test_fused_net_keeps_the_activation_behind_a_layer_of_another_class(kind):
    """a subclass of nn.Linear, a layer with a parametrization (torch gives it a class of its own): left alone, with its LeakyReLU"""
    torch.manual_seed(0)
    make = {"subclass": lambda: _Doubled(5, 6), "weight_norm": lambda: nn.utils.parametrizations.weight_norm(nn.Linear(5, 6)),
            "spectral_norm": lambda: nn.utils.parametrizations.spectral_norm(nn.Linear(5, 6))}[kind]
    net = nn.Sequential(make(), nn.LeakyReLU(0.2), nn.Linear(6, 4), nn.LeakyReLU(0.1)).eval()
    fused = M.fuse_linears(copy.deepcopy(net))
    assert type(fused[0]) is type(net[0]) and type(fused[1]) is nn.LeakyReLU
    assert type(fused[2]) is M.Linear and fused[2].activation == "leaky_relu" and type(fused[3]) is nn.Identity
    _same(net, fused, torch.randn(7, 5))


def test_fused_net_applies_no_activation_to_a_layers_other_uses():
    """one layer in several places, with a LeakyReLU behind it in some of them: each place keeps its own activation"""
    torch.manual_seed(1)
    layer = nn.Linear(5, 5)
    for net in (nn.Sequential(layer, nn.LeakyReLU(0.2), layer), nn.Sequential(layer, nn.LeakyReLU(0.2), layer, nn.LeakyReLU(0.4)),
                nn.Sequential(nn.Sequential(layer, nn.LeakyReLU(0.2)), nn.Sequential(layer, nn.LeakyReLU(0.2))),
                nn.Sequential(nn.Sequential(layer, nn.LeakyReLU(0.2)), nn.ModuleDict(dict(other=layer))["other"])):
        net = copy.deepcopy(net)
        _same(net, M.fuse_linears(copy.deepcopy(net)), torch.randn(7, 5))
    inner = nn.Sequential(nn.Linear(5, 5), nn.LeakyReLU(0.2))               # a block in several places: fused once, the same everywhere
    net = nn.Sequential(inner, inner)
    fused = M.fuse_linears(copy.deepcopy(net))
    assert fused[1][0].activation == "leaky_relu"
    _same(net, fused, torch.randn(7, 5))


class _Skips(nn.Sequential):
    def forward(self, x):                                                   # another order than a Sequential's
        return self[1](x) + self[0](x)


def test_fused_net_leaves_a_sequential_with_a_forward_of_its_own():
    torch.manual_seed(2)
    net = _Skips(nn.Linear(5, 5), nn.LeakyReLU(0.2))
    _same(net, M.fuse_linears(copy.deepcopy(net)), torch.randn(7, 5))


def test_fused_net_keeps_what_hooks_see():
    """a hook on a layer's output or its gradient sees the product, not the activation; a hook on the LeakyReLU still runs"""
    torch.manual_seed(3)
    for where, hook in ((0, "register_forward_hook"), (0, "register_full_backward_hook"), (1, "register_forward_hook"),
                        (1, "register_forward_pre_hook"), (1, "register_full_backward_hook"), (1, "register_full_backward_pre_hook")):
        seen = []
        net = nn.Sequential(nn.Linear(5, 6), nn.LeakyReLU(0.2))
        plain = copy.deepcopy(net)
        for m in (plain, net):
            getattr(m[where], hook)(lambda mod, *a: seen.append([t.detach().clone() for v in a for t in (v if isinstance(v, tuple) else (v,)) if t is not None]))
        fused = M.fuse_linears(net)
        x = torch.randn(7, 5)
        for m in (plain, fused):
            m(x.clone().requires_grad_(True)).square().sum().backward()
        assert len(seen) == 2, hook
        assert len(seen[0]) == len(seen[1]) and all(torch.equal(a, b) for a, b in zip(*seen)), hook


@pytest.mark.parametrize("slope", [-0.25, float("nan")])
def test_fused_net_keeps_a_leaky_relu_that_the_operator_refuses(slope):
    """linear_act takes slopes >= 0: the sign of its output has to be that of the pre-activation"""
    torch.manual_seed(4)
    net = nn.Sequential(nn.Linear(5, 6), nn.LeakyReLU(slope))
    fused = M.fuse_linears(copy.deepcopy(net))
    assert fused[0].activation == "none" and type(fused[1]) is nn.LeakyReLU
    x = torch.randn(7, 5)
    assert torch.equal(torch.nan_to_num(net(x)), torch.nan_to_num(fused(x)))


# ---------------------------------------------------------------------------------------------- fold_for_inference
def _normed(n, **kw):
    bn = nn.BatchNorm1d(n, **kw).double()
    if bn.running_mean is not None:
        bn.running_mean.normal_(0, 0.3), bn.running_var.uniform_(0.5, 2.0)
    if bn.weight is not None:
        bn.weight.data.uniform_(0.5, 1.5), bn.bias.data.normal_(0, 0.1)
    return bn


@pytest.mark.parametrize("kind", ["subclass", "weight_norm", "spectral_norm"])
def test_folded_net_leaves_a_layer_of_another_class(kind):
    torch.manual_seed(5)
    make = {"subclass": lambda: _Doubled(5, 6), "weight_norm": lambda: nn.utils.parametrizations.weight_norm(nn.Linear(5, 6)),
            "spectral_norm": lambda: nn.utils.parametrizations.spectral_norm(nn.Linear(5, 6))}[kind]
    net = nn.Sequential(make().double(), _normed(6), nn.LeakyReLU(0.2)).eval()
    _same(net, M.fold_for_inference(net), torch.randn(7, 5).double(), exact=False)


def test_folded_net_folds_each_place_of_a_shared_layer_by_itself():
    """one layer, or one weight, in front of two batch norms"""
    torch.manual_seed(6)
    x = torch.randn(7, 5).double()
    layer = nn.Linear(5, 5).double()
    net = nn.Sequential(layer, _normed(5), nn.LeakyReLU(0.2), layer, _normed(5)).eval()
    _same(net, M.fold_for_inference(net), x, exact=False)
    tied = nn.Linear(5, 5).double()
    tied.weight, tied.bias = layer.weight, layer.bias
    for other in (tied, nn.Sequential(tied, nn.LeakyReLU(0.1))):             # ... or alone
        net = nn.Sequential(layer, _normed(5), nn.LeakyReLU(0.2), other, layer).eval()
        _same(net, M.fold_for_inference(net), x, exact=False)
    inner = nn.Sequential(layer, _normed(5))                                # a block in two places
    net = nn.Sequential(inner, nn.LeakyReLU(0.2), inner).eval()
    _same(net, M.fold_for_inference(net), x, exact=False)


def test_folded_net_keeps_a_batch_norm_that_has_no_fixed_map():
    """no bias, no affine map: folded all the same; statistics of the batch, of other dimensions than the layer's outputs: kept"""
    torch.manual_seed(7)
    x = torch.randn(7, 5).double()
    for bias, kw in ((False, {}), (True, dict(affine=False)), (False, dict(affine=False))):
        net = nn.Sequential(nn.Linear(5, 6, bias=bias).double(), _normed(6, **kw), nn.LeakyReLU(0.2)).eval()
        folded = M.fold_for_inference(net)
        assert len(folded) == 2
        _same(net, folded, x, exact=False)
    net = nn.Sequential(nn.Linear(5, 6).double(), _normed(6, track_running_stats=False)).eval()
    _same(net, M.fold_for_inference(net), x)
    net = nn.Sequential(nn.Linear(5, 6).double(), _normed(3)).eval()         # [B, 3, 5]: a batch norm over the middle dimension
    _same(net, M.fold_for_inference(net), torch.randn(7, 3, 5).double())


def test_folded_net_leaves_hooked_layers_and_sequentials_with_a_forward_of_their_own():
    torch.manual_seed(8)
    x = torch.randn(7, 5).double()
    for where in (0, 1):
        net = nn.Sequential(nn.Linear(5, 6).double(), _normed(6), nn.LeakyReLU(0.2)).eval()
        net[where].register_forward_hook(lambda mod, inp, out: out + 1)
        _same(net, M.fold_for_inference(net), x)
    net = _Skips(nn.Linear(5, 5), _normed(5)).double().eval()
    _same(net, M.fold_for_inference(net), x)


# ---------------------------------------------------------------------------------------------- the cameras' three layers
def _predictor(seed=9):
    torch.manual_seed(seed)
    net = M.MultiCamPredictor(12, 4)
    for m in net.modules():
        if isinstance(m, nn.Linear):
            m.weight.data.normal_(0, 0.3)
        if isinstance(m, nn.BatchNorm1d):
            m.running_mean.normal_(0, 0.3), m.running_var.uniform_(0.5, 2.0)
    return net.double().eval()


def _same_cameras(net, folded, feat):
    outs = []
    for m in (net, folded):
        torch.manual_seed(5)
        outs.append(m(feat, with_logits=True))
    for a, b in zip(*outs):
        assert a.dtype == b.dtype and float((a - b).abs().max()) <= 1e-7 * max(1.0, float(a.abs().max()))


def test_cameras_that_differ_from_each_other_stay_apart():
    """another slope, another scale, a layer of another class, a hook, another stack, something that is not a Camera: what three layers for
    all cheaply cannot hold; and a predictor that is folded already"""
    feat = torch.randn(6, 12).double()

    def slope(net):
        net.camera_predictor[2].fc_layer[0][2] = nn.LeakyReLU(0.5)

    def subclass(net):
        old, new = net.camera_predictor[1].prob_predictor, _Doubled(12, 1).double()
        new.load_state_dict(old.state_dict())
        net.camera_predictor[1].prob_predictor = new

    def hook(net):
        net.camera_predictor[3].trans_predictor.pred_layer.register_forward_hook(lambda m, i, o: o + 1)

    def no_batch_norm(net):
        net.camera_predictor[0].fc_layer = M.fc_stack(12, 12, 3).double().eval()

    def another_norm(net):
        net.camera_predictor[0].fc_layer[1][1] = _normed(12, track_running_stats=False)

    def wrapped(net):
        net.camera_predictor[0] = nn.Sequential(net.camera_predictor[0])
    for change in (lambda net: None, slope, subclass, hook, no_batch_norm, another_norm, wrapped):
        net = _predictor()
        change(net)
        _same_cameras(net, M.fold_for_inference(net), feat)
    folded = M.fold_for_inference(_predictor())
    assert isinstance(folded.camera_predictor, M.FoldedCameras)
    _same_cameras(folded, M.fold_for_inference(folded), feat)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64], ids=str)
def test_folded_cameras_keep_the_networks_type_and_scales(dtype):
    """outputs in the type of the network, before and after a conversion; scale_lr and scale_bias are constants of that type's arithmetic, as
    in Camera; cameras with scales of their own stay apart"""
    net = _predictor()
    for k, c in enumerate(net.camera_predictor):
        c.scale_lr, c.scale_bias = 0.05 + 0.01 * k, 1.0 / 3
    _same_cameras(net, M.fold_for_inference(net), torch.randn(6, 12).double())
    for c in net.camera_predictor:
        c.scale_lr = 0.05
    feat = torch.randn(6, 12).to(dtype)
    before, after = M.fold_for_inference(copy.deepcopy(net).to(dtype)), M.fold_for_inference(net).to(dtype)
    for folded in (before, after):
        outs = [m(feat, with_logits=True) for m in (copy.deepcopy(net).to(dtype), folded)]
        for i in (3, 4, 5):
            a, b = outs[0][i], outs[1][i]
            assert a.dtype == b.dtype == dtype
            if dtype is torch.float64:                                       # (sums in another order)
                assert float((a - b).abs().max()) <= 1e-13 * max(1.0, float(a.abs().max()))


@pytest.mark.parametrize("after", [nn.Dropout(0.5, inplace=True), nn.ReLU(inplace=True)], ids=str)
def test_fused_net_keeps_a_leaky_relu_whose_output_the_next_module_changes_in_place(after):
    """on the GPU the fused layer keeps its output for the backward call, so changing it raises; nn.LeakyReLU keeps its input"""
    net = nn.Sequential(nn.Linear(5, 6), nn.LeakyReLU(0.2), copy.deepcopy(after))
    fused = M.fuse_linears(copy.deepcopy(net))
    assert fused[0].activation == "none" and type(fused[1]) is nn.LeakyReLU
    net[2].inplace = False
    assert M.fuse_linears(net)[0].activation == "leaky_relu"


def test_a_forward_of_an_instances_own_is_respected():
    """module.forward replaced on the instance, as offloading wrappers do it: on a layer, its LeakyReLU, the Sequential, a camera"""
    torch.manual_seed(10)
    x = torch.randn(7, 5).double()

    def replaced(m):
        old = m.forward
        m.forward = lambda v: old(v) + 1
        return m
    for where in (0, 1, 2, None):
        def build():
            torch.manual_seed(11)
            net = nn.Sequential(nn.Linear(5, 5).double(), nn.LeakyReLU(0.2), _normed(5)).eval()
            if where is None:
                return replaced(net)
            replaced(net[where])
            return net
        assert torch.equal(build()(x), M.fuse_linears(build())(x)), where

        def folding():
            torch.manual_seed(12)
            net = nn.Sequential(nn.Linear(5, 5).double(), _normed(5), nn.LeakyReLU(0.2)).eval()
            replaced(net if where is None else net[where])
            return net
        assert torch.allclose(folding()(x), M.fold_for_inference(folding())(x), rtol=0, atol=1e-12), where
    net = _predictor()
    replaced(net.camera_predictor[1])
    _same_cameras(net, M.fold_for_inference(net), torch.randn(6, 12).double())
