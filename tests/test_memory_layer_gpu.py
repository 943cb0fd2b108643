"""GPU: the memory layer with a graph is still a module made of modules: hooks fire, replaced parts are the ones that run.

The layer is compared with a 64-bit copy of itself on the host: 1e-4 of a result's 2-norm is what f32 products of up to
256 terms, eight layers deep, may lose (2^-24 * 1024 = 6e-5).  A norm takes the mean away: an input of size m that is held in f32
is off by half a step, 2^-24 m, and the norm divides that by sqrt(var + eps) as it does the deviation itself, so results and
gradients behind it may also lose the ratio of the two, which the host copy knows (6e-8 where the mean is about zero; a
hook that adds 1 to values of 1e-4 makes it 3e-4)."""
import copy

import pytest
import torch
from torch import nn

from oracle import ref_cpu as R

gpu = pytest.mark.gpu


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def layer_of(dim=96, heads=2, hd=64):
    from vit_amd import surgical_world_model as swm
    layer = swm.GatedDeltaLayer(dim, num_heads=heads, head_dim=hd)
    P = R.fill_state_dict_({f"ly.{k}": v for k, v in layer.state_dict().items()})
    layer.load_state_dict({k[3:]: v for k, v in P.items()})
    return layer.eval()


def against_the_host(layer, change, L=70):
    """`change` made to a device copy and a 64-bit host copy of the layer: outputs and every gradient alike."""
    ref, dev = copy.deepcopy(layer).double(), copy.deepcopy(layer).cuda()
    for m in (ref, dev):
        change(m)
    ref.double()
    dev.cuda()
    lost = []

    def conditioning(mod, args, out):
        held = args[0].detach()
        spread = (held.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        lost.append(((2.0 ** -24 * held / spread).norm() / ((held - held.mean(-1, keepdim=True)) / spread).norm()).item())

    ref.o_norm.register_forward_hook(conditioning)
    x = R.hashed_uniform("ly.x", (2, L, layer.hidden_size), 1.0)
    go = R.hashed_uniform("ly.go", x.shape, 1.0)
    xr, xd = x.double().requires_grad_(), x.cuda().requires_grad_()
    want, got = ref(xr), dev(xd)
    tol = 1e-4 + lost[0]
    assert rel(got[0], want[0]) < tol and rel(got[1], want[1]) < 1e-4
    wanted = torch.autograd.grad(want[0], [xr, *ref.parameters()], go.double(), allow_unused=True)
    grads = torch.autograd.grad(got[0], [xd, *dev.parameters()], go.cuda(), allow_unused=True)
    for name, g, w in zip(["x"] + [n for n, _ in ref.named_parameters()], grads, wanted):
        assert (g is None) == (w is None), name
        assert g is None or rel(g, w) < tol, name


class ScaledNorm(nn.LayerNorm):
    def forward(self, x):
        return 3.0 * super().forward(x)


def norm_without_bias(m):
    m.o_norm = nn.LayerNorm(m.num_heads * m.head_dim, bias=False)


def norm_without_parameters(m):
    m.o_norm = nn.LayerNorm(m.num_heads * m.head_dim, elementwise_affine=False)


def norm_of_a_subclass(m):
    old, m.o_norm = m.o_norm, ScaledNorm(m.num_heads * m.head_dim)
    m.o_norm.load_state_dict(old.state_dict())


def norm_with_its_own_forward(m):
    m.o_norm.forward = lambda x: 2.0 * x


def norm_over_heads(m):
    m.o_norm = nn.Sequential(nn.Unflatten(-1, (m.num_heads, m.head_dim)), nn.LayerNorm(m.head_dim), nn.Flatten(-2))


def no_norm(m):
    m.o_norm = nn.Identity()


def other_activation(m):
    m.silu = nn.Softplus()


def scaling_hook(m):
    m.o_norm.register_forward_hook(lambda mod, args, out: 2.0 * out)


def scaling_pre_hook(m):
    m.o_norm.register_forward_pre_hook(lambda mod, args: (args[0] * 2.0 + 1.0,))


def gradient_hook(m):
    m.o_norm.register_full_backward_hook(lambda mod, grad_in, grad_out: (grad_in[0] * 0.5,))


def activation_hook(m):
    m.silu.register_forward_hook(lambda mod, args, out: out + 0.25)


@gpu
@pytest.mark.parametrize("change", [lambda m: None, norm_without_bias, norm_without_parameters, norm_of_a_subclass,
                                    norm_with_its_own_forward, norm_over_heads, no_norm, other_activation, scaling_hook,
                                    scaling_pre_hook, gradient_hook, activation_hook])
def test_parts_of_the_layer_are_the_ones_that_run(change):
    against_the_host(layer_of(), change)


@gpu
def test_hooks_of_all_modules_see_the_norm():
    layer, seen = layer_of().cuda(), []
    x = R.hashed_uniform("ly.x", (1, 5, 96), 1.0).cuda().requires_grad_()
    handle = nn.modules.module.register_module_forward_hook(lambda mod, args, out: seen.append(type(mod).__name__))
    try:
        layer(x)
    finally:
        handle.remove()
    assert "LayerNorm" in seen
