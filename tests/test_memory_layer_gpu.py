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


def off_by_one(t):
    """The same numbers contiguous, one element past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    view = flat[1:1 + t.numel()].view(t.shape)
    view.copy_(t.detach())
    assert view.data_ptr() % 16 != 0 and view.is_contiguous()
    return view


@gpu
def test_a_norm_whose_parameters_are_views_of_a_flat_buffer():
    def flatten(m):
        for name in ("weight", "bias"):
            p = getattr(m.o_norm, name)
            if p.is_cuda:
                setattr(m.o_norm, name, nn.Parameter(off_by_one(p)))
    layer = layer_of()
    dev = layer.cuda()
    flatten(dev)
    assert dev.o_norm.weight.data_ptr() % 16 != 0
    ref = copy.deepcopy(layer).double().cpu()
    x = R.hashed_uniform("ly.x", (2, 9, 96), 1.0)
    s = R.hashed_uniform("ly.s", (2, 2, 64, 64), 0.2)
    sd = off_by_one(s.cuda()).requires_grad_()
    sr = s.double().requires_grad_()
    got, want = dev(x.cuda(), sd), ref(x.double(), sr)
    assert rel(got[0], want[0]) < 1e-4 and rel(got[1], want[1]) < 1e-4
    grads = torch.autograd.grad(got[0].sum() + got[1].pow(2).sum(), [dev.o_norm.weight, dev.o_norm.bias, sd])
    wanted = torch.autograd.grad(want[0].sum() + want[1].pow(2).sum(), [ref.o_norm.weight, ref.o_norm.bias, sr])
    for g, w in zip(grads, wanted):
        assert rel(g, w) < 1e-4


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_and_operands_off_a_16_byte_boundary(dtype):
    """The differentiable operators take gradients, states and rows wherever they lie."""
    from vit_amd import module_ops, ops
    B, L, H, hd = 2, 70, 2, 64
    q, k, v = (R.hashed_uniform(f"of.{n}", (B, L, H, hd), 0.1).to(dtype).cuda() for n in "qkv")
    a, b = R.hashed_uniform("of.a", (B, L, H), 0.2, 0.8).cuda(), R.hashed_uniform("of.b", (B, L, H), 0.5, 0.5).cuda()
    s = R.hashed_uniform("of.s", (B, H, hd, hd), 0.4).cuda()
    go, gs = R.hashed_uniform("of.go", (B, L, H, hd), 1.0).to(dtype).cuda(), R.hashed_uniform("of.gs", s.shape, 0.5).cuda()
    results = []
    for state, d_out, d_state in ((s, go, gs), (off_by_one(s), off_by_one(go), off_by_one(gs))):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, a, b, state)]
        results.append(torch.autograd.grad(module_ops.gated_delta(*leaves), leaves, (d_out, d_state)))
    assert all(torch.equal(x, y) for x, y in zip(*results))
    rows = [R.hashed_uniform(f"of.r{n}", (9, 96), 1.0).to(dtype).cuda() for n in range(3)]
    scale, shift = (R.hashed_uniform(f"of.{n}", (96,), 0.5, 1.0).cuda() for n in ("gamma", "beta"))
    dy, results = R.hashed_uniform("of.dy", (9, 96), 1.0).to(dtype).cuda(), []
    for move in (lambda t: t, off_by_one):
        leaves = [move(t).detach().requires_grad_() for t in (*rows, scale, shift)]
        y = module_ops.gated_layernorm(*leaves)
        results.append([y, *torch.autograd.grad(y, leaves, move(dy))])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    if dtype == torch.bfloat16:                                # 8 bytes are enough for bf16 rows, the gradient's too
        flat = torch.empty(go.numel() + 4, dtype=dtype, device="cuda")
        moved = flat[4:].view(go.shape).copy_(go)
        for x, y in zip(ops.gated_delta_bwd(moved, gs, q, k, v, a, b, s), ops.gated_delta_bwd(go, gs, q, k, v, a, b, s)):
            assert torch.equal(x, y)
