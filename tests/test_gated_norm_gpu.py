"""GPU: LayerNorm((o * gate) * silu(g)) with its gradients, rows of any width, against 64 bits.

Tolerances.  f32 arithmetic: a row's mean and variance are sums of at most 4096 terms held by at most 16 elements per lane
and added pairwise across lanes, the logistic is good to a few steps of 2^-24; 1e-5 (168 half steps) of the result's size
covers a row's results, and 1e-5 of the 2-norm the column sums.  bf16 results are rounded once, by at most 2^-8."""
import pytest
import torch

from oracle import ref_cpu as R

gpu = pytest.mark.gpu


def inputs(M, D, dtype):
    o, gate, g = (R.hashed_uniform(f"gn.{n}", (M, D), s).to(dtype) for n, s in (("o", 1.5), ("gate", 1.0), ("g", 4.0)))
    return o, gate, g, R.hashed_uniform("gn.gamma", (D,), 0.5, 1.0), R.hashed_uniform("gn.beta", (D,), 0.3)


def formula(o, gate, g, gamma, beta, eps=1e-5):
    x = o * gate * (g * torch.sigmoid(g))
    return torch.nn.functional.layer_norm(x, x.shape[-1:], gamma, beta, eps)


def close(got, want, dtype, name):
    err, half = (got.double().cpu() - want).abs(), 2.0 ** -8 if got.dtype == torch.bfloat16 else 0.0
    scale = want.abs().amax(-1, keepdim=True) if want.dim() > 1 else want.abs().max()
    assert torch.isfinite(got).all(), name
    assert bool((err <= half * want.abs() * (1 + 1e-3) + 4e-5 * (want.abs() + scale) + 1e-7).all()), (name, err.max().item())
    if half == 0.0:
        assert err.norm() <= 1e-5 * want.norm() + 1e-7, (name, (err.norm() / want.norm()).item())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,D", [(1, 4), (3, 60), (5, 256), (197, 384), (2, 516), (9, 1024), (4099, 1024), (7, 1028), (33, 2048),
                                 (3, 2052), (1000, 4096)])
def test_forward_and_gradients(M, D, dtype):
    from vit_amd import module_ops
    args = inputs(M, D, dtype)
    dy = R.hashed_uniform("gn.dy", (M, D), 1.0).to(dtype)
    ref = [t.double().requires_grad_() for t in args]
    want = formula(*ref)
    grads = torch.autograd.grad(want, ref, dy.double())
    dev = [t.cuda().requires_grad_() for t in args]
    y = module_ops.gated_layernorm(*dev, 1e-5)
    assert y.dtype == dtype
    close(y.detach(), want.detach(), dtype, "y")
    for name, x, w in zip(("o", "gate", "g", "gamma", "beta"), torch.autograd.grad(y, dev, dy.cuda()), grads):
        close(x, w, dtype, name)


@gpu
def test_gradients_against_differences():
    """Central differences of the 64-bit formula along the signs of the kernel's gradients: the quotient is then the 1-norm
    of the gradient, off by h^2 of the third derivative."""
    from vit_amd import module_ops
    args = inputs(6, 96, torch.float32)
    dy = R.hashed_uniform("gn.dy", (6, 96), 1.0)
    dev = [t.cuda().requires_grad_() for t in args]
    got = torch.autograd.grad(module_ops.gated_layernorm(*dev, 1e-5), dev, dy.cuda())
    h = 1e-5
    for i, g in enumerate(got):
        d = torch.sign(g.double().cpu())
        at = [t.double() for t in args]
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        quotient = ((formula(*up) - formula(*down)) * dy.double()).sum().item() / (2 * h)
        slope = (g.double().cpu() * d).sum().item()
        assert abs(quotient - slope) <= 1e-4 * abs(slope), (i, quotient, slope)


@gpu
def test_a_row_does_not_depend_on_its_neighbours_and_repeats_exactly():
    from vit_amd import ops
    args = [t.cuda() for t in inputs(3001, 1024, torch.float32)]
    dy = R.hashed_uniform("gn.dy", (3001, 1024), 1.0).cuda()
    y, mean, rstd = ops.gated_layernorm_fwd(*args)
    one = ops.gated_layernorm_fwd(*(t[70:73].contiguous() for t in args[:3]), *args[3:])[0]
    assert torch.equal(y[70:73], one)
    assert torch.equal(y, ops.gated_layernorm_fwd(*args, keep=False)[0])
    a, b = (ops.gated_layernorm_bwd(dy, *args[:4], mean, rstd) for _ in range(2))
    assert all(torch.equal(x, z) for x, z in zip(a, b))


@gpu
def test_strided_views_graph_replays_and_large_arguments():
    from vit_amd import module_ops, ops
    o, gate, g, gamma, beta = (t.cuda() for t in inputs(64, 512, torch.float32))
    wide = torch.cat([o, gate, g], 1)
    views = [wide[:, i * 512:(i + 1) * 512] for i in range(3)]          # the differentiable form takes any strides
    assert torch.equal(module_ops.gated_layernorm(*views, gamma, beta), module_ops.gated_layernorm(o, gate, g, gamma, beta))
    g = g * 1e3                                                          # silu far outside exp's range: 0 or g
    want = formula(*(t.double().cpu() for t in (o, gate, g, gamma, beta)))
    close(module_ops.gated_layernorm(o, gate, g, gamma, beta), want, torch.float32, "large")
    dy = torch.ones_like(o)

    def step():
        y, mean, rstd = ops.gated_layernorm_fwd(o, gate, g, gamma, beta)
        return [y, *ops.gated_layernorm_bwd(dy, o, gate, g, gamma, mean, rstd)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        o.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        for x, z in zip(held, step()):
            assert torch.equal(x, z), i


@gpu
def test_refusals():
    from vit_amd import ops
    o, gate, g, gamma, beta = (t.cuda() for t in inputs(8, 64, torch.float32))
    for bad in ((o[:, :63].contiguous(), gate[:, :63].contiguous(), g[:, :63].contiguous(), gamma[:63], beta[:63]),
                (o, gate.bfloat16(), g, gamma, beta), (o, gate[:4], g, gamma, beta), (o.double(), gate.double(), g.double(), gamma, beta),
                (o, gate, g, gamma[:32], beta), (o, gate, g, gamma.bfloat16(), beta), (o.t(), gate.t(), g.t(), gamma, beta),
                (o[:0], gate[:0], g[:0], gamma, beta)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.gated_layernorm_fwd(*bad)
    wide = [torch.zeros(2, 4100, device="cuda")] * 3
    with pytest.raises(RuntimeError):
        ops.gated_layernorm_fwd(*wide, torch.ones(4100, device="cuda"), torch.ones(4100, device="cuda"))
    _, mean, rstd = ops.gated_layernorm_fwd(o, gate, g, gamma, beta)
    with pytest.raises(ValueError):
        ops.gated_layernorm_bwd(o, o, gate, g, gamma, mean[:4], rstd)
    # no broadcasting between the three, and no gradient of the gradient
    from vit_amd import module_ops
    with pytest.raises(ValueError):
        module_ops.gated_layernorm(o, gate[:1], g, gamma, beta)


def test_refusals_without_a_gpu():
    from vit_amd import _lib, ops
    args = inputs(4, 64, torch.float32)
    with pytest.raises(_lib.VitAmdError):
        ops.gated_layernorm_fwd(*args)
    with pytest.raises(_lib.VitAmdError):
        ops.gated_layernorm_bwd(args[0], *args[:4], torch.zeros(4), torch.zeros(4))


@pytest.mark.parametrize("M,D", [(0, 64), (1 << 26, 64), (1 << 24, 1028), (4, 66), (4, 4100)])
def test_sizes_that_no_launch_can_take_are_refused(M, D):
    """Before anything is launched: the addresses are never looked at."""
    from vit_amd import _lib
    lib = _lib.load()
    assert lib.va_gated_layernorm_fwd(16, 16, 16, 0, 16, 16, 16, None, None, M, D, 1e-5, None) != 0
    assert lib.va_gated_layernorm_bwd(*[16] * 4, 0, *[16] * 9, M, D, None) != 0


@gpu
def test_second_derivatives():
    """From the formula in torch, f32; 1e-4 as for sums within sums good to 1e-5 each."""
    from vit_amd import module_ops
    args, dy = inputs(7, 96, torch.float32), R.hashed_uniform("gn.dy", (7, 96), 1.0)

    def second(f, leaves, dy):
        leaves = [t.requires_grad_() for t in leaves]
        first = torch.autograd.grad((f(*leaves, 1e-5) * dy).sum(), leaves, create_graph=True)
        return torch.autograd.grad(sum((g * (i + 1)).pow(2).sum() for i, g in enumerate(first)), leaves[:4])

    want = second(formula, [t.double() for t in args], dy.double())
    dev = [t.cuda() for t in args]
    for g, w in zip(second(module_ops.gated_layernorm, dev, dy.cuda()), want):
        assert (g.double().cpu() - w).norm() <= 1e-4 * w.norm()
    y, seeds = module_ops.gated_layernorm(*dev, 1e-5), torch.stack([dy, dy.flip(0)]).cuda()
    many = torch.autograd.grad(y, dev, seeds, is_grads_batched=True, retain_graph=True)
    for i in range(2):
        for a, b in zip(many, torch.autograd.grad(y, dev, seeds[i], retain_graph=True)):
            assert (a[i] - b).norm() <= 1e-4 * b.norm()


def test_where_torch_must_see_every_operation():
    from vit_amd import module_ops
    assert not module_ops.by_torch_alone()
    torch.set_autocast_enabled("cuda", True)
    try:
        assert module_ops.by_torch_alone()
    finally:
        torch.set_autocast_enabled("cuda", False)
    with torch.autograd.forward_ad.dual_level():
        assert module_ops.by_torch_alone()
    seen = []
    torch.func.vmap(lambda x: (seen.append(module_ops.by_torch_alone()), x)[1])(torch.zeros(2))
    assert seen == [True] and not module_ops.by_torch_alone()
