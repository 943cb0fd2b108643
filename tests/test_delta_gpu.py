"""GPU: the gated delta rule in its chunked form (forward, gradients) and for single tokens, against the token-by-token
recurrence in 64 bits.

Tolerances.  The kernels' products and states are f32: a value is a sum of at most a few hundred products, each addition
off by at most 2^-24 of a partial sum, so the 2-norm of the error stays below 168 * 2^-24 = 1e-5 of the result's.  Results
of type bf16 are rounded once, by at most 2^-8 of their value."""
import pytest
import torch

from oracle import ref_cpu as R

gpu = pytest.mark.gpu
F32_REL = 1e-5
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def inputs(B, L, H, hd, dtype, state, seed="d", unit=False):
    """Keys and queries of norm below one per head (a whole row is normalised, as the layer does) or of norm one."""
    F = torch.nn.functional
    q, k = (R.hashed_uniform(f"{seed}.{n}", (B, L, H * hd), 1.0, 0.3) for n in "qk")
    if unit:
        q, k = (F.normalize(x.view(B, L, H, hd), dim=-1) for x in (q, k))
    else:
        q, k = (F.normalize(x, dim=-1).view(B, L, H, hd) for x in (q, k))
    v = R.hashed_uniform(f"{seed}.v", (B, L, H, hd), 1.0)
    a = R.hashed_uniform(f"{seed}.a", (B, L, H), 0.2, 0.8)
    b = R.hashed_uniform(f"{seed}.b", (B, L, H), 0.5, 0.5)
    s = R.hashed_uniform(f"{seed}.s", (B, H, hd, hd), 0.4) if state else None
    return q.to(dtype), k.to(dtype), v.to(dtype), a, b, s


def recurrence(q, k, v, a, b, s):
    """Token by token, in the inputs' 64 bits."""
    B, L, H, hd = q.shape
    S = torch.zeros(B, H, hd, hd, dtype=q.dtype) if s is None else s
    outs = []
    for t in range(L):
        kt, at, bt = k[:, t, :, :, None], a[:, t, :, None, None], b[:, t, :, None, None]
        S = at * (S - bt * (S @ kt) * kt.transpose(-1, -2)) + bt * v[:, t, :, :, None] * kt.transpose(-1, -2)
        outs.append((S @ q[:, t, :, :, None])[..., 0])
    return torch.stack(outs, 1), S


def close(got, want, name=""):
    err = (got.double().cpu() - want).abs()
    half = HALF_STEP[got.dtype]
    bound = half * want.abs() * (1 + 1e-3) + F32_REL * (want.norm() / want.numel() ** 0.5 + want.abs()) * 4
    assert torch.isfinite(got).all(), name
    assert bool((err <= bound).all()), (name, (err - bound).max().item())
    if half == 0.0:
        assert err.norm() <= F32_REL * want.norm(), (name, (err.norm() / want.norm()).item())


def gpu_args(args):
    return [None if t is None else t.cuda() for t in args]


SHAPES = [(1, 1, 1, 64), (2, 1, 3, 128), (1, 63, 2, 128), (1, 64, 2, 64), (2, 65, 3, 64), (3, 130, 2, 128), (1, 257, 8, 128)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("B,L,H,hd", SHAPES)
def test_forward(B, L, H, hd, state, dtype):
    from vit_amd import ops
    args = inputs(B, L, H, hd, dtype, state)
    want, want_s = recurrence(*(None if t is None else t.double() for t in args))
    out, s = ops.gated_delta_fwd(*gpu_args(args))
    assert out.dtype == dtype and s.dtype == torch.float32
    close(out, want, "out")
    close(s, want_s, "state")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,hd,state", [(1, 1, 1, 64, True), (2, 65, 3, 64, True), (1, 64, 1, 128, False), (2, 131, 2, 128, True),
                                            (1, 200, 3, 64, False)])
def test_gradients(B, L, H, hd, state, dtype):
    from vit_amd import module_ops
    args = inputs(B, L, H, hd, dtype, state, seed="dg")
    go = R.hashed_uniform("dg.go", (B, L, H, hd), 1.0).to(dtype)
    gs = R.hashed_uniform("dg.gs", (B, H, hd, hd), 0.5)
    ref = [None if t is None else t.double().requires_grad_() for t in args]
    leaves = [t for t in ref if t is not None]
    want = torch.autograd.grad(recurrence(*ref), leaves, (go.double(), gs.double()))
    dev = [None if t is None else t.cuda().requires_grad_() for t in args]
    got = torch.autograd.grad(module_ops.gated_delta(*dev), [t for t in dev if t is not None], (go.cuda(), gs.cuda()))
    for name, g, w, t in zip(("q", "k", "v", "alpha", "beta", "state"), got, want, leaves):
        assert g.shape == t.shape
        close(g, w, name)


@gpu
def test_gradients_against_differences():
    """Central differences of the kernel's own f32 forward along random directions: with step h the quotient is off by the
    forward's error over h (1e-5 |f| / h) and by the third derivative (h^2)."""
    from vit_amd import module_ops
    args = inputs(1, 97, 2, 64, torch.float32, True, seed="dd")
    go, gs = R.hashed_uniform("dd.go", (1, 97, 2, 64), 1.0).cuda(), R.hashed_uniform("dd.gs", (1, 2, 64, 64), 0.5).cuda()
    dev = [t.cuda().requires_grad_() for t in args]
    got = torch.autograd.grad(module_ops.gated_delta(*dev), dev, (go, gs))
    h = 0.02
    with torch.no_grad():
        def value(xs):
            o, s = module_ops.gated_delta(*xs)
            return (o.double() * go).sum().item() + (s.double() * gs).sum().item()
        for i, g in enumerate(got):
            direction = torch.sign(g)             # along it the quotient is the gradient's 1-norm: no cancellation
            direction = direction * (0.1 / max(1.0, direction.numel() ** 0.5))
            up, down = list(dev), list(dev)
            up[i], down[i] = dev[i] + h * direction, dev[i] - h * direction
            quotient = (value(up) - value(down)) / (2 * h)
            slope = (g.double() * direction).sum().item()
            assert abs(quotient - slope) <= 2e-2 * abs(slope) + 1e-4, (i, quotient, slope)


@gpu
def test_decays_of_zero_one_and_tiny_and_correlated_keys():
    """Decays of exactly 0 and 1, products that underflow, and keys of norm one that hardly differ (the triangular system
    is then far from diagonal): forward and every gradient."""
    from vit_amd import module_ops
    q, k, v, a, b, s = inputs(2, 140, 2, 64, torch.float32, True, seed="dz", unit=True)
    k = torch.nn.functional.normalize(k[:, :1] + 0.05 * k, dim=-1)
    a[0, 10] = 0.0
    a[0, 63:66] = 0.0
    a[1, 5:60] = 1.0
    a[1, 70:75] = 1e-30
    b[0, 20:30] = 1.0
    b[1, 20:30] = 0.0
    args = (q, k, v, a, b, s)
    go, gs = R.hashed_uniform("dz.go", q.shape, 1.0), R.hashed_uniform("dz.gs", s.shape, 0.5)
    ref = [t.double().requires_grad_() for t in args]
    out = recurrence(*ref)
    want = torch.autograd.grad(out, ref, (go.double(), gs.double()))
    dev = [t.cuda().requires_grad_() for t in args]
    res = module_ops.gated_delta(*dev)
    got = torch.autograd.grad(res, dev, (go.cuda(), gs.cuda()))
    for name, x, y in zip(("out", "state", "q", "k", "v", "alpha", "beta", "s0"), list(res) + list(got), list(out) + list(want)):
        close(x.detach(), y.detach(), name)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_a_wider_matrix_and_two_calls(dtype):
    """q, k, v as column blocks of one matrix; a sequence in two calls with the state carried equals one call."""
    from vit_amd import ops
    B, L, H, hd = 2, 150, 2, 64
    args = inputs(B, L, H, hd, dtype, True, seed="dw")
    wide = torch.full((B, L, 3 * H * hd + 8), float("nan"), dtype=dtype)
    for i in range(3):
        wide[..., i * H * hd:(i + 1) * H * hd] = args[i].reshape(B, L, -1)
    wide = wide.cuda()
    views = [wide[..., i * H * hd:(i + 1) * H * hd].unflatten(-1, (H, hd)) for i in range(3)]
    rest = gpu_args(args[3:])
    out, s = ops.gated_delta_fwd(*views, *rest)
    one, s1 = ops.gated_delta_fwd(*gpu_args(args))
    assert torch.equal(out, one) and torch.equal(s, s1)
    grads = ops.gated_delta_bwd(one, s1, *views, *rest)
    for x, y in zip(grads, ops.gated_delta_bwd(one, s1, *gpu_args(args))):
        assert torch.equal(x, y)
    dev = gpu_args(args)
    cut = 101
    o1, sm = ops.gated_delta_fwd(*(t[:, :cut].contiguous() for t in dev[:5]), dev[5])
    o2, sf = ops.gated_delta_fwd(*(t[:, cut:].contiguous() for t in dev[:5]), sm)
    want, want_s = recurrence(*(t.double() for t in args))
    close(torch.cat([o1, o2], 1), want)
    close(sf, want_s)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,hd", [(1, 1, 64), (1, 8, 128), (5, 3, 64), (70, 8, 128)])
def test_single_tokens(B, H, hd, dtype):
    """Three tokens one by one, the state updated in place."""
    from vit_amd import ops
    args = inputs(B, 3, H, hd, dtype, True, seed="ds")
    want, want_s = recurrence(*(t.double() for t in args))
    q, k, v, a, b, s = gpu_args(args)
    for t in range(3):
        o = ops.gated_delta_step_(q[:, t], k[:, t], v[:, t], a[:, t].contiguous(), b[:, t].contiguous(), s)
        close(o, want[:, t], t)
    close(s, want_s)


@gpu
def test_many_heads_take_the_other_launch_shape():
    """Enough heads that all columns of one share a workgroup: each head equals the same head alone (and the same sums)."""
    from vit_amd import ops
    for hd, B, H in ((128, 32, 8), (64, 64, 8)):
        args = gpu_args(inputs(B, 70, H, hd, torch.float32, True, seed="dm"))
        out, s = ops.gated_delta_fwd(*args)
        few, s_few = ops.gated_delta_fwd(*(t[3:5].contiguous() for t in args))
        assert torch.equal(out[3:5], few) and torch.equal(s[3:5], s_few)
        grads = ops.gated_delta_bwd(out, s, *args)
        few = ops.gated_delta_bwd(out[3:5].contiguous(), s[3:5].contiguous(), *(t[3:5].contiguous() for t in args))
        for x, y in zip(grads, few):
            assert torch.equal(x[3:5], y)


@gpu
def test_graph_replays_and_other_streams():
    from vit_amd import ops
    args = gpu_args(inputs(2, 100, 2, 128, torch.float32, True, seed="dr"))
    go, gs = torch.ones_like(args[0]), torch.ones_like(args[5])

    def step():
        out, s = ops.gated_delta_fwd(*args)
        return [out, s, *ops.gated_delta_bwd(go, gs, *args)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, y in zip(step(), want):
            assert torch.equal(x, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    base = args[2].clone()
    for i in range(3):
        args[2].copy_(base * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, step()):
            assert torch.equal(x, y), i


@gpu
def test_refusals():
    from vit_amd import module_ops, ops
    q, k, v, a, b, s = gpu_args(inputs(2, 5, 2, 64, torch.float32, True, seed="df"))
    bad = [(q[..., :32], k[..., :32], v[..., :32], a, b, None),                        # head dim
           (q.double(), k.double(), v.double(), a, b, s), (q, k.bfloat16(), v, a, b, s),
           (q, k[:, :4], v, a, b, s), (q, k, v, a[:, :4], b, s), (q, k, v, a, b.double(), s),
           (q, k, v, a, b, s[:1]), (q, k, v, a, b, s.transpose(-1, -2)), (q[:, :0], k[:, :0], v[:, :0], a[:, :0], b[:, :0], s),
           (q.transpose(1, 2).contiguous().transpose(1, 2), k, v, a, b, s)]             # heads apart
    for args in bad:
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.gated_delta_fwd(*args)
    with pytest.raises(ValueError):
        ops.gated_delta_step_(q[:, 0], k[:, 0], v[:, 0], a[:, 0].contiguous(), b[:, 0].contiguous(), None)
    with pytest.raises(ValueError):
        ops.gated_delta_bwd(torch.ones_like(q).transpose(0, 1), None, q, k, v, a, b, s)
    odd = torch.zeros(2 * 5 * 2 * 64 + 1, device="cuda")[1:].view(2, 5, 2, 64)           # four bytes past 16
    with pytest.raises(RuntimeError):
        ops.gated_delta_fwd(odd, k, v, a, b, s)
    assert module_ops.gated_delta(q, k, v, a, b, s)[0].shape == q.shape


def test_refusals_without_a_gpu():
    """A host tensor is refused before anything is loaded or launched."""
    from vit_amd import _lib, ops
    args = inputs(1, 3, 2, 64, torch.float32, True)
    with pytest.raises(_lib.VitAmdError):
        ops.gated_delta_fwd(*args)
    with pytest.raises(_lib.VitAmdError):
        ops.gated_delta_bwd(args[0], None, *args)
    with pytest.raises(_lib.VitAmdError):
        ops.gated_delta_step_(*(t[:, 0] for t in args[:5]), args[5])


def test_row_strides():
    from vit_amd.ops import _heads_ld
    x = torch.zeros(3, 5, 2, 64)
    assert _heads_ld(x, "x") == 128 and _heads_ld(x[:, :1], "x") == 640 and _heads_ld(x[:1, :1], "x") == 128
    assert _heads_ld(x[..., :1, :], "x") == 128 and _heads_ld(x[:, 2], "x") == 640
    assert _heads_ld(torch.zeros(3, 5, 400)[..., 8:136].unflatten(-1, (2, 64)), "x") == 400
    for bad in (x[:, :4], x[:, ::2], x.transpose(0, 1), x.transpose(1, 2), x[..., ::2]):
        with pytest.raises(ValueError):
            _heads_ld(bad, "x")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,hd", [(2, 131, 2, 128), (1, 64, 3, 64), (33, 70, 4, 128)])
def test_what_the_forward_keeps_equals_what_the_gradient_computes_again(B, L, H, hd, dtype):
    from vit_amd import ops
    args = gpu_args(inputs(B, L, H, hd, dtype, True, seed="dk"))
    out, s, kept = ops.gated_delta_fwd(*args, keep=True)
    one, s1 = ops.gated_delta_fwd(*args)
    assert torch.equal(out, one) and torch.equal(s, s1)
    for x, y in zip(ops.gated_delta_bwd(out, s, *args, kept=kept), ops.gated_delta_bwd(out, s, *args)):
        assert torch.equal(x, y)
    with pytest.raises(ValueError):
        ops.gated_delta_bwd(out, s, *args, kept=kept[1:])


@gpu
def test_a_non_finite_token_stays_in_its_head_and_stream():
    """Through the state it spreads over what follows; other heads and streams, and the chunks before, give the bits they give
    without it."""
    from vit_amd import ops
    args = gpu_args(inputs(2, 200, 3, 64, torch.float32, True, seed="dn"))
    out, s = ops.gated_delta_fwd(*args)
    bad = [t.clone() for t in args]
    bad[2][0, 130, 1, 5] = float("nan")
    got, sg = ops.gated_delta_fwd(*bad)
    assert torch.equal(got[1], out[1]) and torch.equal(sg[1], s[1])
    assert torch.equal(got[0, :, [0, 2]], out[0, :, [0, 2]]) and torch.equal(sg[0, [0, 2]], s[0, [0, 2]])
    assert torch.equal(got[0, :128, 1], out[0, :128, 1])
    assert bool(torch.isnan(got[0, 130:, 1]).any()) and bool(torch.isnan(sg[0, 1]).any())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,hd,state", [(2, 150, 2, 64, True), (1, 130, 3, 128, False), (65, 70, 2, 128, True)])
def test_what_the_recurrence_leaves_finite_is_finite(B, L, H, hd, state, dtype):
    """NaN and infinities in a value, a key, a query, both gates and the state: the same elements are non-finite as token by
    token, and the others as close as ever."""
    from vit_amd import ops
    nan, inf = float("nan"), float("inf")
    args = inputs(B, L, H, hd, dtype, state, seed="dx")
    q, k, v, a, b, s = args
    v[0, L - 20, 0, 5] = nan
    v[B - 1, 10, 1, hd - 1] = -inf
    k[0, 66, 1, 3] = nan
    if B > 1:
        q[1, 9, 0, 0] = inf
        b[1, L - 3, 1] = nan
    if B > 2:
        a[2, 65, 0] = nan
        k[3, 40, 1, 7] = inf
        s[4, 1, 17, 2] = nan
    want, want_s = recurrence(*(None if t is None else t.double() for t in args))
    dev = gpu_args(args)
    for keep in (False, True):
        out, st = ops.gated_delta_fwd(*dev, keep=keep)[:2]
        for name, got, ref in (("out", out, want), ("state", st, want_s)):
            ok = torch.isfinite(ref)
            assert torch.equal(torch.isfinite(got).cpu(), ok), name
            close(torch.where(ok.cuda(), got, torch.zeros_like(got)), torch.where(ok, ref, torch.zeros_like(ref)), name)


@gpu
def test_a_state_changed_in_place_is_not_used_by_a_gradient():
    from vit_amd import module_ops, ops
    q, k, v, a, b, s = gpu_args(inputs(1, 5, 1, 64, torch.float32, True, seed="dv"))
    v.requires_grad_()
    out, _ = module_ops.gated_delta(q, k, v, a, b, s)
    ops.gated_delta_step_(q[:, 0], k[:, 0], v.detach()[:, 0], a[:, 0], b[:, 0], s)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def second_derivatives(f, args, directions):
    """Gradients of sum(gradients of f * directions) in every input."""
    leaves = [t.requires_grad_() for t in args]
    out, s = f(*leaves)
    first = torch.autograd.grad((out * directions[0]).sum() + (s * directions[1]).sum(), leaves, create_graph=True)
    return torch.autograd.grad(sum((g * (i + 1)).pow(2).sum() for i, g in enumerate(first)), leaves)


@gpu
def test_second_derivatives_and_batched_gradients():
    """They come from the formula in torch, f32: sums of a few hundred products within sums of a few hundred products, each good
    to 1e-5 of its 2-norm; 1e-4 leaves room for both and for the tokens behind one another."""
    from vit_amd import module_ops
    args = inputs(2, 6, 2, 64, torch.float32, True, seed="d2")
    go, gs = R.hashed_uniform("d2.go", (2, 6, 2, 64), 1.0), R.hashed_uniform("d2.gs", (2, 2, 64, 64), 0.5)
    want = second_derivatives(recurrence, [t.double() for t in args], (go.double(), gs.double()))
    got = second_derivatives(module_ops.gated_delta, gpu_args(args), (go.cuda(), gs.cuda()))
    for g, w in zip(got, want):
        assert (g.double().cpu() - w).norm() <= 1e-4 * w.norm()
    # one tensor as two inputs
    def twice(f, q, *rest):
        out, s = f(q, q, *rest)
        (first,) = torch.autograd.grad(out.pow(2).sum(), q, create_graph=True)
        return torch.autograd.grad(first.pow(2).sum(), q)[0]
    rest = [t.detach() for t in args[2:]]
    want = twice(recurrence, args[0].detach().double().requires_grad_(), *(t.double() for t in rest))
    got = twice(module_ops.gated_delta, args[0].detach().cuda().requires_grad_(), *gpu_args(rest))
    assert (got.double().cpu() - want).norm() <= 1e-4 * want.norm()
    # several gradients at once
    dev = [t.detach().cuda().requires_grad_() for t in args]
    out, _ = module_ops.gated_delta(*dev)
    seeds = R.hashed_uniform("d2.seeds", (3, 2, 6, 2, 64), 1.0).cuda()
    many = torch.autograd.grad(out, dev, seeds, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(many, torch.autograd.grad(out, dev, seeds[i], retain_graph=True)):
            assert (a[i] - b).norm() <= 1e-4 * b.norm()
