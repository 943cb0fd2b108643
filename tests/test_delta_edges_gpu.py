"""GPU: gradients of the chunked delta rule where an input, a gate, a state or an incoming gradient is not finite: the same
elements are non-finite as in the gradients of the token-by-token recurrence, and the others as close as ever (tolerances as
in test_delta_gpu.py)."""
import pytest
import torch

from oracle import ref_cpu as R
from test_delta_gpu import close, gpu_args, inputs, recurrence

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
NAMES = ("q", "k", "v", "alpha", "beta", "state")


def gradients(args, go, gs):
    leaves = [None if t is None else t.requires_grad_() for t in args]
    return torch.autograd.grad(recurrence(*leaves), [t for t in leaves if t is not None], (go, gs))


def check(args, go, gs):
    """The kernel's gradients, with what the forward keeps and without, against those of the recurrence in 64 bits."""
    from vit_amd import ops
    want = gradients([None if t is None else t.detach().double() for t in args], go.double(), gs.double())
    dev = gpu_args([None if t is None else t.detach() for t in args])
    out, s, kept = ops.gated_delta_fwd(*dev, keep=True)
    got_both = []
    for have in (None, kept, kept):                            # what is kept is not changed by a gradient
        got = ops.gated_delta_bwd(go.cuda(), gs.cuda(), *dev, kept=have)
        got = got if args[5] is not None else got[:5]
        got_both.append(got)
        for name, g, w in zip(NAMES, got, want):
            ok = torch.isfinite(w)
            assert torch.equal(torch.isfinite(g).cpu(), ok), name
            if bool(ok.any()):
                close(torch.where(ok.cuda(), g, torch.zeros_like(g)), torch.where(ok, w, torch.zeros_like(w)), name)
    for x, y in zip(got_both[1], got_both[2]):
        assert torch.equal(x.nan_to_num(7.0, 8.0, 9.0), y.nan_to_num(7.0, 8.0, 9.0))
    return want


# which operand, where: a value, a key, a query, the gates; the first token, in a chunk, at its border, the last token
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which,at,what", [(2, (0, 130, 1, 5), NAN), (2, (0, 0, 0, 63), INF), (1, (1, 64, 0, 3), NAN),
                                           (1, (0, 149, 1, 0), -INF), (0, (1, 63, 1, 7), NAN), (0, (0, 149, 0, 7), INF),
                                           (3, (1, 70, 1), NAN), (4, (0, 20, 0), NAN), (5, (1, 0, 17, 2), NAN)])
def test_one_bad_number(which, at, what, dtype):
    B, L, H, hd = 2, 150, 2, 64
    args = list(inputs(B, L, H, hd, dtype, True, seed="eg"))
    go, gs = R.hashed_uniform("eg.go", (B, L, H, hd), 1.0).to(dtype), R.hashed_uniform("eg.gs", (B, H, hd, hd), 0.5)
    args[which][at] = what
    want = check(args, go, gs)
    assert not all(bool(torch.isfinite(w).all()) for w in want)
    assert all(bool(torch.isfinite(w[1 - at[0]]).all()) for w in want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bad_incoming_gradient(dtype):
    B, L, H, hd = 2, 140, 2, 128
    args = inputs(B, L, H, hd, dtype, True, seed="eh")
    go, gs = R.hashed_uniform("eh.go", (B, L, H, hd), 1.0).to(dtype), R.hashed_uniform("eh.gs", (B, H, hd, hd), 0.5)
    go[0, 70, 1, 5] = NAN
    gs[1, 0, 3, 4] = INF
    check(args, go, gs)


@pytest.mark.parametrize("B,L,H,hd", [(1, 1, 1, 64), (1, 5, 3, 128), (2, 65, 2, 128), (65, 70, 2, 128), (1, 200, 1, 64)])
def test_shapes_without_a_state(B, L, H, hd):
    args = list(inputs(B, L, H, hd, torch.float32, False, seed="ei"))
    args[2][0, L // 2, H - 1, 9] = NAN
    args[2][B - 1, L - 1, 0, hd - 1] = INF
    go, gs = R.hashed_uniform("ei.go", (B, L, H, hd), 1.0), R.hashed_uniform("ei.gs", (B, H, hd, hd), 0.5)
    check(args, go, gs)


def test_rows_of_a_wider_matrix_and_other_heads_keep_their_bits():
    from vit_amd import ops
    B, L, H, hd = 2, 130, 3, 64
    args = gpu_args(inputs(B, L, H, hd, torch.float32, True, seed="ej"))
    go, gs = R.hashed_uniform("ej.go", (B, L, H, hd), 1.0).cuda(), R.hashed_uniform("ej.gs", (B, H, hd, hd), 0.5).cuda()
    clean = ops.gated_delta_bwd(go, gs, *args)
    args[2][0, 100, 1, 5] = NAN
    wide = torch.full((B, L, 3 * H * hd + 8), NAN, device="cuda")
    for i in range(3):
        wide[..., i * H * hd:(i + 1) * H * hd] = args[i].reshape(B, L, -1)
    views = [wide[..., i * H * hd:(i + 1) * H * hd].unflatten(-1, (H, hd)) for i in range(3)]
    one, two = ops.gated_delta_bwd(go, gs, *args), ops.gated_delta_bwd(go, gs, *views, *args[3:])
    for x, y, z in zip(one, two, clean):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
        heads = x if x.dim() == 4 and x.shape[1] == H else x.transpose(1, 2)           # the state's are [B, H, ..]
        before = z if z.dim() == 4 and z.shape[1] == H else z.transpose(1, 2)
        assert torch.equal(heads[1], before[1]) and torch.equal(heads[0, [0, 2]], before[0, [0, 2]])
        assert not torch.equal(heads[0, 1], before[0, 1])


def test_replays_follow_what_the_inputs_hold():
    """Captured with finite inputs, replayed with a bad one and with finite ones again."""
    from vit_amd import ops
    B, L, H, hd = 1, 100, 2, 64
    args = gpu_args(inputs(B, L, H, hd, torch.float32, True, seed="ek"))
    go, gs = torch.ones_like(args[0]), torch.ones_like(args[5])

    def step():
        return ops.gated_delta_bwd(go, gs, *args)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for bad in (False, True, False, True):
        args[2][0, 70, 1, 3] = NAN if bad else 0.5
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, step()):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))
        assert bool(torch.isnan(held[1]).any()) == bad and bool(torch.isfinite(held[1][:, :70]).all())
