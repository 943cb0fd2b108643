"""GPU: the memory layer with gradients, and the predictor run timestep by timestep from its cache.

The layer's gradients are compared with a 64-bit copy of the layer on the host (torch's f32 layers around the kernels: 1e-4 of
a gradient's 2-norm is what their f32 products of 1024 terms, eight layers deep, may lose; 2^-24 * 1024 = 6e-5).
A stream whose tokens fit the open block of its cache (64) rounds exactly what the whole-sequence path rounds, bf16 operands,
in another order of summation: the repository's bf16 tolerance of 2e-2.  Longer ones also round every key and value of a
whole block to e4m3, by at most 2^-4 of it, which the attention's average over keys can only reduce."""
import pytest
import torch

from oracle import ref_cpu as R

pytestmark = pytest.mark.gpu
REL_TOL = 2e-2


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def filled(module, seed):
    P = R.fill_state_dict_({f"{seed}.{k}": v for k, v in module.state_dict().items()})
    module.load_state_dict({k[len(seed) + 1:]: v for k, v in P.items()})
    return module.eval()


@pytest.mark.parametrize("heads,hd,L", [(4, 128, 70), (3, 64, 131)])
def test_memory_layer_gradients(heads, hd, L):
    from vit_amd import surgical_world_model as swm
    dim, B = 192, 2
    layer = filled(swm.GatedDeltaLayer(dim, num_heads=heads, head_dim=hd), "ml")
    x = R.hashed_uniform("ml.x", (B, L, dim), 1.0)
    s0 = R.hashed_uniform("ml.s", (B, heads, hd, hd), 0.2)
    go, gs = R.hashed_uniform("ml.go", (B, L, dim), 1.0), R.hashed_uniform("ml.gs", s0.shape, 0.3)
    import copy
    ref = copy.deepcopy(layer).double()
    xr, sr = x.double().requires_grad_(), s0.double().requires_grad_()
    want = ref(xr, sr)
    wanted = torch.autograd.grad(want, [xr, sr, *ref.parameters()], (go.double(), gs.double()))
    layer = layer.cuda()
    xg, sg = x.cuda().requires_grad_(), s0.cuda().requires_grad_()
    got = layer(xg, sg)
    assert rel(got[0], want[0]) < 1e-4 and rel(got[1], want[1]) < 1e-4
    grads = torch.autograd.grad(got, [xg, sg, *layer.parameters()], (go.cuda(), gs.cuda()))
    for name, g, w in zip(["x", "state"] + [n for n, _ in layer.named_parameters()], grads, wanted):
        assert rel(g, w) < 1e-4, name
    # a frozen layer behind trainable features, no gradient through the state
    layer.requires_grad_(False)
    (gx,) = torch.autograd.grad(layer(xg, s0.cuda()), [xg], (go.cuda(), gs.cuda()))
    assert rel(gx, wanted[0]) < 1e-4


def block(heads, deltanet=True):
    from vit_amd import surgical_world_model as swm
    return swm, filled(swm.HybridPredictorBlock(1024, heads, use_deltanet=deltanet), "ps").cuda()


@pytest.mark.parametrize("deltanet,tpt,calls", [(True, 10, (10, 20, 10, 10)), (True, 1, (1, 1, 2, 1, 30, 1)), (False, 16, (16, 48))])
def test_stream_within_the_open_block(deltanet, tpt, calls):
    swm, blk = block(8, deltanet)
    B, L = 3, sum(calls)
    x = R.hashed_uniform("ps.x", (B, L, 1024), 1.0).cuda()
    with torch.no_grad():
        want, state = blk(x, attn_mask=swm.BlockCausalMask.create_mask(L, tpt, x.device))
        stream = blk.new_stream(B, 64, x.device)
        for _ in range(2):                                    # and again after a reset
            at, got = 0, []
            for n in calls:
                got.append(blk.stream(x[:, at:at + n], stream, tpt))
                at += n
            assert rel(torch.cat(got, 1), want) < REL_TOL
            if deltanet:
                assert rel(stream.state, state) < REL_TOL
            stream.reset()


def test_stream_over_many_blocks():
    swm, blk = block(8)
    B, tpt, T = 2, 258, 4
    x = R.hashed_uniform("pm.x", (B, T * tpt, 1024), 1.0).cuda()
    with torch.no_grad():
        want, state = blk(x, attn_mask=swm.BlockCausalMask.create_mask(T * tpt, tpt, x.device))
        stream = blk.new_stream(B, T * tpt, x.device)
        got = torch.cat([blk.stream(x[:, t * tpt:(t + 1) * tpt], stream, tpt) for t in range(T)], 1)
    # what the block adds to its input, 2^-4 of it at most through the codes
    assert rel(got - x, want - x) < REL_TOL + 2.0 ** -4
    assert rel(stream.state, state) < REL_TOL + 2.0 ** -4
    assert stream.kv.lengths.tolist() == [T * tpt] * B
    with pytest.raises(ValueError), torch.no_grad():
        blk.stream(x[:, :tpt], stream, tpt)                   # the cache is full


def test_stream_refusals():
    swm, blk = block(8)
    from vit_amd import _lib
    x = R.hashed_uniform("pr.x", (2, 6, 1024), 1.0).cuda()
    stream = blk.new_stream(2, 64, x.device)
    with pytest.raises(_lib.VitAmdError):
        blk.stream(x, stream, 3)                              # grad mode on
    with torch.no_grad():
        for bad, tpt in ((x[:1], 3), (x, 4), (x[:, :0], 3)):
            with pytest.raises(ValueError):
                blk.stream(bad, stream, tpt)
        with pytest.raises(_lib.VitAmdError):
            blk.stream(x.cpu(), stream, 3)
        with pytest.raises(_lib.VitAmdError):
            swm.HybridPredictorBlock(512, 8).cuda().stream(x[..., :512], stream, 3)


def test_world_model_timestep_by_timestep():
    """`predict_stream` on the interleaved tokens of each timestep equals the predictor blocks and the norm on all of them."""
    from vit_amd import surgical_world_model as swm
    model = filled(swm.SurgicalActionConditionedWorldModel(img_size=32, num_frames=8, encoder_depth=1, encoder_heads=16,
                                                           predictor_depth=3, predictor_heads=8), "wm").cuda()
    B, T, per = 2, 12, model.tokens_per_frame + 2
    tokens = R.hashed_uniform("wm.tokens", (B, T * per, 1024), 1.0).cuda()
    with torch.no_grad():
        mask, x = swm.BlockCausalMask.create_mask(T * per, per, tokens.device), tokens
        for blk in model.predictor_blocks:
            x, _ = blk(x, attn_mask=mask)
        want = model.predictor_norm(x)
    streams = model.new_predictor_streams(B, T, tokens.device)
    got = torch.cat([model.predict_stream(tokens[:, t * per:(t + 1) * per], streams) for t in range(T)], 1)
    assert got.shape == want.shape and rel(got, want) < REL_TOL + 2.0 ** -4
    with pytest.raises(ValueError):
        model.predict_stream(tokens[:, :per], streams[:2])
    assert all(s.kv.lengths.tolist() == [T * per] * B for s in streams)


def test_memory_layer_where_torch_must_see_every_operation():
    """torch.func transforms, forward-mode derivatives, second derivatives, one state for all streams: what a layer of
    torch operations allows."""
    from vit_amd import surgical_world_model as swm
    layer = filled(swm.GatedDeltaLayer(64, num_heads=2, head_dim=64), "mt").cuda()
    x, t = (R.hashed_uniform(f"mt.{n}", (2, 9, 64), 1.0).cuda() for n in "xt")
    s1 = R.hashed_uniform("mt.s", (1, 2, 64, 64), 0.2).cuda()
    value = lambda y: layer(y)[0].pow(2).sum()                 # noqa: E731
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(value(leaf), leaf, create_graph=True)
    assert rel(torch.func.grad(value)(x), want) < 1e-4
    _, slope = torch.func.jvp(value, (x,), (t,))
    assert abs(slope.item() - (want * t).sum().item()) <= 1e-4 * (want.norm() * t.norm()).item()
    (second,) = torch.autograd.grad((want * t).sum(), leaf)
    h = 1e-2
    up, down = (torch.func.grad(value)(x + d * t) for d in (h, -h))
    assert rel(second, (up - down) / (2 * h)) < 1e-2           # third derivatives times h^2, f32 noise over h
    assert rel(layer(leaf, s1)[0], layer(leaf, s1.expand(2, 2, 64, 64).contiguous())[0]) == 0.0
    with pytest.raises(ValueError):
        layer(leaf[:0])
