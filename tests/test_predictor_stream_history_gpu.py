"""GPU: a stream reads its history.  One block, attention branch alone, timesteps of 258 tokens over a cache of many blocks,
against a 64-bit attention over what the cache stands for at the time of each call: e4m3 codes times their scale for the
blocks that are whole by then, bf16 for the open one.

Both sides round the same bf16 operands (normalised rows, projections, attention output), so what is left is a rounding that
falls on the other side of a border: the repository's bf16 tolerance of 2e-2, with nothing added for the codes.  The same
attention without the history differs by a multiple of that, which the test asserts too."""
import math

import pytest
import torch

from oracle import ref_cpu as R

pytestmark = pytest.mark.gpu
REL_TOL = 2e-2
BF16, F64 = torch.bfloat16, torch.float64


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def through_codes(x, tokens):
    """[B, H, n, hd] as a cache of `tokens` tokens holds them: whole blocks of 64 rounded to e4m3 under one power of two."""
    B, H, _, hd = x.shape
    whole = tokens // 64 * 64
    w = x[:, :, :whole].reshape(B, H, -1, 64, hd)
    scale = torch.exp2(torch.ceil(torch.log2(w.abs().amax((-1, -2), keepdim=True) / 448)))
    w = (w / scale).float().to(torch.float8_e4m3fn).double() * scale
    return torch.cat([w.view(B, H, whole, hd), x[:, :, whole:tokens]], 2)


def test_the_attention_branch_reads_all_earlier_timesteps():
    from vit_amd import surgical_world_model as swm
    heads, tpt, T, B = 8, 258, 4, 2
    blk = swm.HybridPredictorBlock(1024, heads, use_deltanet=False)
    P = R.fill_state_dict_({f"hi.{k}": v for k, v in blk.state_dict().items()})
    blk.load_state_dict({k[3:]: v for k, v in P.items()})
    with torch.no_grad():
        for p in (blk.mlp[2].weight, blk.mlp[2].bias):
            p.zero_()                                          # what the block adds is its attention branch
    blk = blk.eval().cuda()
    a, N, hd = blk.spatial_attn, T * tpt, 1024 // heads
    x = R.hashed_uniform("hi.x", (B, N, 1024), 1.0).cuda()
    with torch.no_grad():
        stream = blk.new_stream(B, N, x.device)
        got = torch.cat([blk.stream(x[:, t * tpt:(t + 1) * tpt], stream, tpt) for t in range(T)], 1) - x
        ln = torch.nn.functional.layer_norm(x.double(), (1024,), blk.norm1.weight.double(), blk.norm1.bias.double(), blk.norm1.eps)
        qkv = ln.to(BF16).double() @ a.in_proj_weight.to(BF16).double().T + a.in_proj_bias.double()
        q, k, v = qkv.to(BF16).double().view(B, N, 3, heads, hd).permute(2, 0, 3, 1, 4)
        rows = {"all": [], "own timestep": []}
        for t in range(T):
            held = (t + 1) * tpt
            keys, values = through_codes(k, held), through_codes(v, held)
            for name, first in (("all", 0), ("own timestep", t * tpt)):
                w = torch.softmax(q[:, :, t * tpt:held] @ keys[:, :, first:].transpose(-1, -2).contiguous() / math.sqrt(hd), -1)
                o = (w @ values[:, :, first:]).transpose(1, 2).reshape(B, tpt, 1024)
                rows[name].append(o.to(BF16).double() @ a.out_proj.weight.to(BF16).double().T + a.out_proj.bias.double())
        want, without = (torch.cat(r, 1) for r in rows.values())
    for t in range(T):
        part = slice(t * tpt, (t + 1) * tpt)
        assert rel(got[:, part], want[:, part]) < REL_TOL, t
        if t > 0:
            assert rel(without[:, part], want[:, part]) > 5 * REL_TOL, t


def test_states_that_do_not_fit_are_refused_before_any_block_has_taken_the_tokens():
    from vit_amd import surgical_world_model as swm
    model = swm.SurgicalActionConditionedWorldModel(img_size=32, num_frames=4, encoder_depth=1, encoder_heads=16,
                                                    predictor_depth=2, predictor_heads=8).cuda()
    B, per = 2, model.tokens_per_frame + 2
    tokens = R.hashed_uniform("hi.w", (B, per, 1024), 1.0).cuda()
    steps = 128 // per                                         # timesteps that a cache of two blocks holds
    for spoil in ("batch", "capacity"):
        streams = model.new_predictor_streams(B, steps + 70, tokens.device)
        streams[1] = model.predictor_blocks[1].new_stream(B + (spoil == "batch"), 128 if spoil == "capacity" else 512, tokens.device)
        taken = 0
        while spoil == "capacity" and taken < steps:
            model.predict_stream(tokens, streams)
            taken += 1
        with pytest.raises(ValueError):
            model.predict_stream(tokens, streams)
        assert streams[0].kv.lengths.tolist() == [taken * per] * B
