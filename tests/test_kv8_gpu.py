"""GPU: the 8-bit key/value cache and the attention over it.

The cache is compared exactly: a scale is a power of two, so a code is one rounding of a bf16 number to e4m3, which the host
computes too.  Attention is compared with a 64-bit softmax over the numbers that the codes stand for: scores and sums are f32,
each weight is rounded to bf16 once (2^-8 of it) and so is the result, so a result is off by at most
2^-8 |o| + 2^-8 sum_j w_j |v_j| plus f32 noise (1e-5 of sum_j w_j |v_j| for the exponentials of scores up to about 40)."""
import math

import pytest
import torch

from oracle import ref_cpu as R

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def tokens(B, n, H, hd, name="kv", scale=2.0):
    return R.hashed_uniform(name, (B, n, H, hd), scale).to(BF16)


def encode(block):
    """Codes and scale of one block [64, hd] bf16 as the definition says them."""
    x = block.double()
    finite = x[torch.isfinite(x)].abs()
    top = finite.max().item() if finite.numel() else 0.0
    e = 0 if top == 0 else max(-100, math.ceil(math.log2(top / 448)))
    y = (x / 2.0 ** e).float()
    y[~torch.isfinite(y)] = float("nan")
    return y.to(torch.float8_e4m3fn), 2.0 ** e


def check_cache(cache, k, v, lens):
    """Every stream's whole blocks and open block against its tokens k, v (lists of [len, H, hd])."""
    assert cache.lengths.tolist() == lens
    for codes, scales, opened, x in ((cache.k8, cache.k_scale, cache.k_open, k), (cache.v8, cache.v_scale, cache.v_open, v)):
        codes, scales, opened = codes.view(torch.uint8).cpu(), scales.cpu(), opened.cpu()
        for b, n in enumerate(lens):
            for h in range(codes.shape[1]):
                for j in range(n // 64):
                    want, s = encode(x[b][64 * j:64 * j + 64, h])
                    assert scales[b, h, j] == s, (b, h, j)
                    got = codes[b, h, 64 * j:64 * j + 64].view(torch.float8_e4m3fn).float()
                    assert torch.equal(torch.nan_to_num(got, 999.0), torch.nan_to_num(want.float(), 999.0)), (b, h, j)
                rest = n % 64
                assert torch.equal(opened[b, h, :rest].view(torch.int16), x[b][n - rest:n, h].view(torch.int16)), (b, h)


def held(cache, b, h):
    """Keys and values of one stream and head as 64-bit numbers."""
    n = int(cache.lengths[b])
    out = []
    for codes, scales, opened in ((cache.k8, cache.k_scale, cache.k_open), (cache.v8, cache.v_scale, cache.v_open)):
        w = n // 64 * 64
        x = codes[b, h, :w].cpu().double() * scales[b, h, :n // 64].cpu().double().repeat_interleave(64)[:, None]
        out.append(torch.cat([x, opened[b, h, :n - w].cpu().double()]))
    return out


def attention(q, cache, new, tpt, scale=None):
    """(result, sum_j w_j |v_j|) in 64 bits."""
    B, n, Hq, hd = q.shape
    out, size = torch.zeros(B, n, Hq, hd, dtype=torch.float64), torch.zeros(B, n, Hq, hd, dtype=torch.float64)
    for b in range(B):
        total = int(cache.lengths[b])
        for h in range(Hq):
            k, v = held(cache, b, h // (Hq // cache.heads))
            for i in range(new[b]):
                p = total - new[b] + i
                end = total if tpt == 0 else min(total, (p // tpt + 1) * tpt)
                w = torch.softmax((k[:end] @ q[b, i, h].double()) * (hd ** -0.5 if scale is None else scale), 0)
                out[b, i, h], size[b, i, h] = w @ v[:end], w @ v[:end].abs()
    return out, size


def close(got, want, size):
    err = (got.double().cpu() - want).abs()
    bound = 2.0 ** -8 * want.abs() * (1 + 2.0 ** -7) + (2.0 ** -8 + 1e-5) * size
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), (err - bound).max().item()


def filled(B, H, hd, lens, capacity=None, steps=(1.0,), name="kv"):
    """A cache brought to `lens` in calls of the given shares."""
    from vit_amd import ops
    cache = ops.KVCache8.empty(B, H, hd, capacity or max(lens), "cuda")
    most = max(lens)
    k, v = tokens(B, most, H, hd, name + ".k"), tokens(B, most, H, hd, name + ".v")
    if most:
        lens_t = torch.tensor(lens)
        at = 0
        for cut in [int(most * s) for s in steps]:
            if cut > at:
                new = (lens_t.clamp(max=cut) - at).clamp(min=0).to(torch.int32)
                ops.kv8_append_(cache, k[:, at:cut].cuda(), v[:, at:cut].cuda(), new=new.cuda())
                at = cut
    return cache, k, v


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,steps", [([1], (1.0,)), ([64, 63, 65], (1.0,)), ([0, 130, 64], (0.2, 0.5, 1.0)),
                                        ([300, 17, 255, 256], (0.01, 0.3, 0.31, 0.9, 1.0))])
def test_append(lens, steps, hd):
    cache, k, v = filled(len(lens), 3, hd, lens, steps=steps)
    check_cache(cache, k, v, lens)


@gpu
def test_append_of_single_tokens_equals_one_call_and_touches_nothing_else():
    from vit_amd import ops
    B, H, hd, n = 2, 2, 64, 130
    k, v = tokens(B, n, H, hd, "a.k").cuda(), tokens(B, n, H, hd, "a.v").cuda()
    caches = [ops.KVCache8.empty(B, H, hd, 256, "cuda") for _ in range(2)]
    for c in caches:
        c.k8.view(torch.uint8).fill_(17)
        c.v_scale.fill_(3.0)
        c.k_open.fill_(float("nan"))
    ops.kv8_append_(caches[0], k, v)
    for t in range(n):
        ops.kv8_append_(caches[1], k[:, t:t + 1], v[:, t:t + 1])
    for c in caches:
        check_cache(c, k.cpu(), v.cpu(), [n, n])
        assert bool((c.k8.view(torch.uint8)[:, :, 128:] == 17).all()) and bool((c.v_scale[:, :, 2:] == 3.0).all())
    assert torch.equal(caches[0].k8.view(torch.uint8), caches[1].k8.view(torch.uint8))
    # rows of the open block behind the tokens: as they were in the one call, older tokens or as they were in the other
    assert bool(torch.isnan(caches[0].k_open[:, :, 2:]).all())


@gpu
def test_append_of_zeros_extremes_infinities_and_nan():
    from vit_amd import ops
    k = tokens(1, 256, 2, 64, "x.k")
    k[0, :64, 0] = 0.0
    k[0, 3, 1, 5], k[0, 9, 1, 6] = float("nan"), float("inf")
    k[0, 64:128, 0] *= 1e-36                                   # scales stop at 2^-100
    k[0, 64:128, 1] = 2.0 ** 120
    k[0, 128:192, 0] = 448.0
    k[0, 128:192, 1] = 450.0                                   # the next bf16 number: one more step of the scale
    k[0, 192:, 0] = float("nan")
    cache = ops.KVCache8.empty(1, 2, 64, 256, "cuda")
    ops.kv8_append_(cache, k.cuda(), k.cuda())
    check_cache(cache, k, k, [256])


@gpu
def test_append_strided_and_full():
    """Column blocks of a packed projection output; a device-side length that would pass the capacity stays at it."""
    from vit_amd import ops
    B, n, H, hd = 2, 70, 2, 64
    packed = R.hashed_uniform("s.qkv", (B, n, 3 * H * hd), 1.0).to(BF16).cuda()
    q, k, v = (packed[..., i * H * hd:(i + 1) * H * hd].unflatten(-1, (H, hd)) for i in range(3))
    cache = ops.KVCache8.empty(B, H, hd, 128, "cuda")
    ops.kv8_append_(cache, k, v)
    check_cache(cache, k.cpu(), v.cpu(), [n, n])
    out = ops.kv8_attn(q, cache, tokens_per_timestep=1)
    assert torch.equal(out, ops.kv8_attn(q.contiguous(), cache, tokens_per_timestep=1))
    close(out, *attention(q.cpu(), cache, [n, n], 1))
    with pytest.raises(ValueError):
        ops.kv8_append_(cache, k, v)                           # 70 + 70 > 128
    cache.max_len = 0                                          # as after replays that the host has not seen
    ops.kv8_append_(cache, k, v)
    both_k, both_v = torch.cat([k, k], 1).cpu(), torch.cat([v, v], 1).cpu()
    check_cache(cache, both_k[:, :128], both_v[:, :128], [128, 128])


ROWS = [([1], 1, 1), ([64], 1, 1), ([65, 200], 1, 4), ([130, 0, 67], 1, 2), ([700], 3, 4), ([257], 16, 1), ([1500, 1499], 2, 8)]
TILES = [([17], 17, 1), ([258, 516], 258, 1), ([64, 129, 300], 40, 1), ([1000], 33, 4), ([520, 130], 130, 2)]


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,n,group", ROWS + TILES)
@pytest.mark.parametrize("tpt", [0, 1, 130])
def test_attention(lens, n, group, tpt, hd):
    from vit_amd import ops
    B, H = len(lens), 2
    cache, _, _ = filled(B, H, hd, lens, steps=(0.4, 1.0), capacity=max(lens) + 64)
    q = tokens(B, n, H * group, hd, "at.q", 3.0)
    counts = [min(n, x) for x in lens]
    new = torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = ops.kv8_attn(q.cuda(), cache, new=new, tokens_per_timestep=tpt)
    want, size = attention(q, cache, counts, tpt)
    close(out, want, size)
    for b, c in enumerate(counts):
        assert bool((out[b, c:] == 0).all())                  # padded rows
    if all(c == n for c in counts):
        assert torch.equal(out, ops.kv8_attn(q.cuda(), cache, tokens_per_timestep=tpt))


@gpu
def test_attention_with_large_scores_and_a_scale():
    """Scores of some hundreds: the running maximum moves; a scale of its own."""
    from vit_amd import ops
    cache, _, _ = filled(1, 1, 128, [900], name="big")
    for n in (1, 50):
        q = tokens(1, n, 1, 128, "big.q", 8.0)
        out = ops.kv8_attn(q.cuda(), cache, tokens_per_timestep=1, scale=0.5)
        want, size = attention(q, cache, [n], 1, 0.5)
        err = (out.double().cpu() - want).abs()
        # an f32 score s of size 600 is off by at most 600 * 2^-24 * 20 (64 products in 20 rounded levels): weights by 1e-3
        assert bool((err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2e-3) * size).all())


@gpu
@pytest.mark.parametrize("n", [2, 64])
def test_what_a_query_must_not_see_does_not_reach_it(n):
    """NaN and infinities in tokens behind a query's timestep, in the open block's unused rows and in padded query rows."""
    from vit_amd import ops
    B, H, hd, total = 2, 2, 64, 160 + n
    k, v = tokens(B, total, H, hd, "n.k"), tokens(B, total, H, hd, "n.v")
    q = tokens(B, n, H, hd, "n.q")
    clean = ops.KVCache8.empty(B, H, hd, total, "cuda")
    ops.kv8_append_(clean, k.cuda(), v.cuda())
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, -1, 0], bad_v[:, -1, 1] = float("nan"), float("inf")
    bad_v[:, -1, 0, 3] = float("nan")
    dirty = ops.KVCache8.empty(B, H, hd, total, "cuda")
    dirty.k_open.fill_(float("nan"))
    dirty.v_open.fill_(float("inf"))
    ops.kv8_append_(dirty, bad_k.cuda(), bad_v.cuda())
    assert total % 64 != 0                                     # the bad token lies in the open block: no scale is shared
    good = ops.kv8_attn(q.cuda(), clean, tokens_per_timestep=1)
    got = ops.kv8_attn(q.cuda(), dirty, tokens_per_timestep=1)
    # the last query sees the bad token, the others do not
    assert torch.equal(got[:, :-1], good[:, :-1])
    assert not bool(torch.isfinite(got[:, -1, 0]).any())
    assert bool(torch.isinf(got[:, -1, 1]).all())
    new = torch.tensor([n, 1], dtype=torch.int32, device="cuda")
    q[1, 1:] = float("nan")
    out = ops.kv8_attn(q.cuda(), clean, new=new, tokens_per_timestep=1)
    assert bool(torch.isfinite(out).all()) and bool((out[1, 1:] == 0).all())
    # a whole block with non-finite values, in 8 bits: queries before it
    late = ops.KVCache8.empty(1, 1, hd, 192, "cuda")
    bad_v = tokens(1, 192, 1, hd, "n.w")
    bad_k = tokens(1, 192, 1, hd, "n.z")
    ref = ops.KVCache8.empty(1, 1, hd, 192, "cuda")
    ops.kv8_append_(ref, bad_k.cuda(), bad_v.cuda())
    bad_v[0, 191, 0, 7] = float("nan")
    ops.kv8_append_(late, bad_k.cuda(), bad_v.cuda())
    q = tokens(1, n, 1, hd, "n.y").cuda()
    a, b = ops.kv8_attn(q, late, tokens_per_timestep=1), ops.kv8_attn(q, ref, tokens_per_timestep=1)
    assert torch.equal(a[:, :-1], b[:, :-1]) and bool(torch.isnan(a[0, -1, 0, 7])) and int(torch.isnan(a).sum()) == 1


@gpu
def test_far_offsets():
    """The second stream's codes lie more than 2^32 elements behind the first's."""
    from vit_amd import ops
    B, H, hd, cap = 2, 8, 128, 1 << 22
    k8, v8 = (torch.empty(B, H, cap, hd, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    small = ops.KVCache8.empty(B, H, hd, 320, "cuda")
    far = ops.KVCache8(k8, v8, torch.ones(B, H, cap // 64, device="cuda"), torch.ones(B, H, cap // 64, device="cuda"),
                       small.k_open.clone(), small.v_open.clone(), torch.zeros(B, dtype=torch.int32, device="cuda"), max_len=0)
    k, v = tokens(B, 300, H, hd, "f.k").cuda(), tokens(B, 300, H, hd, "f.v").cuda()
    for c in (small, far):
        ops.kv8_append_(c, k, v)
    for n in (1, 64):
        q = tokens(B, n, H, hd, "f.q").cuda()
        assert torch.equal(ops.kv8_attn(q, far, tokens_per_timestep=1), ops.kv8_attn(q, small, tokens_per_timestep=1))
    # the last blocks of the capacity
    far.lengths.fill_(cap - 100)
    far.max_len = cap - 100
    far.lengths[0] = 0
    ops.kv8_append_(far, k[:, :100], v[:, :100], new=torch.tensor([0, 100], dtype=torch.int32, device="cuda"))
    codes, scale = encode(k[1, 36:100, 7].cpu())
    assert torch.equal(far.k8[1, 7, cap - 64:].cpu().view(torch.uint8), codes.view(torch.uint8)) and far.k_scale[1, 7, -1] == scale


@gpu
def test_graph_replays_and_other_streams():
    """Append and attend of one token captured once and replayed, against the same calls made eagerly on another cache."""
    from vit_amd import ops
    B, H, hd = 2, 2, 128
    caches = [filled(B, H, hd, [190, 120], capacity=512)[0] for _ in range(2)]
    k, v, q = (tokens(B, 1, H, hd, f"g.{c}").cuda() for c in "kvq")

    def step(c):
        ops.kv8_append_(c, k, v)
        return ops.kv8_attn(q, c, tokens_per_timestep=1)

    warm = filled(B, H, hd, [190, 120], capacity=512)[0]
    step(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
    side = torch.cuda.Stream()
    for i in range(6):
        for t in (k, v, q):
            t.copy_(torch.roll(t, 1, -1))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step(caches[1])
        torch.cuda.current_stream().wait_stream(side)
        # pieces of the keys are chosen by the host's bound at capture time: other orders of the same sums
        assert (out.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max(), i
        assert torch.equal(caches[0].lengths, caches[1].lengths)
    assert torch.equal(caches[0].k8.view(torch.uint8), caches[1].k8.view(torch.uint8))
    assert caches[0].lengths.tolist() == [196, 126]


@gpu
def test_refusals():
    from vit_amd import ops
    cache, _, _ = filled(2, 2, 64, [10, 20])
    k = tokens(2, 3, 2, 64).cuda()
    for bad in (k.float(), k[:1], k[:, :0], k[..., :32], k.transpose(1, 2), k[:, :, :1], k[0]):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.kv8_append_(cache, bad, bad)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.kv8_attn(bad, cache)
    odd = torch.zeros(2 * 3 * 2 * 64 + 1, dtype=BF16, device="cuda")[1:].view(2, 3, 2, 64)
    with pytest.raises(RuntimeError):
        ops.kv8_attn(odd, cache)
    with pytest.raises(ValueError):
        ops.kv8_attn(k, cache, new=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        ops.kv8_attn(k, cache, new=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError):
        ops.kv8_attn(k, cache, tokens_per_timestep=-1)
    with pytest.raises(RuntimeError):
        ops.kv8_attn(tokens(1, 1, 1, 32).cuda(), ops.KVCache8.empty(1, 1, 32, 64, "cuda"))        # head dim
    with pytest.raises(ValueError):
        ops.KVCache8(cache.k8[:, :, :60], cache.v8, cache.k_scale, cache.v_scale, cache.k_open, cache.v_open, cache.lengths)
    with pytest.raises((ValueError, TypeError)):
        ops.KVCache8(cache.k8, cache.v8, cache.k_scale[:1], cache.v_scale, cache.k_open, cache.v_open, cache.lengths)


def test_refusals_without_a_gpu():
    from vit_amd import _lib, ops
    with pytest.raises(_lib.VitAmdError):
        ops.KVCache8.empty(1, 1, 64, 64, "cpu")
    with pytest.raises(ValueError):
        ops.KVCache8(torch.zeros(1, 1, 60, 64), *([None] * 6))


@gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [40, 130])
def test_attention_of_more_streams_than_there_are_compute_units(n, hd):
    """The other launch shape, with full and ragged row tiles; then a bad last token, which only the last query sees."""
    from vit_amd import ops
    B, H = 66, 4
    lens = [n + 1 + (37 * b) % 90 for b in range(B)]
    cache, k, v = filled(B, H, hd, lens, steps=(0.5, 1.0))
    q = tokens(B, n, H, hd, "mu.q", 3.0)
    out = ops.kv8_attn(q.cuda(), cache, tokens_per_timestep=1)
    some = [0, 1, 33, B - 1]

    class Some:
        heads, lengths = H, cache.lengths[some]
    for name in ("k8", "v8", "k_scale", "v_scale", "k_open", "v_open"):
        t = getattr(cache, name)
        setattr(Some, name, t.view(torch.uint8)[some].view(t.dtype) if t.dtype == torch.float8_e4m3fn else t[some])
    close(out[some], *attention(q[some], Some, [n] * len(some), 1))
    assert torch.isfinite(out).all()
    dirty = ops.KVCache8.empty(B, H, hd, max(lens), "cuda")
    for b, m in enumerate(lens):
        v[b, m - 1, :, 3] = float("nan")
    new = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ops.kv8_append_(dirty, k.cuda(), v.cuda(), new=new)
    got = ops.kv8_attn(q.cuda(), dirty, tokens_per_timestep=1)
    assert torch.equal(got[:, :-1, :, :3], out[:, :-1, :, :3]) and torch.equal(got[:, :-1, :, 4:], out[:, :-1, :, 4:])
    assert torch.isfinite(got[:, :-1]).all() and torch.isnan(got[:, -1, :, 3]).all()
