"""GPU: attention over the 8-bit cache where it can go wrong without a wrong answer showing in ordinary inputs: NaN that
queries do see, whatever the launch shape."""
import pytest
import torch

from oracle import ref_cpu as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def tokens(B, n, H, hd, name, scale=2.0):
    return R.hashed_uniform(name, (B, n, H, hd), scale).to(BF16)


def cache_of(k, v, capacity=None):
    from vit_amd import ops
    cache = ops.KVCache8.empty(k.shape[0], k.shape[2], k.shape[3], capacity or k.shape[1], "cuda")
    return ops.kv8_append_(cache, k.cuda(), v.cuda())


# (tokens held, queries): few rows in one piece and in several, many rows in one piece (both tile shapes) and in several
SHAPES = [(200, 1), (2900, 1), (2900, 16), (200, 64), (200, 150), (2900, 64), (2900, 150)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("total,n", SHAPES)
def test_a_nan_query_gives_nan_and_no_other_row_changes(total, n, hd):
    from vit_amd import ops
    B, H = 2, 2
    cache = cache_of(tokens(B, total, H, hd, "e.k"), tokens(B, total, H, hd, "e.v"))
    q = tokens(B, n, H, hd, "e.q").cuda()
    clean = ops.kv8_attn(q, cache, tokens_per_timestep=1)
    assert torch.isfinite(clean).all()
    q[1, n - 1, 0, 5] = float("nan")
    got = ops.kv8_attn(q, cache, tokens_per_timestep=1)
    assert torch.isnan(got[1, n - 1, 0]).all()
    got[1, n - 1, 0] = clean[1, n - 1, 0]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("total,n", SHAPES)
def test_a_block_of_nan_keys_reaches_every_query_that_sees_it(total, n, hd):
    """A wave or a piece of the keys may hold nothing but such a block; its place makes it the first, a middle or the last
    one of the tokens."""
    from vit_amd import ops
    B, H = 1, 2
    k, v, q = tokens(B, total, H, hd, "b.k"), tokens(B, total, H, hd, "b.v"), tokens(B, n, H, hd, "b.q").cuda()
    clean = ops.kv8_attn(q, cache_of(k, v), tokens_per_timestep=1)
    for block in sorted({0, 1, total // 64 - 1}):
        bad = k.clone()
        bad[:, 64 * block:64 * block + 64, 1] = float("nan")
        got = ops.kv8_attn(q, cache_of(bad, v), tokens_per_timestep=1)
        sees = total - n + torch.arange(n) >= 64 * block
        assert torch.isnan(got[0, sees, 1]).all(), block
        assert torch.equal(got[0, ~sees, 1], clean[0, ~sees, 1]) and torch.equal(got[:, :, 0], clean[:, :, 0]), block


@pytest.mark.parametrize("n", [1, 17, 140])
def test_a_stream_of_one_nan_token_beside_streams_without_tokens(n):
    from vit_amd import ops
    hd = 64
    k, v, q = tokens(3, n, 1, hd, "o.k"), tokens(3, n, 1, hd, "o.v"), tokens(3, n, 1, hd, "o.q").cuda()
    k[1, 0] = float("nan")
    cache = ops.KVCache8.empty(3, 1, hd, 4096, "cuda")
    new = torch.tensor([0, 1, n], dtype=torch.int32, device="cuda")
    ops.kv8_append_(cache, k.cuda(), v.cuda(), new=new)
    for bound in (n, 4096):                                   # the host's bound decides on the pieces
        cache.max_len = bound
        got = ops.kv8_attn(q, cache, new=new)
        assert bool((got[0] == 0).all()) and bool((got[1, 1:] == 0).all())
        assert torch.isnan(got[1, 0]).all() and torch.isfinite(got[2]).all()


@pytest.mark.parametrize("n", [1, 64])
@pytest.mark.parametrize("total", [200, 2900])
def test_a_nan_value_whose_weight_underflows_is_not_lost(total, n):
    """Token 3's score lies some hundred below the others': its weight is zero in f32, and zero times NaN is NaN in every
    launch shape."""
    from vit_amd import ops
    hd = 64
    k, v, q = (torch.ones(1, m, 1, hd, dtype=BF16) for m in (total, total, n))
    k[0, :64] = -4.0                                           # whole blocks apart: waves and pieces of their own
    v[0, 3, 0, 7] = float("nan")
    got = ops.kv8_attn(q.cuda() * 4, cache_of(k, v), scale=1.0)
    assert torch.isnan(got[0, :, 0, 7]).all()
    got[..., 7] = 1.0
    assert bool((got == 1.0).all())


@pytest.mark.parametrize("heads,group", [(512, 1), (1, 1024)])
def test_a_maximum_that_stays_fades_nothing(heads, group):
    """All keys alike, scores of some thousand: every weight is the same, so the result is the share of values that are one
    (a half), however many tiles come after the one that set the maximum.  Few rows, many heads: one piece of the keys, four
    waves; many rows: one workgroup walks all 512 tiles.  A weight is rounded to bf16 and so is the result: 2^-8 of it each."""
    from vit_amd import ops
    hd, total, n = 64, 32768, 1 if group == 1 else 64
    code = lambda x: int(torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8))      # noqa: E731
    k8 = torch.full((1, heads, total, hd), code(3.5), dtype=torch.uint8, device="cuda")
    v8 = torch.zeros(1, heads, total, hd, dtype=torch.uint8, device="cuda")
    v8[:, :, :total // 2] = code(1.0)
    ones = torch.ones(1, heads, total // 64, device="cuda")
    opened = torch.zeros(1, heads, 64, hd, dtype=BF16, device="cuda")
    cache = ops.KVCache8(k8.view(torch.float8_e4m3fn), v8.view(torch.float8_e4m3fn), ones, ones.clone(), opened, opened.clone(),
                         torch.full((1,), total, dtype=torch.int32, device="cuda"))
    heights = 3.0 + torch.arange(heads * group, device="cuda") % 32 / 64.0               # exact in bf16, other scores for each
    q = heights.view(1, 1, -1, 1).expand(1, n, heads * group, hd).contiguous().to(BF16)
    out = ops.kv8_attn(q, cache, scale=37.0).float()
    worst = (out - 0.5).abs().max().item()
    assert worst <= 2 * 2.0 ** -8 * 0.5 + 1e-5, worst


def test_padded_appends_are_refused_only_when_a_stream_is_full(monkeypatch):
    """The host's bound counts the padding of ragged appends; when it passes the capacity the lengths themselves decide."""
    from vit_amd import ops
    B, H, hd, n = 3, 1, 64, 40
    cache, twin = (ops.KVCache8.empty(B, H, hd, 128, "cuda") for _ in range(2))
    k, v = tokens(B, n, H, hd, "p.k").cuda(), tokens(B, n, H, hd, "p.v").cuda()
    counts = [[40, 0, 5], [0, 40, 5], [40, 0, 5], [0, 40, 5], [0, 0, 5], [0, 0, 0], [40, 40, 5]]
    lens = [0] * B
    for row in counts:                                         # 280 padded tokens, at most 120 in a stream
        new = torch.tensor(row, dtype=torch.int32, device="cuda")
        ops.kv8_append_(cache, k, v, new=new)
        lens = [x + y for x, y in zip(lens, row)]
        assert cache.lengths.tolist() == lens and max(lens) <= cache.max_len <= cache.capacity
        for b, m in enumerate(row):                            # the same tokens, each stream by itself, never padded
            if m:
                one = torch.zeros(B, dtype=torch.int32, device="cuda")
                one[b] = m
                twin.max_len = max(lens) - m
                ops.kv8_append_(twin, k[:, :m], v[:, :m], new=one)
    assert lens == [120, 120, 30]
    for name in ("k8", "v8", "k_scale", "v_scale", "k_open", "v_open", "lengths"):
        x, y = getattr(cache, name), getattr(twin, name)
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
    with pytest.raises(ValueError):                            # stream 1 would hold 129
        ops.kv8_append_(cache, k, v, new=torch.tensor([0, 9, 0], dtype=torch.int32, device="cuda"))
    assert cache.lengths.tolist() == lens
    ops.kv8_append_(cache, k, v, new=torch.tensor([8, -3, 40], dtype=torch.int32, device="cuda"))
    assert cache.lengths.tolist() == [128, 120, 70]
    with pytest.raises(ValueError):
        ops.kv8_append_(cache, k[:, :1], v[:, :1])
    with monkeypatch.context() as m:                           # a capture must not ask the device
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(ValueError):
            ops.kv8_append_(cache, k, v, new=torch.zeros(B, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError):
            cache.sync_length()
    cache.lengths.copy_(torch.tensor([3, 70, 0]))
    assert cache.sync_length() == 70 == cache.max_len
