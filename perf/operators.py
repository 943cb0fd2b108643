"""Cases, plain forms and exact results of the predictor's sequence operators.

Three operators, in the forms a program meets them:

  gated delta rule    S_t = a_t S_{t-1} (I - b_t k_t k_t^T) + b_t v_t k_t^T,   o_t = S_t q_t
      delta_fwd       a whole sequence, with or without a carried state
      delta_train     a whole sequence with the gradients of every input
      delta_step      one token per stream, the state updated in place
  8-bit key/value cache, one power-of-two scale per block of 64 tokens and head; the open block stays in bfloat16
      kv8_append      tokens written behind the streams' lengths, blocks quantised as they fill
      kv8_attend      the newest tokens of every stream attend over its cache
  gated layer norm    y = LayerNorm((o * gate) * silu(g)) with the gradients of all inputs, any width
      gated_norm

`own` False computes the plain forms (elementary torch operations in 32 bits), True calls vit_amd.
"""
import math

import torch

own = False

BLOCK = 64            # tokens that share one scale
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one timestep of one video stream (256 patches + action + state) through the memory layer, state carried
        dict(name="delta_fwd_timestep", kind="delta_fwd", B=1, L=258, H=8, hd=128, type="bf16", state=True),
        # the memory layer over 8 timesteps of context, the world model's inference batch
        dict(name="delta_fwd_context", kind="delta_fwd", B=64, L=2064, H=8, hd=128, type="f32", state=False),
        # training the predictor's memory layer on 5 timesteps
        dict(name="delta_train_f32", kind="delta_train", B=4, L=1290, H=8, hd=128, type="f32", state=False),
        # training with 16 narrow heads, an odd length and a carried state, activations in bfloat16
        dict(name="delta_train_bf16_odd", kind="delta_train", B=3, L=517, H=16, hd=64, type="bf16", state=True),
        # one token of one stream: latency
        dict(name="delta_step_one", kind="delta_step", B=1, H=8, hd=128, type="f32"),
        # one token of each of many streams: the states' bandwidth
        dict(name="delta_step_many", kind="delta_step", B=256, H=8, hd=128, type="bf16"),
        # one new token per stream, ragged and long caches, four query heads to a key/value head
        dict(name="kv8_attend_token", kind="kv8_attend", B=32, H=8, group=4, hd=128, n=1, length=8256, tpt=1, ragged=True),
        # a new timestep of every stream attends block-causally over 8 timesteps
        dict(name="kv8_attend_timestep", kind="kv8_attend", B=16, H=8, group=1, hd=128, n=258, length=2064, tpt=258, ragged=True),
        # single tokens after an odd prompt
        dict(name="kv8_append_tokens", kind="kv8_append", B=16, H=8, hd=128, prompt=61, n=1, steps=4),
        # the timesteps of a context, one append each
        dict(name="kv8_append_timesteps", kind="kv8_append", B=16, H=8, hd=128, prompt=1290, n=258, steps=3),
        # output stage of the memory layer, forward and backward, the training batch
        dict(name="gated_norm_1024", kind="gated_norm", M=16512, D=1024, type="f32"),
        # a narrower layer on few rows, bfloat16 activations
        dict(name="gated_norm_384_odd", kind="gated_norm", M=197, D=384, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta_fwd", "delta_train", "delta_step", "kv8_append", "kv8_attend", "gated_norm"])
    hd, typ = rng.choice([64, 128]), rng.choice(["f32", "bf16"])
    if kind == "delta_fwd":
        L, H = _log(rng, 1, 4200), rng.randint(1, 16)
        B = max(1, min(_log(rng, 1, 64), 1056000 // (L * H)))
        return dict(kind=kind, B=B, L=L, H=H, hd=hd, type=typ, state=rng.random() < 0.5)
    if kind == "delta_train":
        L, H = _log(rng, 1, 2600), rng.randint(1, 16)
        B = max(1, min(_log(rng, 1, 16), 41000 // (L * H)))
        return dict(kind=kind, B=B, L=L, H=H, hd=hd, type=typ, state=rng.random() < 0.5)
    if kind == "delta_step":
        return dict(kind=kind, B=_log(rng, 1, 256), H=rng.randint(1, 8), hd=hd, type=typ)
    if kind == "kv8_append":
        n = _log(rng, 1, 300)
        return dict(kind=kind, B=rng.randint(1, 16), H=rng.randint(1, 8), hd=hd, prompt=_log(rng, 1, 1290), n=n,
                    steps=rng.randint(1, 3))
    if kind == "kv8_attend":
        many = rng.random() < 0.5
        n = _log(rng, 20, 258) if many else rng.randint(1, 4)
        return dict(kind=kind, B=rng.randint(1, 16), H=rng.randint(1, 8), group=1 if many else rng.choice([1, 2, 4]), hd=hd,
                    n=n, length=n + _log(rng, 1, 1800 if many else 8000), tpt=rng.choice([0, 1, n]), ragged=rng.random() < 0.7)
    return dict(kind=kind, M=_log(rng, 1, 16512), D=4 * _log(rng, 8, 256), type=typ)


def _lengths(case):
    """Tokens held by every stream, and how many of them are new.  Ragged: from the full length down to about half of
    it; the last stream has fewer new tokens than the others (none where the call brings one)."""
    B, n, length = case["B"], case["n"], case["length"]
    if not case["ragged"]:
        return [length] * B, [n] * B
    lens = [max(n, length - (length - n) * i // (2 * B) - 7 * (i % 3)) for i in range(B)]
    new = [n] * B
    if B > 1:
        lens[-1] -= n - n // 2
        new[-1] = n // 2
    return lens, new


def _visible(case):
    """Query-key pairs that the mask leaves, over all streams, and the tokens that are read."""
    lens, new = _lengths(case)
    pairs = 0
    for total, m in zip(lens, new):
        for i in range(m):
            p, t = total - m + i, case["tpt"]
            pairs += total if t == 0 else min(total, (p // t + 1) * t)
    return pairs, sum(t for t, m in zip(lens, new) if m)


def work(case):
    kind = case["kind"]
    if kind == "kv8_attend":
        pairs, read = _visible(case)
        B, n, H, G, hd = (case[x] for x in ("B", "n", "H", "group", "hd"))
        return {"bytes": read * H * hd * 2 + 2 * 2 * B * n * H * G * hd, "flops": 4.0 * pairs * H * G * hd}
    if kind == "kv8_append":
        tokens = case["B"] * (case["prompt"] + case["n"] * case["steps"]) * case["H"] * case["hd"]
        return {"bytes": 2 * tokens * 3, "flops": 4.0 * tokens}          # two bytes read, one written, keys and values
    es = TYPES[case["type"]].itemsize
    if kind == "gated_norm":
        n = case["M"] * case["D"]
        return {"bytes": n * es * (3 + 1 + 1 + 3 + 3), "flops": 40.0 * n}  # forward: 3 in, 1 out; backward: dy and 3 in, 3 out
    B, H, hd = case["B"], case["H"], case["hd"]
    states = 4 * B * H * hd * hd
    if kind == "delta_step":
        return {"bytes": 2 * states + B * H * (4 * hd * es + 8), "flops": 6.0 * B * H * hd * hd}
    rows = B * case["L"] * H
    # the recurrence as it stands: S k, the rank-1 update, S q; the gradient: twice that and the states again
    if kind == "delta_fwd":
        return {"bytes": rows * (4 * hd * es + 8) + states * (2 if case["state"] else 1), "flops": 6.0 * rows * hd * hd}
    return {"bytes": rows * ((4 + 4 + 3) * hd * es + 8 + 16) + states * (6 if case["state"] else 3),
            "flops": 24.0 * rows * hd * hd}


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """[..., blocks, BLOCK, hd] -> e4m3 codes and the scale of every block, the smallest power of two (2^-100 at least)
    that brings the block's largest magnitude to 448 or below."""
    amax = x.float().abs().amax((-1, -2))
    m, e = torch.frexp(amax)                                             # amax = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.clamp(min=-100)), 1.0)
    return (x.float() / scale[..., None, None]).to(F8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind.startswith("delta"):
        B, H, hd, t = case["B"], case["H"], case["hd"], TYPES[case["type"]]
        lead = (B,) if kind == "delta_step" else (B, case["L"])
        # as the layer makes them: SiLU behind the convolution, q and k normalised over the whole inner width
        x = {n: torch.nn.functional.silu(rand(*lead, H * hd)) for n in "qkv"}
        s = {"case": case, "v": x["v"].view(*lead, H, hd).to(t)}
        for n in "qk":
            s[n] = (x[n] / x[n].norm(dim=-1, keepdim=True)).view(*lead, H, hd).to(t)
        s["alpha"] = torch.sigmoid(2 * rand(*lead, H) + 2)
        s["beta"] = torch.sigmoid(rand(*lead, H))
        s["state"] = 0.3 * rand(B, H, hd, hd) if kind == "delta_step" or case["state"] else None
        if kind == "delta_train":
            s["d_out"], s["d_state"] = rand(*lead, H, hd).to(t), 0.1 * rand(B, H, hd, hd)
            for n in ("q", "k", "v", "alpha", "beta"):
                s[n].requires_grad_()
            if case["state"]:
                s["state"].requires_grad_()
        return s
    if kind == "gated_norm":
        M, D, t = case["M"], case["D"], TYPES[case["type"]]
        s = {"case": case, "o": (0.2 * rand(M, D)).to(t), "gate": torch.nn.functional.silu(rand(M, D)).to(t),
             "g": (1.5 * rand(M, D)).to(t), "gamma": 1 + 0.1 * rand(D), "beta": 0.1 * rand(D), "dy": rand(M, D).to(t)}
        for n in ("o", "gate", "g", "gamma", "beta"):
            s[n].requires_grad_()
        return s
    B, H, hd = case["B"], case["H"], case["hd"]
    spread = 0.5 + torch.rand(H, 1, hd, generator=g, device="cuda") * 3    # some channels are larger than others
    if kind == "kv8_append":
        total = case["prompt"] + case["n"] * case["steps"]
        cap = -(-total // BLOCK) * BLOCK
        kv = {n: (rand(B, total, H, hd) * spread[:, 0]).to(BF16) for n in "kv"}
        lens = [0] * B
        full = {n: torch.zeros(B, H, cap // BLOCK, BLOCK, hd, device="cuda", dtype=BF16) for n in "kv"}
    else:
        lens, new = _lengths(case)
        cap = -(-max(lens) // BLOCK) * BLOCK
        held = torch.tensor(lens, device="cuda")[:, None, None, None]
        full = {}
        for n in "kv":
            x = (rand(B, H, cap, hd) * spread).to(BF16)
            x = torch.where(torch.arange(cap, device="cuda")[:, None] < held, x, torch.zeros((), device="cuda", dtype=BF16))
            full[n] = x.view(B, H, cap // BLOCK, BLOCK, hd)
    s = {"case": case, "lengths": torch.tensor(lens, device="cuda", dtype=torch.int32)}
    open_block = s["lengths"].long() // BLOCK
    for n in "kv":
        # whole blocks in 8 bits, the open one in bfloat16 beside them
        codes, scale = _quantise(full[n])
        whole = torch.arange(cap // BLOCK, device="cuda") < open_block[:, None]
        s[n + "8"] = torch.where(whole[:, None, :, None, None], codes.view(torch.uint8), 0).view(F8).view(B, H, cap, hd)
        s[n + "_scale"] = torch.where(whole[:, None], scale, 1.0)
        at = open_block.clamp(max=cap // BLOCK - 1)
        tail = full[n][torch.arange(B, device="cuda"), :, at]
        s[n + "_open"] = torch.where((open_block < cap // BLOCK)[:, None, None, None], tail, torch.zeros_like(tail)).contiguous()
    if kind == "kv8_append":
        s["k"], s["v"] = kv["k"], kv["v"]
        # every second stream's last append brings one token less than the others'
        s["last"] = torch.tensor([case["n"] - (i % 2) for i in range(B)], device="cuda", dtype=torch.int32)
    else:
        s["q"] = (rand(B, case["n"], H * case["group"], hd)).to(BF16)
        s["new"] = torch.tensor(new, device="cuda", dtype=torch.int32)
    return s


# ------------------------------------------------------------------ plain forms
def _delta(q, k, v, a, b, state):
    """The recurrence chunk by chunk (64 tokens), in 32 bits: inside a chunk the rank-1 updates u_i solve
    (I + strictly lower(diag(b) decay * K K^T)) U = diag(b) (V - diag(decay from the start) K S^T)."""
    B, L, H, hd = q.shape
    C = 64
    n = -(-L // C)

    def chunks(x, fill=0.0):
        x = torch.nn.functional.pad(x.float(), (0, 0) * (x.dim() - 2) + (0, n * C - L), value=fill)
        return x.view(B, n, C, *x.shape[2:]).transpose(2, 3)             # [B, n, H, C, ...]

    q, k, v, a, b = chunks(q), chunks(k), chunks(v), chunks(a, 1.0), chunks(b)
    logs = a.double().log().cumsum(-1)                                   # decays as differences of long sums
    below = torch.ones(C, C, device=q.device, dtype=torch.bool).tril()
    decay = torch.where(below, (logs[..., :, None] - logs[..., None, :]).masked_fill(~below, 0.0).exp().float(), 0.0)
    first = logs.exp().float()
    kk = (k @ k.transpose(-1, -2)) * decay * b[..., None]
    p = (q @ k.transpose(-1, -2)) * decay
    eye = torch.eye(C, device=q.device)
    T = torch.linalg.solve_triangular(kk.tril(-1) + eye, eye.expand_as(kk), upper=False, unitriangular=True)
    M = torch.zeros(B, H, hd, hd, device=q.device) if state is None else state.transpose(-1, -2)
    outs = []
    for c in range(n):
        g = first[:, c, :, :, None]
        u = T[:, c] @ (b[:, c, :, :, None] * (v[:, c] - g * (k[:, c] @ M)))
        outs.append(g * (q[:, c] @ M) + p[:, c] @ u)
        M = g[:, :, -1:] * M + (decay[:, c, :, -1, :, None] * k[:, c]).transpose(-1, -2) @ u
    out = torch.stack(outs, 1).transpose(2, 3).reshape(B, n * C, H, hd)[:, :L]
    return out, M.transpose(-1, -2)


def _plain_step(s):
    q, k, v = (s[n].float() for n in "qkv")
    a, b, S = s["alpha"][..., None], s["beta"][..., None], s["state"]
    u = b * (v - a * (S @ k[..., None])[..., 0])
    S.mul_(a[..., None]).add_(u[..., None] * k[..., None, :])
    return {"out": (S @ q[..., None])[..., 0].to(s["q"].dtype), "state": S}


def _seen(case, lengths, new, cap):
    """[B, n, cap]: which keys every query sees."""
    i = torch.arange(case["n"], device=lengths.device)
    p = (lengths - new)[:, None] + i
    end = lengths[:, None].expand_as(p)
    if case["tpt"]:
        end = torch.minimum(end, (p // case["tpt"] + 1) * case["tpt"])
    end = torch.where(i < new[:, None], end, 0)
    return torch.arange(cap, device=lengths.device) < end[..., None]


def _dense(s, n, to):
    """The cache's keys or values as numbers [B, H, capacity, hd]: whole blocks times their scale, the open block."""
    codes, scale, tail = s[n + "8"], s[n + "_scale"], s[n + "_open"]
    B, H, cap, hd = codes.shape
    x = codes.to(to).view(B, H, cap // BLOCK, BLOCK, hd) * scale.to(to)[..., None, None]
    at = s["lengths"].long() // BLOCK
    inside = at < cap // BLOCK
    here = torch.arange(cap // BLOCK, device=codes.device) == at[:, None]
    x = torch.where((here & inside[:, None])[:, None, :, None, None], tail.to(to)[:, :, None], x)
    return x.view(B, H, cap, hd)


def _attend(s, to):
    case = s["case"]
    B, n, Hq, hd = s["q"].shape
    H, G = case["H"], case["group"]
    q = s["q"].to(to).view(B, n, H, G, hd).permute(0, 2, 3, 1, 4).reshape(B, H, G * n, hd)
    k, v = _dense(s, "k", to), _dense(s, "v", to)
    seen = _seen(case, s["lengths"].long(), s["new"].long(), k.shape[2])
    seen = seen[:, None].expand(B, G, n, -1).reshape(B, 1, G * n, -1)
    x = (q @ k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = (e @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(B, H, G, n, hd).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, hd)


def _plain_append(s, k, v, new):
    """Tokens behind the streams' lengths: the open block and the new tokens side by side, whole blocks quantised."""
    B, n, H, hd = k.shape
    cap = s["k8"].shape[2]
    old = s["lengths"].long()
    total = old + new
    first = old // BLOCK
    span = -(-n // BLOCK) + 1                                            # blocks that n tokens can touch
    rows = torch.arange(B, device=k.device)[:, None]

    def source(place):
        src = place - old[:, None]                                       # which new token lands at a place
        return src.clamp(0, n - 1), (src >= 0) & (src < new[:, None])

    src, fresh = source(first[:, None] * BLOCK + torch.arange(span * BLOCK, device=k.device))
    open_src, open_fresh = source(total[:, None] // BLOCK * BLOCK + torch.arange(BLOCK, device=k.device))
    block = torch.arange(cap // BLOCK, device=k.device)
    j = block - first[:, None]                                           # of every block of the cache: its place in the span
    filled = (j >= 0) & (j < span) & ((block + 1) * BLOCK <= total[:, None])
    j = j.clamp(0, span - 1)
    for name, x in (("k", k), ("v", v)):
        tail = s[name + "_open"]
        buf = torch.nn.functional.pad(tail, (0, 0, 0, (span - 1) * BLOCK))
        buf = torch.where(fresh[:, None, :, None], x[rows, src].transpose(1, 2), buf).view(B, H, span, BLOCK, hd)
        codes, scale = _quantise(buf)
        dst = s[name + "8"].view(torch.uint8).view(B, H, cap // BLOCK, BLOCK, hd)
        put = codes.view(torch.uint8).transpose(1, 2)[rows, j].transpose(1, 2)
        dst.copy_(torch.where(filled[:, None, :, None, None], put, dst))
        put = scale.transpose(1, 2)[rows, j].transpose(1, 2)
        s[name + "_scale"].copy_(torch.where(filled[:, None], put, s[name + "_scale"]))
        tail.copy_(torch.where(open_fresh[:, None, :, None], x[rows, open_src].transpose(1, 2), tail))
    s["lengths"].add_(new.to(torch.int32))


def _norm(o, gate, g, gamma, beta):
    x = (o.float() * gate.float()) * (g.float() * torch.sigmoid(g.float()))
    x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * gamma + beta


CACHE = ("k8", "v8", "k_scale", "v_scale", "k_open", "v_open", "lengths")


def _cache(s):
    from vit_amd import ops
    return ops.KVCache8(*(s[n] for n in CACHE))


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from vit_amd import module_ops, ops
    if kind == "delta_fwd":
        args = [s[n] for n in ("q", "k", "v", "alpha", "beta", "state")]
        if own:
            out, state = ops.gated_delta_fwd(*args)
        else:
            out, state = _delta(*args)
            out = out.to(s["q"].dtype)
        return {"out": out, "state": state}
    if kind == "delta_train":
        names = ["q", "k", "v", "alpha", "beta"] + (["state"] if case["state"] else [])
        args = [s[n] for n in ("q", "k", "v", "alpha", "beta", "state")]
        if own:
            out, state = module_ops.gated_delta(*args)
        else:
            out, state = _delta(*args)
            out = out.to(s["q"].dtype)
        grads = torch.autograd.grad((out, state), [s[n] for n in names], (s["d_out"], s["d_state"]))
        return {"out": out, "state": state, **{"d_" + n: x for n, x in zip(names, grads)}}
    if kind == "delta_step":
        if own:
            out = ops.gated_delta_step_(s["q"], s["k"], s["v"], s["alpha"], s["beta"], s["state"])
            return {"out": out, "state": s["state"]}
        return _plain_step(s)
    if kind == "kv8_attend":
        if own:
            return {"out": ops.kv8_attn(s["q"], _cache(s), new=s["new"], tokens_per_timestep=case["tpt"])}
        return {"out": _attend(s, F32).to(BF16)}
    if kind == "kv8_append":
        cuts = [0] + [case["prompt"] + case["n"] * i for i in range(case["steps"] + 1)]
        if own:
            cache = _cache(s)
            cache.reset()
        else:
            s["lengths"].zero_()
        for i, (x, y) in enumerate(zip(cuts, cuts[1:])):
            k, v, last = s["k"][:, x:y], s["v"][:, x:y], i == case["steps"]
            if own:
                ops.kv8_append_(cache, k, v, new=s["last"] if last else None)
            else:
                _plain_append(s, k, v, s["last"].long() if last else torch.full_like(s["last"], y - x).long())
        return {n: s[n] for n in CACHE}
    names = ("o", "gate", "g", "gamma", "beta")
    if own:
        y = module_ops.gated_layernorm(*(s[n] for n in names), 1e-5)
    else:
        y = _norm(*(s[n] for n in names)).to(s["o"].dtype)
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y, **{"d_" + n: x for n, x in zip(names, grads)}}


# ------------------------------------------------------------------ exact results, 64 bits, from the definitions
def _exact_delta(s, train):
    q, k, v, a, b = (s[n].detach().double() for n in ("q", "k", "v", "alpha", "beta"))
    B, L, H, hd = q.shape
    S = torch.zeros(B, H, hd, hd, device=q.device, dtype=F64) if s["state"] is None else s["state"].detach().double()
    before, out = [], torch.empty_like(v)
    for t in range(L):
        if train:
            before.append(S)
        A, bt = a[:, t, :, None, None], b[:, t, :, None, None]
        S = A * (S - bt * (S @ k[:, t, :, :, None]) * k[:, t, :, None, :]) + bt * v[:, t, :, :, None] * k[:, t, :, None, :]
        out[:, t] = (S @ q[:, t, :, :, None])[..., 0]
    res = {"out": out, "state": S}
    if not train:
        return res
    d_out, G = s["d_out"].double(), s["d_state"].double()
    d = {n: torch.empty_like(x) for n, x in (("q", q), ("k", k), ("v", v), ("alpha", a), ("beta", b))}
    for t in reversed(range(L)):
        P, kt, vt, do = before[t], k[:, t, :, :, None], v[:, t, :, :, None], d_out[:, t, :, :, None]
        A, bt = a[:, t, :, None, None], b[:, t, :, None, None]
        Pk = P @ kt
        S = A * (P - bt * Pk @ kt.mT) + bt * vt @ kt.mT
        d["q"][:, t] = (S.mT @ do)[..., 0]
        G = G + do @ q[:, t, :, None, :]
        Gk = G @ kt
        d["v"][:, t] = (bt * Gk)[..., 0]
        d["alpha"][:, t] = (G * (P - bt * Pk @ kt.mT)).sum((-1, -2))
        d["beta"][:, t] = (Gk * (vt - A * Pk)).sum((-1, -2))
        d["k"][:, t] = (bt * (G.mT @ vt) - A * bt * (P.mT @ Gk + G.mT @ Pk))[..., 0]
        G = A * (G - bt * Gk @ kt.mT)
    res.update({"d_" + n: x for n, x in d.items()})
    if s["state"] is not None:
        res["d_state"] = G
    return res


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("delta_fwd", "delta_train"):
        cells = case["B"] * case["H"] * case["hd"] ** 2
        if cells * case["L"] > (2e9 if kind == "delta_train" else 6e10):
            return None
        return _exact_delta(s, kind == "delta_train")
    if kind == "delta_step":
        q, k, v, a, b, S = (s[n].double() for n in ("q", "k", "v", "alpha", "beta", "state"))
        I = torch.eye(case["hd"], device=q.device, dtype=F64)
        kk = k[..., :, None] * k[..., None, :]
        S = a[..., None, None] * (S @ (I - b[..., None, None] * kk)) + b[..., None, None] * v[..., :, None] * k[..., None, :]
        return {"out": (S @ q[..., None])[..., 0], "state": S}
    if kind == "kv8_attend":
        B, n, Hq, hd = s["q"].shape
        out = torch.zeros(B, n, Hq, hd, device="cuda", dtype=F64)
        lens, new = _lengths(case)
        for i in range(B):
            total, m, t = lens[i], new[i], case["tpt"]
            blocks = total // BLOCK
            x = {}
            for c in "kv":
                w = s[c + "8"][i, :, :blocks * BLOCK].double().view(case["H"], blocks, BLOCK, hd) * s[c + "_scale"][i, :, :blocks, None, None].double()
                x[c] = torch.cat([w.view(case["H"], -1, hd), s[c + "_open"][i, :, :total % BLOCK].double()], 1)
            for h in range(Hq):
                k, v = x["k"][h // case["group"]], x["v"][h // case["group"]]
                sc = (s["q"][i, :m, h].double() @ k.T) * hd ** -0.5
                if t:
                    p = torch.arange(total - m, total, device="cuda")
                    sc[torch.arange(total, device="cuda") // t > (p // t)[:, None]] = -math.inf
                out[i, :m, h] = torch.softmax(sc, -1) @ v
        return {"out": out}
    if kind == "kv8_append":
        # the codes, the scales and the open block of the tokens as they lie, from the definition of a block
        total = [case["prompt"] + case["n"] * (case["steps"] - 1) + int(m) for m in s["last"].tolist()]
        res = {"lengths": None}
        for c in "kv":
            codes, scales, tails = s[c + "8"].double(), s[c + "_scale"].double(), s[c + "_open"].double()
            for i, m in enumerate(total):
                x = s[c][i, :m].double().transpose(0, 1)
                w = x[:, :m // BLOCK * BLOCK].reshape(case["H"], -1, BLOCK, case["hd"])
                if w.shape[1]:
                    sc = torch.exp2(torch.ceil(torch.log2(w.abs().amax((-1, -2)) / 448)))
                    y = w / sc[..., None, None]
                    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                    codes[i, :, :m // BLOCK * BLOCK] = (torch.round(y / step) * step).reshape(case["H"], -1, case["hd"])
                    scales[i, :, :m // BLOCK] = sc
            res.update({c + "8": codes, c + "_scale": scales, c + "_open": None})
        return res
    o, gate, g, gamma, beta, dy = (s[n].detach().double() for n in ("o", "gate", "g", "gamma", "beta", "dy"))
    sig = 1 / (1 + torch.exp(-g))
    x = o * gate * g * sig
    mean, var = x.mean(-1, keepdim=True), x.var(-1, keepdim=True, unbiased=False)
    r = 1 / torch.sqrt(var + 1e-5)
    xn = (x - mean) * r
    w = dy * gamma
    dx = r * (w - w.mean(-1, keepdim=True) - xn * (w * xn).mean(-1, keepdim=True))
    return {"y": xn * gamma + beta, "d_o": dx * gate * g * sig, "d_gate": dx * o * g * sig,
            "d_g": dx * o * gate * sig * (1 + g * (1 - sig)), "d_gamma": (dy * xn).sum(0), "d_beta": dy.sum(0)}
