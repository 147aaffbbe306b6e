"""The token operators behind a foveated patch embedding, as a program calls them: layer norm, rotary positions with several
axes, and cross attention to an encoder's states of another length.

Sizes are those of the vision-transformer configurations that the package's patch embeddings serve (384 channels in 6 heads, 1280 in 20,
64 channels a head; 64 or 256 tokens per fixation and a class token; 4 or 8 fixations), and generic ones around them.

  norm     layer norm over the last axis; a training pass also gives the gradients of the input, the weight and the bias
  rotary   [B, L, H, D] rotated by positions of up to three axes; a training pass also gives the input's gradient
  attend   queries [B, Lq, H, D] over states [B, Lk, Hkv, D]; a training pass also gives the gradients of all three

With `own` false, `run` computes the formulas with elementary torch operations in float32; with `own` true it calls
fovi_b200.tokens.  `exact` states the definitions in 64 bits.
"""
import math

import torch

own = False
DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # training the small transformer: every token of 256 images x 4 fixations, 256 tokens and a class token each
        dict(name="norm_train", op="norm", train=True, dtype="bf16", rows=256 * 4 * 257, dim=384),
        # the large transformer's width in float32, an uneven last batch
        dict(name="norm_train_f32", op="norm", train=True, dtype="f32", rows=16 * 257 - 13, dim=1280),
        # serving one fixation of 64 tokens and a class token: latency
        dict(name="norm_one", op="norm", train=False, dtype="bf16", rows=65, dim=384),
        # height and width: every image's tokens lie where its own fixation put them; the class token has no place
        dict(name="rotary_train", op="rotary", train=True, dtype="bf16", batch=256, tokens=257, prefix=1, heads=6, dim=64, axes=2, shared=False, pairing="halves"),
        # time, height and width over the tokens of four fixations, neighbouring channels paired, five tokens without a place
        dict(name="rotary_time", op="rotary", train=True, dtype="f32", batch=7, tokens=4 * 256 + 5, prefix=5, heads=20, dim=64, axes=3, shared=True, pairing="pairs"),
        # one new query token of the large transformer: latency
        dict(name="rotary_one", op="rotary", train=False, dtype="bf16", batch=1, tokens=1, prefix=0, heads=20, dim=64, axes=3, shared=False, pairing="halves"),
        # serving: one query token per image over the states of eight fixations, ragged lengths
        dict(name="attend_one", op="attend", train=False, dtype="bf16", batch=64, queries=1, keys=8 * 257, heads=20, kv_heads=20, dim=64, lengths=True, masked=False),
        # training: one fixation's tokens read the states of four
        dict(name="attend_train", op="attend", train=True, dtype="bf16", batch=256, queries=257, keys=4 * 257, heads=6, kv_heads=6, dim=64, lengths=False, masked=False),
        # evaluation over the long history of 64 fixations
        dict(name="attend_long", op="attend", train=False, dtype="bf16", batch=8, queries=257, keys=64 * 257, heads=20, kv_heads=20, dim=64, lengths=False, masked=False),
        # training with shared state heads of 128 channels and states dropped at random, odd lengths
        dict(name="attend_masked", op="attend", train=True, dtype="bf16", batch=24, queries=131, keys=701, heads=16, kv_heads=4, dim=128, lengths=True, masked=True),
        # training: sixteen learned queries read one fixation out
        dict(name="attend_few", op="attend", train=True, dtype="bf16", batch=512, queries=16, keys=261, heads=6, kv_heads=6, dim=64, lengths=False, masked=False),
        # parity runs in float32
        dict(name="attend_f32", op="attend", train=True, dtype="f32", batch=16, queries=65, keys=257, heads=6, kv_heads=6, dim=64, lengths=True, masked=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attend", "attend"])
    train = rng.random() < 0.6
    dtype = "bf16" if rng.random() < 0.7 else "f32"
    if op == "norm":
        dim = rng.choice([384, 1280, 768, _log(rng, 8, 4096)])
        rows = min(_log(rng, 1, 263168), 101056512 // dim // (1 if dtype == "bf16" else 2))
        return dict(op=op, train=train, dtype=dtype, rows=rows, dim=dim)
    if op == "rotary":
        heads, dim, tokens = rng.choice([6, 12, 16, 20]), rng.choice([64, 64, 32, 80, 128]), _log(rng, 1, 2061)
        prefix = rng.choice([0, 1, 5]) if tokens > 8 else 0
        batch = max(1, min(_log(rng, 1, 512), 25264128 // (tokens * heads * dim) // (1 if dtype == "bf16" else 2)))
        return dict(op=op, train=train, dtype=dtype, batch=batch, tokens=tokens, prefix=prefix, heads=heads, dim=dim, axes=rng.choice([1, 2, 3]),
                    shared=rng.random() < 0.5, pairing=rng.choice(["halves", "pairs"]))
    heads = rng.choice([6, 12, 16, 20])
    dim = rng.choice([64, 64, 64, 32, 80, 128])
    kv_heads = rng.choice([heads, heads, heads // 2, 1 if heads == 6 else heads // 4])
    queries, keys = _log(rng, 1, 514), _log(rng, 1, 16448)
    most = 256 * 6 * 257 * 1028 * 64 // (1 if dtype == "bf16" else 40)             # the largest listed case's products
    keys = max(1, min(keys, most // (heads * dim * queries)))
    batch = max(1, min(_log(rng, 1, 512), most // (heads * dim * queries * keys), 100000000 // (keys * kv_heads * dim)))
    return dict(op=op, train=train, dtype=dtype, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim,
                lengths=rng.random() < 0.5, masked=rng.random() < 0.3)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        # x and the upstream gradient read, y and the input's gradient written; weight, bias and their gradients in float32
        return dict(bytes=n * size * (4 if case["train"] else 2) + 4 * case["dim"] * (4 if case["train"] else 2), flops=n * (22 if case["train"] else 8))
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        places = (1 if case["shared"] else case["batch"]) * (case["tokens"] - case["prefix"]) * case["axes"]
        return dict(bytes=n * size * (4 if case["train"] else 2) + 4 * places, flops=n * 3 * (2 if case["train"] else 1))
    q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
    kv = 2 * case["batch"] * case["keys"] * case["kv_heads"] * case["dim"]
    products = case["batch"] * case["heads"] * case["queries"] * case["keys"] * case["dim"]
    share = 1.0
    if case["lengths"]:                 # lengths are uniform over 0 .. keys: what lies behind them need not be read
        share = 0.5
    mask = case["batch"] * case["keys"] if case["masked"] else 0
    if not case["train"]:
        return dict(bytes=size * (2 * q + share * kv) + mask, flops=4 * share * products)
    return dict(bytes=size * (4 * q + (1 + share) * kv) + mask, flops=14 * share * products)


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(1000003 * (int(seed) + 1))


def _frequencies(case):
    """(pairs of each axis, frequency of every pair): 2 pi / period for places in [-1, 1], periods 100^(j / n) of the axis's n pairs; time counts in whole steps."""
    pairs, axes = case["dim"] // 2, case["axes"]
    sections = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    f = []
    for a, n in enumerate(sections):
        unit = 1.0 if axes == 3 and a == 0 else 2 * math.pi
        f += [unit * 100.0 ** (-j / n) for j in range(n)]
    return tuple(sections), torch.tensor(f, dtype=torch.float32, device=DEVICE)


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16) * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "norm":
        # activations of a residual stream: channels of unequal spread and a mean of their own
        spread = torch.rand(case["dim"], generator=g, device=DEVICE) * 1.5 + 0.5
        s["x"] = normal(case["rows"], case["dim"]).mul_(spread.to(dt)).add_(normal(case["dim"], scale=0.5))
        s["weight"] = torch.rand(case["dim"], generator=g, device=DEVICE) + 0.5
        s["bias"] = 0.2 * torch.randn(case["dim"], generator=g, device=DEVICE)
        leaves = ("x", "weight", "bias")
        out = (case["rows"], case["dim"])
    elif case["op"] == "rotary":
        s["sections"], s["frequencies"] = _frequencies(case)
        n = case["tokens"] - case["prefix"]
        places = torch.rand((n, case["axes"]) if case["shared"] else (case["batch"], n, case["axes"]), generator=g, device=DEVICE) * 2 - 1
        if case["axes"] == 3:
            places[..., 0] = torch.floor(torch.arange(n, device=DEVICE) / 256)          # the fixation's number
        s["positions"] = places
        out = (case["batch"], case["tokens"], case["heads"], case["dim"])
        s["x"] = normal(*out)
        leaves = ("x",)
    else:
        B, H, D = case["batch"], case["heads"], case["dim"]
        out = (B, case["queries"], H, D)
        s["q"] = normal(*out, scale=1.5)
        s["k"] = normal(B, case["keys"], case["kv_heads"], D)
        s["v"] = normal(B, case["keys"], case["kv_heads"], D)
        s["key_lengths"] = torch.randint(0, case["keys"] + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32) if case["lengths"] else None
        s["key_mask"] = torch.rand((B, case["keys"]), generator=g, device=DEVICE) < 0.8 if case["masked"] else None
        leaves = ("q", "k", "v")
    if case["train"]:
        s["grad"] = normal(*out)
        for name in leaves:
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from fovi_b200 import tokens
    case = s["case"]
    if case["op"] == "norm":
        leaves = (s["x"], s["weight"], s["bias"])
        y = tokens.layer_norm(*leaves, eps=EPS)
    elif case["op"] == "rotary":
        leaves = (s["x"],)
        y = tokens.rotary(s["x"], s["positions"], s["frequencies"], s["sections"], prefix=case["prefix"], pairing=case["pairing"])
    else:
        leaves = (s["q"], s["k"], s["v"])
        y = tokens.cross_attention(*leaves, key_lengths=s["key_lengths"], key_mask=s["key_mask"])
    if not case["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, leaves, s["grad"])


@torch.no_grad()
def _run_plain(s):
    return dict(norm=_norm, rotary=_rotary, attend=_attend)[s["case"]["op"]](s)


def _norm(s):
    x, dt = s["x"].float(), s["x"].dtype
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    r = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xh = centred * r
    y = (xh * s["weight"] + s["bias"]).to(dt)
    if not s["case"]["train"]:
        return y
    dy = s["grad"].float()
    g = dy * s["weight"]
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, dx.to(dt), (dy * xh).sum(0), dy.sum(0)


def _turn(x, cos, sin, case):
    n, p = case["prefix"], cos.shape[-1]
    head, x = x[:, :n], x[:, n:].float()
    if case["pairing"] == "halves":
        u, v, rest = x[..., :p], x[..., p:2 * p], x[..., 2 * p:]
        y = torch.cat([u * cos - v * sin, v * cos + u * sin, rest], -1)
    else:
        u, v, rest = x[..., 0:2 * p:2], x[..., 1:2 * p:2], x[..., 2 * p:]
        y = torch.cat([torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2), rest], -1)
    return torch.cat([head, y.to(head.dtype)], 1)


def _rotary(s):
    case = s["case"]
    axis = torch.tensor([a for a, n in enumerate(s["sections"]) for _ in range(n)], device=DEVICE)
    angle = (s["positions"][..., axis] * s["frequencies"]).unsqueeze(-2)                # [(B,) L, 1, pairs]
    cos, sin = torch.cos(angle), torch.sin(angle)
    y = _turn(s["x"], cos, sin, case)
    return (y, _turn(s["grad"], cos, -sin, case)) if case["train"] else y


def _allowed(s):
    """[B, 1, 1, Lk] truth values: the keys that a query may read, or None for all."""
    case, ok = s["case"], None
    if s["key_lengths"] is not None:
        ok = torch.arange(case["keys"], device=DEVICE) < s["key_lengths"][:, None]
    if s["key_mask"] is not None:
        ok = s["key_mask"] if ok is None else ok & s["key_mask"]
    return None if ok is None else ok[:, None, None, :]


def _attend(s):
    case, dt = s["case"], s["q"].dtype
    B, H, D, G = case["batch"], case["heads"], case["dim"], case["kv_heads"]
    # the heads that share a state head stand side by side as rows
    def rows(t): return t.float().transpose(1, 2).reshape(B, G, -1, D)
    def heads(t): return t.reshape(B, H, -1, D).transpose(1, 2).to(dt)
    q, k, v = rows(s["q"]), rows(s["k"]), rows(s["v"])
    scale = D ** -0.5
    p = (q @ k.transpose(2, 3)).mul_(scale)
    ok = _allowed(s)
    if ok is not None:
        p = p.masked_fill_(~ok, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    o = heads(p @ v)
    if not case["train"]:
        return o
    do = rows(s["grad"])
    dv = p.transpose(2, 3) @ do
    ds = do @ v.transpose(2, 3)
    ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    def states(t): return t.transpose(1, 2).to(dt)
    return o, heads(ds @ k), states(ds.transpose(2, 3) @ q), states(dv)


# ------------------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return dict(norm=_exact_norm, rotary=_exact_rotary, attend=_exact_attend)[case["op"]](s)


def _exact_norm(s):
    weight, bias = (s[n].detach().double().requires_grad_(s["case"]["train"]) for n in ("weight", "bias"))
    outs, parts = [], []
    for x, g in zip(s["x"].detach().split(65536), s["grad"].split(65536) if s["case"]["train"] else s["x"].split(65536)):
        x = x.double().requires_grad_(s["case"]["train"])
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * weight + bias
        outs.append(y.detach())
        if s["case"]["train"]:
            parts.append(torch.autograd.grad(y, (x, weight, bias), g.double()))
    y = torch.cat(outs)
    if not s["case"]["train"]:
        return y
    return y, torch.cat([p[0] for p in parts]), sum(p[1] for p in parts), sum(p[2] for p in parts)


def _exact_rotary(s):
    case = s["case"]
    n, pairs = case["prefix"], len(s["frequencies"])
    which = [a for a, m in enumerate(s["sections"]) for _ in range(m)]
    angle = s["positions"].double()[..., which] * s["frequencies"].double()
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(-2)                    # a pair is a complex number
    first = torch.arange(pairs, device=DEVICE) * (1 if case["pairing"] == "halves" else 2)
    second = first + (pairs if case["pairing"] == "halves" else 1)

    def apply(x, turn):
        y = x.detach().double().clone()
        z = torch.complex(y[:, n:, :, first], y[:, n:, :, second]) * turn
        y[:, n:, :, first] = z.real
        y[:, n:, :, second] = z.imag
        return y

    y = apply(s["x"], turn)
    return (y, apply(s["grad"], turn.conj())) if case["train"] else y


def _exact_attend(s):
    case = s["case"]
    share, train = case["heads"] // case["kv_heads"], case["train"]
    ok = _allowed(s)
    one = case["heads"] * case["queries"] * case["keys"]
    step = max(1, (1 << 28) // one)                                                      # samples at a time: 2 GB of scores
    got = []
    for b in range(0, case["batch"], step):
        q, k, v = (s[n].detach()[b:b + step].double().requires_grad_(train) for n in ("q", "k", "v"))
        scores = torch.einsum("bqhd,bkhd->bhqk", q, k.repeat_interleave(share, 2)) / math.sqrt(case["dim"])
        if ok is not None:
            here = ok[b:b + step]
            scores = scores.masked_fill(~here, float("-inf"))
            empty = ~here.any(-1, keepdim=True)
            p = torch.softmax(scores.masked_fill(empty, 0.0), -1).masked_fill(empty, 0.0)
        else:
            p = torch.softmax(scores, -1)
        o = torch.einsum("bhqk,bkhd->bqhd", p, v.repeat_interleave(share, 2))
        got.append((o.detach(),) + (torch.autograd.grad(o, (q, k, v), s["grad"][b:b + step].double()) if train else ()))
        del scores, p, o
    got = tuple(torch.cat(t) for t in zip(*got))
    return got if train else got[0]
