"""The operators of a token block behind a foveated patch embedding, as a program calls them: root-mean-square norm with the
residual's addition (with gradients, or with its result in 8 bits for serving), the product of 8-bit tokens with 8-bit weights,
and the gated feed-forward block.

Sizes are those of the vision-transformer configurations that the package's patch embeddings serve (384 channels, 1280 channels;
64 or 256 tokens per fixation and a class token; 4 fixations), with hidden layers of 8/3 or 4 times the channels, and generic ones
around them.

  rms    root-mean-square norm over the last axis, of x or of x + residual (which is returned too); a training pass also gives the
         gradients of x, the residual and the weight; the 8-bit form gives whole numbers of -127 .. 127 and a scale for each row
  int8   y[m, n] = scale[m] weight_scale[n] sum over k of q[m, k] weight[n, k] + bias[n]
  ffn    y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd; a training pass also gives the gradients of x, the weights and the biases

With `own` false, `run` computes the formulas with elementary torch operations in float32; with `own` true it calls
fovi_b200.tokens.  `exact` states the definitions in 64 bits.
"""
import math

import torch

own = False
DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
TINY = torch.finfo(torch.float32).tiny          # a row's scale is at least the smallest normal number: a row of zeros stays one


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # training the small transformer: the residual stream of 256 images x 4 fixations, 256 tokens and a class token each
        dict(name="rms_train", op="rms", form="train", residual=True, dtype="bf16", rows=256 * 4 * 257, dim=384),
        # the large transformer's width in float32, an uneven last batch, the first norm of a stack (nothing to add yet)
        dict(name="rms_train_f32", op="rms", form="train", residual=False, dtype="f32", rows=16 * 257 - 13, dim=1280),
        # serving a batch in 8 bits: the norm in front of a feed-forward block
        dict(name="rms_int8_batch", op="rms", form="int8", residual=True, dtype="bf16", rows=256 * 257, dim=1280),
        # the same for one query token: latency
        dict(name="rms_int8_one", op="rms", form="int8", residual=True, dtype="bf16", rows=1, dim=1280),
        # one query token through a projection of the large transformer: latency, the weights' bytes
        dict(name="int8_one", op="int8", tokens=1, dim=1280, out=5120, bias=True, out_dtype="bf16"),
        # serving a batch of 64 images
        dict(name="int8_batch", op="int8", tokens=64 * 257, dim=1280, out=5120, bias=True, out_dtype="bf16"),
        # sizes that divide nothing, result in float32
        dict(name="int8_odd", op="int8", tokens=1031, dim=1003, out=2731, bias=False, out_dtype="f32"),
        # one query token through the large transformer's block: latency, the weights' bytes
        dict(name="ffn_one", op="ffn", train=False, dtype="bf16", tokens=1, dim=1280, hidden=5120, bias=True, activation="silu"),
        # serving one fixation of 64 tokens and a class token
        dict(name="ffn_few", op="ffn", train=False, dtype="bf16", tokens=65, dim=1280, hidden=3416, bias=False, activation="silu"),
        # training the small transformer: 256 images of 256 tokens and a class token
        dict(name="ffn_train", op="ffn", train=True, dtype="bf16", tokens=256 * 257, dim=384, hidden=1024, bias=False, activation="silu"),
        # training the large transformer, with biases
        dict(name="ffn_train_large", op="ffn", train=True, dtype="bf16", tokens=64 * 257, dim=1280, hidden=5120, bias=True, activation="silu"),
        # parity runs in float32, an odd hidden layer, the other activation
        dict(name="ffn_train_f32", op="ffn", train=True, dtype="f32", tokens=4 * 257, dim=384, hidden=1021, bias=True, activation="gelu"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "int8", "ffn", "ffn"])
    if op == "rms":
        dtype = "bf16" if rng.random() < 0.7 else "f32"
        dim = rng.choice([384, 1280, 768, _log(rng, 8, 4096)])
        rows = min(_log(rng, 1, 263168), 101056512 // dim // (1 if dtype == "bf16" else 2))
        return dict(op=op, form=rng.choice(["train", "train", "serve", "int8"]), residual=rng.random() < 0.6, dtype=dtype, rows=rows, dim=dim)
    if op == "int8":
        dim, out = rng.choice([384, 1280, _log(rng, 16, 5120)]), rng.choice([384, 1280, 5120, _log(rng, 8, 5120)])
        tokens = max(1, min(_log(rng, 1, 65792), 64 * 257 * 1280 * 5120 // (dim * out)))
        return dict(op=op, tokens=tokens, dim=dim, out=out, bias=rng.random() < 0.5, out_dtype=rng.choice(["bf16", "bf16", "f32"]))
    train, dtype = rng.random() < 0.6, "bf16" if rng.random() < 0.75 else "f32"
    dim = rng.choice([384, 1280, _log(rng, 8, 2048)])
    hidden = rng.choice([dim * 4, -(-dim * 8 // 24) * 8, _log(rng, 8, 5504)])
    hidden = min(hidden, 5504)
    most = 64 * 257 * 1280 * 5120 // (1 if dtype == "bf16" else 40)
    tokens = max(1, min(_log(rng, 1, 65792), most // (dim * hidden)))
    return dict(op=op, train=train, dtype=dtype, tokens=tokens, dim=dim, hidden=hidden, bias=rng.random() < 0.5, activation=rng.choice(["silu", "silu", "gelu"]))


def work(case):
    if case["op"] == "rms":
        n, size, streams = case["rows"] * case["dim"], 2 if case["dtype"] == "bf16" else 4, 2 if case["residual"] else 0
        if case["form"] == "train":
            # x, y, the gradients of both; with a residual also it, the sum and the sum's gradient (the residual's gradient is x's); the weight and its gradient
            return dict(bytes=n * size * (4 + (streams and 3)) + 8 * case["dim"], flops=n * 14)
        out = n + 4 * case["rows"] if case["form"] == "int8" else n * size
        return dict(bytes=n * size * (1 + streams) + out + 4 * case["dim"], flops=n * 5)
    if case["op"] == "int8":
        m, k, n = case["tokens"], case["dim"], case["out"]
        return dict(bytes=m * k + n * k + m * n * (2 if case["out_dtype"] == "bf16" else 4) + 4 * (m + n), flops=2 * m * k * n)
    m, c, f, size = case["tokens"], case["dim"], case["hidden"], 2 if case["dtype"] == "bf16" else 4
    params = 3 * c * f + (2 * f + c if case["bias"] else 0)
    if not case["train"]:
        return dict(bytes=size * (2 * m * c + params), flops=6 * m * c * f)
    return dict(bytes=size * (4 * m * c + 2 * params), flops=18 * m * c * f)


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(1000003 * (int(seed) + 1))


def prepare(case, seed):
    g = _gen(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16) * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "rms":
        # a residual stream: channels of unequal spread and a mean of their own; what a block adds to it is smaller
        dt, shape = DTYPES[case["dtype"]], (case["rows"], case["dim"])
        spread = torch.rand(case["dim"], generator=g, device=DEVICE) * 1.5 + 0.5
        stream = normal(*shape, dtype=dt).mul_(spread.to(dt)).add_(normal(case["dim"], scale=0.5, dtype=dt))
        if case["residual"]:
            s["x"], s["residual"] = normal(*shape, scale=0.5, dtype=dt), stream
        else:
            s["x"], s["residual"] = stream, None
        s["weight"] = torch.rand(case["dim"], generator=g, device=DEVICE) + 0.5
        if case["form"] == "train":
            s["grad"] = normal(*shape, dtype=dt)
            s["grad_stream"] = normal(*shape, dtype=dt) if case["residual"] else None
            s["leaves"] = ["x", "residual", "weight"] if case["residual"] else ["x", "weight"]
    elif case["op"] == "int8":
        # whole numbers as a quantisation of normal values leaves them; rows start on 16-byte boundaries, as the quantising calls lay them out
        def whole(rows):
            buffer = torch.zeros(rows, -(-case["dim"] // 16) * 16, dtype=torch.int8, device=DEVICE)
            buffer[:, :case["dim"]] = normal(rows, case["dim"], scale=35.0).round_().clamp_(-127, 127)
            return buffer[:, :case["dim"]]

        s["q"], s["weight"] = whole(case["tokens"]), whole(case["out"])
        s["scale"] = (torch.rand(case["tokens"], generator=g, device=DEVICE) + 0.5) / 35
        s["weight_scale"] = (torch.rand(case["out"], generator=g, device=DEVICE) + 0.5) / (35 * math.sqrt(case["dim"]))
        s["bias"] = normal(case["out"], scale=0.2) if case["bias"] else None
    else:
        dt, m, c, f = DTYPES[case["dtype"]], case["tokens"], case["dim"], case["hidden"]
        s["x"] = normal(m, c, dtype=dt)                                                     # behind a norm
        s["gate_weight"], s["up_weight"] = (normal(f, c, scale=c ** -0.5, dtype=dt) for _ in range(2))
        s["down_weight"] = normal(c, f, scale=f ** -0.5, dtype=dt)
        names = ["gate_bias", "up_bias", "down_bias"]
        for name, n in zip(names, (f, f, c)):
            s[name] = normal(n, scale=0.2, dtype=dt) if case["bias"] else None
        if case["train"]:
            s["grad"] = normal(m, c, dtype=dt)
            s["leaves"] = ["x", "gate_weight", "up_weight", "down_weight"] + (names if case["bias"] else [])
    for name in s.get("leaves", ()):
        s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from fovi_b200 import tokens
    case = s["case"]
    if case["op"] == "int8":
        return tokens.linear_int8(s["q"], s["scale"], s["weight"], s["weight_scale"], s["bias"], out_dtype=DTYPES[case["out_dtype"]])
    if case["op"] == "ffn":
        y = tokens.gated_feed_forward(s["x"], s["gate_weight"], s["up_weight"], s["down_weight"], s["gate_bias"], s["up_bias"], s["down_bias"],
                                      activation=case["activation"])
        if not case["train"]:
            return y
        outs, grads = (y,), (s["grad"],)
    elif case["form"] == "int8":
        q, scale, *stream = tokens.rms_norm_int8(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        return (torch.mul(q, scale[:, None], out=values), scale, *stream)                  # the values that the 8 bits stand for
    elif case["residual"]:
        outs, grads = tokens.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"]), (s.get("grad"), s.get("grad_stream"))
    else:
        outs, grads = (tokens.rms_norm(s["x"], s["weight"], eps=EPS),), (s.get("grad"),)
    if "leaves" not in s:
        return outs
    return tuple(y.detach() for y in outs) + torch.autograd.grad(outs, [s[name] for name in s["leaves"]], grads)


@torch.no_grad()
def _run_plain(s):
    return dict(rms=_rms, int8=_int8, ffn=_ffn)[s["case"]["op"]](s)


def _rms(s):
    case, dt = s["case"], s["x"].dtype
    x, stream = s["x"].float(), ()
    if case["residual"]:
        total = (x + s["residual"].float()).to(dt)                                          # the stream as it is stored is what the norm is of
        x, stream = total.float(), (total,)
    r = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * r
    y = xh * s["weight"]
    if case["form"] == "int8":
        scale = (y.abs().amax(1, keepdim=True) / 127).clamp_min(TINY)
        q = torch.round(y / scale)
        return ((q * scale).to(torch.bfloat16), scale[:, 0], *stream)
    if case["form"] == "serve":
        return (y.to(dt), *stream)
    dy = s["grad"].float()
    g = dy * s["weight"]
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    if case["residual"]:
        dx = (dx + s["grad_stream"].float()).to(dt)
        return y.to(dt), total, dx, dx, (dy * xh).sum(0)
    return y.to(dt), dx.to(dt), (dy * xh).sum(0)


def _int8(s):
    y = s["q"].float() @ s["weight"].float().T * s["scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[s["case"]["out_dtype"]])


def _ffn(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[name].float() for name in ("x", "gate_weight", "up_weight", "down_weight"))
    g, u = x @ wg.T, x @ wu.T
    if case["bias"]:
        g, u = g + s["gate_bias"].float(), u + s["up_bias"].float()
    if case["activation"] == "silu":
        p = 1 / (1 + torch.exp(-g))
        a = g * p
    else:
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        a = g * p
    h = a * u
    y = h @ wd.T
    if case["bias"]:
        y = y + s["down_bias"].float()
    if not case["train"]:
        return y.to(dt)
    dy = s["grad"].float()
    dh = dy @ wd
    slope = p + a * (1 - p) if case["activation"] == "silu" else p + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    dg, du = dh * u * slope, dh * a
    grads = [dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h]
    if case["bias"]:
        grads += [dg.sum(0), du.sum(0), dy.sum(0)]
    return tuple(t.to(dt) for t in [y] + grads)


# ------------------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return dict(rms=_exact_rms, int8=_exact_int8, ffn=_exact_ffn)[case["op"]](s)


def _exact_rms(s):
    case, dt = s["case"], s["x"].dtype
    train = case["form"] == "train"
    weight = s["weight"].detach().double().requires_grad_(train)
    got = []
    for at in range(0, case["rows"], 65536):
        rows = slice(at, at + 65536)
        x = s["x"].detach()[rows].double()
        if case["residual"]:
            x = (x + s["residual"].detach()[rows].double()).to(dt).double()
        x.requires_grad_(train)
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight
        out = [y.detach()]
        if case["form"] == "int8":
            scale = torch.clamp(y.abs().max(-1).values / 127, min=TINY)
            out = [torch.round(y / scale[:, None]) * scale[:, None], scale]
        if case["residual"]:
            out.append(x.detach())
        if train:
            dx, dw = torch.autograd.grad(y, (x, weight), s["grad"][rows].double())
            if case["residual"]:
                dx = dx + s["grad_stream"][rows].double()
                out.append(dx)
            out += [dx, dw[None]]
        got.append(out)
    got = [torch.cat(t) for t in zip(*got)]
    if train:
        got[-1] = got[-1].sum(0)
    return tuple(got)


def _exact_int8(s):
    y = torch.einsum("mk,nk->mn", s["q"].double(), s["weight"].double())
    y = y * torch.outer(s["scale"].double(), s["weight_scale"].double())
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_ffn(s):
    case = s["case"]
    leaf = {name: None if t is None else t.detach().double().requires_grad_(case["train"]) for name, t in s.items()
            if name == "x" or name.endswith(("weight", "bias"))}
    act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
    linear = torch.nn.functional.linear
    hidden = act(linear(leaf["x"], leaf["gate_weight"], leaf["gate_bias"])) * linear(leaf["x"], leaf["up_weight"], leaf["up_bias"])
    y = linear(hidden, leaf["down_weight"], leaf["down_bias"])
    if not case["train"]:
        return y.detach()
    return (y.detach(),) + torch.autograd.grad(y, [leaf[name] for name in s["leaves"]], s["grad"].double())
