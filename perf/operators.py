"""Performance cases of the feed-forward operators: what a program that trains
or serves the feed-forward half of a residual block asks of them, from one
token to the largest batches.

  norm     s = x + residual; y = s / sqrt(mean(s^2) + eps) * weight, kept in
           the inputs' type or in e4m3 with a scale for each row or for each
           128 columns; and its gradients
  gated    h = act(x Wg + bg) * (x Wu + bu); and its gradients
  linear   y = act(x W + b) + residual; and its gradients
  dropout  y = residual + x * keep / (1 - p), keep drawn from a counter

W is [inputs x outputs], row-major.  A backward case is given what the forward
kept (the sum and 1/rms of the norm, the pre-activations of the products) in
the type it was kept in.  The sizes are the benchmark's own layer widths and
batches (256 to 4096, B = 64 to 4096), their fourfold hidden widths, round
decimal ones, and any others from `draw`.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
GROUP = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # the smallest scale: a row of zeros has it


def norm(name, direction, dtype, rows, cols, residual=True, out="same"):
    return {"name": name, "op": "norm", "dir": direction, "dtype": dtype, "rows": rows, "cols": cols,
            "residual": residual, "out": out}


def gated(name, direction, dtype, rows, inputs, hidden, act="silu", bias=False):
    return {"name": name, "op": "gated", "dir": direction, "dtype": dtype, "rows": rows, "inputs": inputs,
            "hidden": hidden, "act": act, "bias": bias}


def linear(name, direction, dtype, rows, inputs, outputs, act="identity", bias=True, residual=False):
    return {"name": name, "op": "linear", "dir": direction, "dtype": dtype, "rows": rows, "inputs": inputs,
            "outputs": outputs, "act": act, "bias": bias, "residual": residual}


def dropout(name, dtype, rows, cols, p, residual=True):
    return {"name": name, "op": "dropout", "dtype": dtype, "rows": rows, "cols": cols, "p": p, "residual": residual}


def listed():
    return [
        # one token of a generating model: the norm before a product in 8 bits; latency alone
        norm("norm_token_e4m3", "forward", "bf16", 1, 4096, out="e4m3_rows"),
        # a training batch's norm: memory traffic
        norm("norm_forward_8192", "forward", "bf16", 8192, 4096),
        # its gradients, the residual stream's among them
        norm("norm_backward_8192", "backward", "bf16", 8192, 4096),
        # one token through the gated layer: the weights are read once
        gated("gated_token", "forward", "bf16", 1, 4096, 16384),
        # a short prompt, no size a multiple of a tile
        gated("gated_300_rows", "forward", "f16", 300, 1000, 2500, act="gelu", bias=True),
        # a training batch, the pre-activations kept for the backward pass
        gated("gated_train_4096", "train", "bf16", 4096, 2048, 8192),
        # gradients of a large training batch: bound by the matrix cores
        gated("gated_backward_8192", "backward", "bf16", 8192, 4096, 16384),
        # the headline regression model's second layer at its batch, in the framework's first type
        linear("linear_f32_b64", "forward", "f32", 64, 1024, 1024, act="relu"),
        # sixteen sequences decoded together: the block's product back onto the residual stream
        linear("linear_16_rows", "forward", "bf16", 16, 16384, 4096, bias=False, residual=True),
        # a large classifier's round decimal widths, rows of 1500 elements that are not 16-byte aligned
        linear("linear_backward_2000", "backward", "bf16", 2000, 1500, 3000, act="gelu"),
        # the dropout of a training batch, added to the residual stream
        dropout("dropout_8192", "bf16", 8192, 4096, 0.1),
        # a minibatch of 100 images: its gradient's mask, drawn again
        dropout("dropout_b100", "f32", 100, 784, 0.2, residual=False),
    ]


# The most work of a drawn case, under the largest listed one's (4.4e12 flops in 16 bits, of which a
# ragged or 32-bit product does fewer a second).
MOST_FLOPS, MOST_FLOPS_F32, MOST_BYTES = 1.5e12, 1.5e11, 8e8


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width, log-uniform: half multiples of 64, a quarter round decimals, a quarter any number."""
    w, style = _log_int(rng, lo, hi), rng.random()
    if style < 0.5 and w >= 32:
        return max(64, (w + 32) // 64 * 64)
    if style < 0.75 and w >= 20:
        return w // 100 * 100 if w >= 200 else w // 10 * 10
    return w


def _rows(rng):
    """Rows, log-uniform from 1 to 8192: half powers of two, the rest any number."""
    return 2 ** rng.randint(0, 13) if rng.random() < 0.5 else _log_int(rng, 1, 8192)


def draw(rng):
    """One more case of the listed ranges."""
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= (MOST_FLOPS_F32 if c["dtype"] == "f32" else MOST_FLOPS) and w["bytes"] <= MOST_BYTES:
            return c


def _draw(rng):
    op = rng.choice(["norm", "norm", "gated", "gated", "gated", "linear", "linear", "linear", "dropout"])
    dtype, rows = rng.choice(["bf16", "bf16", "f16", "f32"]), _rows(rng)
    act = rng.choice(["silu", "gelu", "relu", "sigmoid", "tanh", "leaky_relu"])
    if op == "norm":
        c = norm("", rng.choice(["forward", "forward", "backward"]), dtype, rows, _width(rng, 16, 16384),
                 residual=rng.random() < 0.7)
        if c["dir"] == "forward":
            c["out"] = rng.choice(["same", "same", "e4m3_rows", "e4m3_groups"])
    elif op == "gated":
        c = gated("", rng.choice(["forward", "train", "backward"]), dtype, rows, _width(rng, 16, 4096),
                  _width(rng, 16, 16384), act=act, bias=rng.random() < 0.3)
    elif op == "linear":
        c = linear("", rng.choice(["forward", "forward", "backward"]), dtype, rows, _width(rng, 16, 16384),
                   _width(rng, 16, 4096), act=rng.choice(["identity", act]), bias=rng.random() < 0.6)
        c["residual"] = c["dir"] == "forward" and rng.random() < 0.5
    else:
        c = dropout("", dtype, rows, _width(rng, 16, 16384), rng.choice([0.1, 0.2, 0.5]), residual=rng.random() < 0.6)
    del c["name"]
    return c


def work(case):
    e, m = 4 if case["dtype"] == "f32" else 2, case["rows"]
    if case["op"] == "norm":
        n, r = m * case["cols"], case["residual"]
        if case["dir"] == "backward":  # dy, s, the sum's gradient; dx, dweight
            return {"bytes": n * e * (3 + r) + case["cols"] * 2 * e + 4 * m, "flops": 9 * n}
        out = {"same": n * e, "e4m3_rows": n + 4 * m, "e4m3_groups": n + 4 * m * -(-case["cols"] // GROUP)}[case["out"]]
        return {"bytes": n * e * (1 + 2 * r) + out + case["cols"] * e + 4 * m, "flops": 5 * n}
    if case["op"] == "dropout":
        return {"bytes": m * case["cols"] * e * (3 if case["residual"] else 2), "flops": 2 * m * case["cols"]}
    two = 2 if case["op"] == "gated" else 1
    k, n = case["inputs"], case["hidden"] if two == 2 else case["outputs"]
    b = two * n if case["bias"] else 0
    if case["dir"] == "backward":
        kept = two if two == 2 or case["act"] != "identity" else 0
        return {"bytes": e * (m * n * (1 + kept) + 2 * m * k + 2 * two * k * n + b), "flops": 4 * two * m * k * n}
    kept = two if case["dir"] == "train" else 0
    residual = m * n if case.get("residual") else 0
    return {"bytes": e * (m * k + two * k * n + m * n * (1 + kept) + residual + b), "flops": 2 * two * m * k * n}


# ---------------------------------------------------------------------------
# Inputs, from the seed alone (on the GPU, so that making them is quick).
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)).to(t)

    m, s = case["rows"], {}
    if case["op"] == "norm":
        c = case["cols"]
        # a residual stream has a few channels far above the others
        loud = 1 + 19 * (torch.rand(c, generator=g, device="cuda") < 0.005).float()
        s["weight"] = (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(t)
        if case["dir"] == "forward":
            s["x"] = normal(m, c)
            s["residual"] = (loud * torch.randn(m, c, generator=g, device="cuda")).to(t) if case["residual"] else None
        else:
            s["sum"] = (loud * torch.randn(m, c, generator=g, device="cuda")).to(t)
            s["rstd"] = torch.rsqrt((s["sum"].double() ** 2).mean(1) + EPS).float()
            s["dy"] = normal(m, c, scale=0.1)
            s["dsum"] = normal(m, c, scale=0.1) if case["residual"] else None
    elif case["op"] == "dropout":
        s["x"] = normal(m, case["cols"])
        s["residual"] = normal(m, case["cols"]) if case["residual"] else None
        s["seed"], s["offset"] = int(seed) * 7919 + 1, int(seed) % 1000003
    else:
        two = case["op"] == "gated"
        k, n = case["inputs"], case["hidden"] if two else case["outputs"]
        s["x"] = normal(m, k)
        s["w"] = [normal(k, n, scale=k ** -0.5) for _ in range(1 + two)]
        if case["dir"] == "backward":
            s["dy"] = normal(m, n, scale=0.1)
            s["pre"] = [normal(m, n) for _ in range(1 + two)] if two or case["act"] != "identity" else []
        else:
            s["b"] = [normal(n, scale=0.1) if case["bias"] else None for _ in range(1 + two)]
            s["residual"] = normal(m, n) if case.get("residual") else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["call"] = _calls(case, s)
    return s


def run(state):
    if own:
        return state["call"]()
    return {"norm": _plain_norm, "gated": _plain_gated, "linear": _plain_linear,
            "dropout": _plain_dropout}[state["case"]["op"]](state["case"], state)


# ---------------------------------------------------------------------------
# The framework's calls: a handle for the sizes, buffers for the outputs and
# the workspace, the current stream.
# ---------------------------------------------------------------------------
def _calls(case, s):
    from volta_amd import ops

    t, m = TYPES[case["dtype"]], case["rows"]
    stream = torch.cuda.current_stream().cuda_stream

    def new(*shape, dtype=t):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    def space(op, backward):
        n = op.workspace_bytes(backward=backward)
        return new(n, dtype=torch.uint8) if n else None

    if case["op"] == "norm":
        c, e4m3 = case["cols"], case["dir"] == "forward" and case["out"] != "same"
        groups = case["dir"] == "forward" and case["out"] == "e4m3_groups"
        op = ops.RmsNorm(m, c, case["dtype"], eps=EPS, out="e4m3" if e4m3 else "same", group=GROUP if groups else 0)
        if case["dir"] == "backward":
            out = {"dx": new(m, c), "dweight": new(c)}
            ws = space(op, True)

            def call():
                op.backward(s["dy"], s["sum"], s["rstd"], out["dx"], weight=s["weight"], dsum=s["dsum"],
                            dweight=out["dweight"], workspace=ws, stream=stream)
                return out
            return call
        out = {"y": new(m, c, dtype=torch.float8_e4m3fn if e4m3 else t), "rstd": new(m, dtype=torch.float32)}
        if case["residual"]:
            out["sum"] = new(m, c)
        if e4m3:
            out["scales"] = new(m, -(-c // GROUP) if groups else 1, dtype=torch.float32)

        def call():
            op.forward(s["x"], out["y"], weight=s["weight"], residual=s["residual"], sum=out.get("sum"),
                       rstd=out["rstd"], scales=out.get("scales"), stream=stream)
            return out
        return call
    if case["op"] == "dropout":
        op, out = ops.Dropout(m, case["cols"], case["dtype"], case["p"]), new(m, case["cols"])

        def call():
            op.forward(s["x"], out, residual=s["residual"], seed=s["seed"], offset=s["offset"], stream=stream)
            return out
        return call
    two = case["op"] == "gated"
    k, n = case["inputs"], case["hidden"] if two else case["outputs"]
    op = (ops.GatedFF if two else ops.Linear)(m, k, n, case["dtype"], case["act"])
    ws = space(op, case["dir"] == "backward")
    if case["dir"] == "backward":
        out = {"dx": new(m, k), "dw": [new(k, n) for _ in s["w"]], "db": [new(n) for _ in s["w"]] if case["bias"] else []}
        db = out["db"] or [None, None]

        def call():
            if two:
                op.backward(s["dy"], s["x"], s["w"][0], s["w"][1], s["pre"][0], s["pre"][1], dx=out["dx"],
                            dw_gate=out["dw"][0], dw_up=out["dw"][1], db_gate=db[0], db_up=db[1], workspace=ws,
                            stream=stream)
            else:
                op.backward(s["dy"], s["x"], s["w"][0], pre=s["pre"][0] if s["pre"] else None, dx=out["dx"],
                            dw=out["dw"][0], db=db[0], workspace=ws, stream=stream)
            return out
        return call
    out = {"y": new(m, n), "pre": [new(m, n) for _ in s["w"]] if case["dir"] == "train" else []}
    pre = out["pre"] or [None, None]

    def call():
        if two:
            op.forward(s["x"], s["w"][0], s["w"][1], out["y"], b_gate=s["b"][0], b_up=s["b"][1], gate=pre[0],
                       up=pre[1], workspace=ws, stream=stream)
        else:
            op.forward(s["x"], s["w"][0], out["y"], bias=s["b"][0], residual=s["residual"], workspace=ws,
                       stream=stream)
        return out
    return call


# ---------------------------------------------------------------------------
# The plain forms, in 32 bits, rounded once at the end.
# ---------------------------------------------------------------------------
GELU_C, GELU_K = 0.7978845608, 0.044715


def _act(act, x):
    if act == "relu":
        return torch.where(x > 0, x, 0.0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    if act == "tanh":
        return torch.tanh(x)
    if act == "leaky_relu":
        return torch.where(x > 0, x, 0.01 * x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(GELU_C * (x + GELU_K * x * x * x)))
    return x


def _act_slope(act, x):
    if act == "relu":
        return torch.where(x > 0, 1.0, 0.0)
    if act == "sigmoid":
        y = 1 / (1 + torch.exp(-x))
        return y * (1 - y)
    if act == "tanh":
        y = torch.tanh(x)
        return 1 - y * y
    if act == "leaky_relu":
        return torch.where(x > 0, 1.0, 0.01)
    if act == "silu":
        y = 1 / (1 + torch.exp(-x))
        return y * (1 + x * (1 - y))
    if act == "gelu":
        y = torch.tanh(GELU_C * (x + GELU_K * x * x * x))
        return 0.5 * (1 + y) + 0.5 * x * (1 - y * y) * GELU_C * (1 + 3 * GELU_K * x * x)
    return torch.ones_like(x)


def _plain_norm(case, s):
    t, c, w = TYPES[case["dtype"]], case["cols"], s["weight"].float()
    if case["dir"] == "backward":
        dy, x, r = s["dy"].float(), s["sum"].float(), s["rstd"][:, None]
        wdy = dy * w
        dx = r * wdy - x * (r * r * r * ((wdy * x).sum(1, keepdim=True) / c))
        if s["dsum"] is not None:
            dx = dx + s["dsum"].float()
        return {"dx": dx.to(t), "dweight": (dy * (x * r)).sum(0).to(t)}
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    rstd = 1 / torch.sqrt((x * x).sum(1) / c + EPS)
    y = x * rstd[:, None] * w
    out = {"rstd": rstd}
    if s["residual"] is not None:
        out["sum"] = x.to(t)
    if case["out"] == "same":
        out["y"] = y.to(t)
        return out
    m, g = case["rows"], GROUP if case["out"] == "e4m3_groups" else c
    parts = torch.nn.functional.pad(y, (0, -c % g)).view(m, -1, g)
    scales = torch.clamp(parts.abs().amax(2) / E4M3_MAX, min=TINY)
    out["scales"] = scales
    out["y"] = (parts * (1 / scales)[:, :, None]).reshape(m, -1)[:, :c].contiguous().to(torch.float8_e4m3fn)
    return out


def _plain_gated(case, s):
    t, act = TYPES[case["dtype"]], case["act"]
    x, wg, wu = s["x"].float(), s["w"][0].float(), s["w"][1].float()
    if case["dir"] == "backward":
        dh, g, u = s["dy"].float(), s["pre"][0].float(), s["pre"][1].float()
        dg, du = dh * u * _act_slope(act, g), dh * _act(act, g)
        db = [dg.sum(0).to(t), du.sum(0).to(t)] if case["bias"] else []
        return {"dx": (dg @ wg.T + du @ wu.T).to(t), "dw": [(x.T @ dg).to(t), (x.T @ du).to(t)], "db": db}
    g, u = x @ wg, x @ wu
    if case["bias"]:
        g, u = g + s["b"][0].float(), u + s["b"][1].float()
    return {"y": (_act(act, g) * u).to(t), "pre": [g.to(t), u.to(t)] if case["dir"] == "train" else []}


def _plain_linear(case, s):
    t, act = TYPES[case["dtype"]], case["act"]
    x, w = s["x"].float(), s["w"][0].float()
    if case["dir"] == "backward":
        dp = s["dy"].float()
        if act != "identity":
            dp = dp * _act_slope(act, s["pre"][0].float())
        return {"dx": (dp @ w.T).to(t), "dw": [(x.T @ dp).to(t)], "db": [dp.sum(0).to(t)] if case["bias"] else []}
    p = x @ w
    if case["bias"]:
        p = p + s["b"][0].float()
    y = _act(act, p)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(t), "pre": []}


def _shr(z, n):
    """Logical shift right of 64-bit words held as signed ones."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _signed(v):
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def _draws(n, seed, offset):
    """32 random bits for each of n elements: output offset + i/2 of the
    splitmix64 stream of `seed`, its low half for even i and its high half for
    odd i (products wrap at 64 bits)."""
    z = torch.arange((n + 1) // 2, device="cuda", dtype=torch.int64) + _signed(offset + 1)
    z = z * _signed(0x9E3779B97F4A7C15) + _signed(seed)
    z = (z ^ _shr(z, 30)) * _signed(0xBF58476D1CE4E5B9)
    z = (z ^ _shr(z, 27)) * _signed(0x94D049BB133111EB)
    z = z ^ _shr(z, 31)
    return torch.stack([z & 0xFFFFFFFF, _shr(z, 32)], 1).reshape(-1)[:n]


def _plain_dropout(case, s):
    x, p = s["x"].float(), case["p"]
    keep = _draws(x.numel(), s["seed"], s["offset"]).reshape(x.shape) >= int(p * 2.0 ** 32)
    y = torch.where(keep, x * torch.tensor(1 / (1 - p), dtype=torch.float32, device="cuda"), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# The definitions, in 64 bits.
# ---------------------------------------------------------------------------
def _f_and_slope(act, x):
    """f(x) and f'(x) by their definitions."""
    if act in ("relu", "leaky_relu"):
        low = 0.0 if act == "relu" else 0.01
        slope = torch.full_like(x, low).masked_fill_(x > 0, 1.0)
        return x * slope, slope
    if act == "sigmoid":
        f = torch.sigmoid(x)
        return f, f * torch.sigmoid(-x)
    if act == "tanh":
        f = torch.tanh(x)
        return f, torch.cosh(x).pow(-2)
    if act == "silu":
        q = torch.sigmoid(x)
        return x * q, q + x * q * torch.sigmoid(-x)
    if act == "gelu":  # x sigmoid(2 v), v = c (x + k x^3)
        v2 = 2 * GELU_C * (x + GELU_K * x ** 3)
        q = torch.sigmoid(v2)
        return x * q, q + x * q * torch.sigmoid(-v2) * 2 * GELU_C * (1 + 3 * GELU_K * x ** 2)
    return x, torch.ones_like(x)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "norm":
        w, c = s["weight"].double(), case["cols"]
        if case["dir"] == "backward":
            x, r, dy = s["sum"].double(), s["rstd"].double().unsqueeze(1), s["dy"].double()
            hat = x * r
            d = dy * w
            dx = (d - hat * torch.mean(d * hat, dim=1, keepdim=True)) * r
            if s["dsum"] is not None:
                dx += s["dsum"].double()
            return {"dx": dx, "dweight": torch.sum(dy * hat, dim=0)}
        x = s["x"].double()
        if s["residual"] is not None:
            x = x + s["residual"].double()
        rstd = torch.rsqrt(x.square().mean(dim=1) + EPS)
        y = x * rstd.unsqueeze(1) * w
        out = {"rstd": rstd, "y": y}
        if s["residual"] is not None:
            out["sum"] = x
        if case["out"] != "same":
            step = GROUP if case["out"] == "e4m3_groups" else c
            cut = list(y.split(step, dim=1))
            out["scales"] = torch.cat([torch.linalg.vector_norm(p, math.inf, dim=1, keepdim=True) for p in cut], 1) / E4M3_MAX
            out["y"] = torch.cat([p / q for p, q in zip(cut, out["scales"].split(1, dim=1))], 1)
        return out
    if case["op"] == "dropout":
        # keep or not is a matter of whole numbers: the words are drawn on the host
        import numpy as np

        n = s["x"].numel()
        with np.errstate(over="ignore"):
            z = (np.arange((n + 1) // 2, dtype=np.uint64) + np.uint64(s["offset"] + 1)) * np.uint64(0x9E3779B97F4A7C15)
            z += np.uint64(s["seed"])
            for shift, factor in ((30, 0xBF58476D1CE4E5B9), (27, 0x94D049BB133111EB)):
                z = (z ^ (z >> np.uint64(shift))) * np.uint64(factor)
            z ^= z >> np.uint64(31)
        keep = torch.from_numpy(z.astype("<u8").view("<u4")[:n] >= np.uint32(int(case["p"] * 2.0 ** 32))).cuda()
        y = s["x"].double() * keep.view(s["x"].shape) / (1 - case["p"])
        return y if s["residual"] is None else y + s["residual"].double()
    act, x, w = case["act"], s["x"].double(), [v.double() for v in s["w"]]
    if case["dir"] == "backward":
        dy = s["dy"].double()
        if case["op"] == "gated":
            f, slope = _f_and_slope(act, s["pre"][0].double())
            d = [dy * slope * s["pre"][1].double(), dy * f]
        else:
            d = [dy * _f_and_slope(act, s["pre"][0].double())[1] if s["pre"] else dy]
        dx = sum(torch.mm(p, v.t()) for p, v in zip(d, w))
        return {"dx": dx, "dw": [torch.mm(x.t(), p) for p in d], "db": [p.sum(dim=0) for p in d] if case["bias"] else []}
    p = [torch.mm(x, v) if b is None else torch.addmm(b.double(), x, v) for v, b in zip(w, s["b"])]
    y = _f_and_slope(act, p[0])[0]
    if case["op"] == "gated":
        return {"y": y * p[1], "pre": p if case["dir"] == "train" else []}
    return {"y": y if s["residual"] is None else y + s["residual"].double(), "pre": []}
