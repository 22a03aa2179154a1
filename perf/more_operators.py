"""Performance cases of the operators around the feed-forward layers: the loss
of a large output layer, the update of the layers' weights by orthogonalised
momentum, and products in 8-bit floating point.

  loss      z = x W + b; lse = log(sum(exp(z))); loss = lse - z[label], a row
            without a label (label < 0): 0; and the gradients of x, W and b
            from the rows' dloss, z formed anew
  muon      m = beta m + g; u = g + beta m; X = u / (|u| + eps), |u| the root
            of the sum of squares; five times X = a X + (b G + c G^2) X with
            G = X X^T (or X (b G + c G^2), G = X^T X, the smaller one); w = (1 -
            lr decay) w - lr scale X; or X alone, from a given u
  quantize  e4m3 codes of a matrix with a scale for each 128 columns of a row,
            or of W transposed with a scale for each block of 128 x 128
  linear8   y = act(x W + b) + residual of such codes and scales

W is [inputs x outputs], row-major; its codes are [outputs x inputs].  The
sizes are the benchmark's own layer widths and batches (256 to 4096, B = 64 to
4096), their fourfold hidden widths, output layers of some hundred to 131072
classes, round decimal ones, and any others from `draw`.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GROUP = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # the smallest scale: a group of zeros has it
EPS = 1e-7
STEPS, COEFFICIENTS = 5, (3.4445, -4.7750, 2.0315)
LR, BETA, DECAY = 0.02, 0.95, 0.1


def loss(name, direction, dtype, rows, inputs, classes, bias=False):
    return {"name": name, "op": "loss", "dir": direction, "dtype": dtype, "rows": rows, "inputs": inputs,
            "classes": classes, "bias": bias}


def muon(name, call, dtype, batch, rows, cols):
    return {"name": name, "op": "muon", "call": call, "dtype": dtype, "batch": batch, "rows": rows, "cols": cols}


def quantize(name, by, dtype, rows, cols):
    return {"name": name, "op": "quantize", "by": by, "dtype": dtype, "rows": rows, "cols": cols}


def linear8(name, dtype, rows, inputs, outputs, act="identity", bias=False, residual=False, scales="groups"):
    return {"name": name, "op": "linear8", "dtype": dtype, "rows": rows, "inputs": inputs, "outputs": outputs,
            "act": act, "bias": bias, "residual": residual, "scales": scales}


def listed():
    return [
        # one token scored against its successor: the output layer's weights are read once
        loss("loss_token", "forward", "bf16", 1, 4096, 32768),
        # a validation batch over a large vocabulary: bound by the matrix cores
        loss("loss_forward_2048", "forward", "bf16", 2048, 4096, 131072),
        # the gradients of a training batch
        loss("loss_backward_4096", "backward", "bf16", 4096, 4096, 65536),
        # a classifier of 10007 classes with biases, no size a multiple of a tile
        loss("loss_backward_1000", "backward", "f16", 1000, 1000, 10007, bias=True),
        # the update of the headline regression model's second layer, in the framework's first type
        muon("muon_step_f32", "step", "f32", 1, 1024, 1024),
        # sixteen small layers of one shape updated together: short dependent products
        muon("muon_step_16", "step", "bf16", 16, 512, 2000),
        # the fourfold hidden layer's gradient made orthogonal: bound by the matrix cores
        muon("muon_large", "orthogonalize", "bf16", 1, 4096, 16384),
        # a training batch's activations before a product in 8 bits: memory traffic
        quantize("quantize_rows_8192", "rows", "bf16", 8192, 4096),
        # a layer's weights laid out for serving
        quantize("quantize_weights", "blocks", "bf16", 4096, 16384),
        # one token through the layer back onto the residual stream: 8-bit weights are read once
        linear8("linear8_token", "bf16", 1, 16384, 4096, residual=True),
        # a short prompt, no size a multiple of a tile
        linear8("linear8_300", "f16", 300, 1000, 2500, act="gelu", bias=True),
        # a long prompt: bound by the matrix cores
        linear8("linear8_8192", "bf16", 8192, 4096, 16384, act="silu"),
    ]


# The most work of a drawn case, under the largest listed one's (6.6e12 flops in 16 bits, of which a
# ragged or 32-bit product does fewer a second).
MOST_FLOPS, MOST_FLOPS_F32, MOST_BYTES = 2e12, 2e11, 8e8


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
    op = rng.choice(["loss", "loss", "loss", "muon", "muon", "quantize", "linear8", "linear8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "loss":
        c = loss("", rng.choice(["forward", "backward"]), dtype, _rows(rng), _width(rng, 16, 4096),
                 _width(rng, 100, 131072), bias=rng.random() < 0.4)
    elif op == "muon":
        rows, cols = _width(rng, 16, 4096), _width(rng, 16, 16384)
        if rng.random() < 0.5:
            rows, cols = cols, rows
        c = muon("", rng.choice(["step", "orthogonalize"]), dtype, rng.choice([1, 1, 2, _log_int(rng, 1, 24)]), rows, cols)
    elif op == "quantize":
        c = quantize("", rng.choice(["rows", "blocks"]), dtype, _rows(rng), _width(rng, 16, 16384))
        if c["by"] == "blocks":
            c["rows"] = _width(rng, 16, 8192)
    else:
        c = linear8("", dtype, _rows(rng), _width(rng, 16, 16384), _width(rng, 16, 16384),
                    act=rng.choice(["identity", "silu", "gelu", "relu", "tanh"]), bias=rng.random() < 0.4,
                    residual=rng.random() < 0.4, scales=rng.choice(["groups", "groups", "rows"]))
    del c["name"]
    return c


def work(case):
    e, m = 4 if case["dtype"] == "f32" else 2, case["rows"]
    if case["op"] == "loss":
        k, n = case["inputs"], case["classes"]
        b, head = (n if case["bias"] else 0), m * k + k * n
        if case["dir"] == "forward":  # x, W, labels; loss and lse
            return {"bytes": e * (head + b) + 16 * m, "flops": 2 * m * k * n}
        return {"bytes": 2 * e * (head + b) + 16 * m, "flops": 6 * m * k * n}
    if case["op"] == "muon":
        size, c = case["rows"] * case["cols"], case["batch"]
        small, large = sorted((case["rows"], case["cols"]))
        # G and G^2 are symmetric: half of their elements, then the product with X
        flops = STEPS * (small * (small + 1) * large + small * (small + 1) * small + 2 * small * small * large)
        # step: g, m and w read, m and w written; else u and X
        return {"bytes": c * size * (e + 8 + 2 * e if case["call"] == "step" else 2 * e), "flops": c * flops}
    if case["op"] == "quantize":
        n, cols = m * case["cols"], -(-case["cols"] // GROUP)
        scales = m * cols if case["by"] == "rows" else -(-m // GROUP) * cols
        return {"bytes": n * (e + 1) + 4 * scales, "flops": 3 * n}
    k, n = case["inputs"], case["outputs"]
    groups = -(-k // GROUP)
    scales = m * (groups if case["scales"] == "groups" else 1) + -(-n // GROUP) * groups
    out = e * (m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0))
    return {"bytes": m * k + k * n + 4 * scales + out, "flops": 2 * m * k * n}


# ---------------------------------------------------------------------------
# Inputs, from the seed alone (on the GPU, so that making them is quick).
# ---------------------------------------------------------------------------
def _codes(x, by):
    """e4m3 codes of x and their scales: by "groups" of 128 columns of a row,
    whole "rows", or "blocks" of 128 x 128 (codes as they lie)."""
    x = x.float()
    m, c = x.shape
    if by == "blocks":
        parts = torch.nn.functional.pad(x, (0, -c % GROUP, 0, -m % GROUP))
        parts = parts.view(-(-m // GROUP), GROUP, -(-c // GROUP), GROUP)
        scales = torch.clamp(parts.abs().amax((1, 3)) / E4M3_MAX, min=TINY)
        y = (parts * (1 / scales)[:, None, :, None]).reshape(-(-m // GROUP) * GROUP, -1)[:m, :c]
    else:
        g = GROUP if by == "groups" else c
        parts = torch.nn.functional.pad(x, (0, -c % g)).view(m, -1, g)
        scales = torch.clamp(parts.abs().amax(2) / E4M3_MAX, min=TINY)
        y = (parts * (1 / scales)[:, :, None]).reshape(m, -1)[:, :c]
    return y.contiguous().to(torch.float8_e4m3fn), scales.contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)).to(t)

    m, s = case["rows"], {}
    if case["op"] == "loss":
        k, n = case["inputs"], case["classes"]
        s["x"], s["w"] = normal(m, k), normal(k, n, scale=2 * k ** -0.5)
        s["b"] = normal(n, scale=0.5) if case["bias"] else None
        labels = torch.randint(0, n, (m,), generator=g, device="cuda", dtype=torch.int32)
        # one row in ten pads its sequence and has no label
        s["labels"] = torch.where(torch.rand(m, generator=g, device="cuda") < 0.1, -1, labels).to(torch.int32)
        if case["dir"] == "backward":
            # the rows' logits, some at a time, and the mean over the rows with a label
            step = max(1, (1 << 28) // n)
            z = [torch.logsumexp(s["x"][i:i + step].float() @ s["w"].float()
                                 + (0 if s["b"] is None else s["b"].float()), 1) for i in range(0, m, step)]
            s["lse"] = torch.cat(z)
            s["dloss"] = (1.0 + torch.rand(m, generator=g, device="cuda")) / max(1, m)
    elif case["op"] == "muon":
        b, c = case["batch"], case["cols"]
        # a few strong directions and noise
        strong = torch.randn(b, m, 8, generator=g, device="cuda") @ torch.randn(b, 8, c, generator=g, device="cuda")
        s["g"] = (1e-3 * (torch.randn(b, m, c, generator=g, device="cuda") + 0.5 * strong)).to(t)
        if case["call"] == "step":
            s["m"] = 5e-3 * torch.randn(b, m, c, generator=g, device="cuda")
            s["w"] = normal(b, m, c, scale=m ** -0.5)
    elif case["op"] == "quantize":
        c = case["cols"]
        loud = 1 + 19 * (torch.rand(c, generator=g, device="cuda") < 0.005).float()
        s["x"] = (loud * torch.randn(m, c, generator=g, device="cuda")).to(t)
    else:
        k, n = case["inputs"], case["outputs"]
        s["x"], s["sx"] = _codes(torch.randn(m, k, generator=g, device="cuda"), case["scales"])
        s["w"], s["sw"] = _codes(k ** -0.5 * torch.randn(n, k, generator=g, device="cuda"), "blocks")
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
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
    return {"loss": _plain_loss, "muon": _plain_muon, "quantize": _plain_quantize,
            "linear8": _plain_linear8}[state["case"]["op"]](state["case"], state)


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

    def space(n):
        return new(n, dtype=torch.uint8) if n else None

    if case["op"] == "loss":
        k, n = case["inputs"], case["classes"]
        op, back = ops.CrossEntropy(m, k, n, case["dtype"]), case["dir"] == "backward"
        ws = space(op.workspace_bytes(backward=back))
        if back:
            out = {"dx": new(m, k), "dw": new(k, n), "db": new(n) if case["bias"] else None}

            def call():
                op.backward(s["x"], s["w"], s["labels"], s["lse"], s["dloss"], bias=s["b"], dx=out["dx"],
                            dw=out["dw"], db=out["db"], workspace=ws, stream=stream)
                return out
            return call
        out = {"loss": new(m, dtype=torch.float32), "lse": new(m, dtype=torch.float32)}

        def call():
            op.forward(s["x"], s["w"], s["labels"], out["loss"], lse=out["lse"], bias=s["b"], workspace=ws,
                       stream=stream)
            return out
        return call
    if case["op"] == "muon":
        c = case["cols"]
        op = ops.Muon(m, c, case["dtype"], batch=case["batch"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        ws = space(op.workspace_bytes())
        if case["call"] == "orthogonalize":
            out = new(case["batch"], m, c)

            def call():
                op.orthogonalize(s["g"], out, workspace=ws, stream=stream)
                return out
            return call
        out = {"w": new(case["batch"], m, c), "m": new(case["batch"], m, c, dtype=torch.float32)}

        def call():
            # a pass starts from the same weights and momentum: the updated ones go elsewhere
            op.step(s["w"], s["g"], s["m"], LR, beta=BETA, decay=DECAY, scale=_scale(case), w_out=out["w"],
                    momentum_out=out["m"], workspace=ws, stream=stream)
            return out
        return call
    if case["op"] == "quantize":
        c, blocks = case["cols"], case["by"] == "blocks"
        op = ops.Quantize(m, c, case["dtype"], by=case["by"])
        y = new(c, m, dtype=torch.float8_e4m3fn) if blocks else new(m, c, dtype=torch.float8_e4m3fn)
        g = -(-c // GROUP)
        out = {"y": y, "scales": new(g, -(-m // GROUP), dtype=torch.float32) if blocks else new(m, g, dtype=torch.float32)}

        def call():
            op.forward(s["x"], out["y"], out["scales"], stream=stream)
            return out
        return call
    op = ops.Linear8(m, case["inputs"], case["outputs"], case["dtype"], case["act"],
                     group=GROUP if case["scales"] == "groups" else 0)
    ws, y = space(op.workspace_bytes()), new(m, case["outputs"])

    def call():
        op.forward(s["x"], s["sx"], s["w"], s["sw"], y, bias=s["b"], residual=s["residual"], workspace=ws,
                   stream=stream)
        return y
    return call


# ---------------------------------------------------------------------------
# The plain forms, in 32 bits, rounded once at the end.
# ---------------------------------------------------------------------------
GELU_C, GELU_K = 0.7978845608, 0.044715


def _act(act, x):
    if act == "relu":
        return torch.where(x > 0, x, 0.0)
    if act == "tanh":
        return torch.tanh(x)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(GELU_C * (x + GELU_K * x * x * x)))
    return x


def _scale(case):
    """What the orthogonal matrix is multiplied by beside the learning rate: tall layers take larger steps."""
    return max(1.0, case["rows"] / case["cols"]) ** 0.5


def _plain_loss(case, s):
    t, x, w = TYPES[case["dtype"]], s["x"].float(), s["w"].float()
    z = x @ w
    if s["b"] is not None:
        z += s["b"].float()
    label, has = s["labels"].long(), s["labels"] >= 0
    if case["dir"] == "forward":
        top = z.amax(1)
        lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
        at = z[torch.arange(case["rows"], device="cuda"), label.clamp(min=0)]
        return {"loss": torch.where(has, lse - at, 0.0), "lse": lse}
    d = torch.exp(z - s["lse"][:, None])
    d[torch.arange(case["rows"], device="cuda"), label.clamp(min=0)] -= 1
    d *= torch.where(has, s["dloss"], 0.0)[:, None]
    return {"dx": (d @ w.T).to(t), "dw": (x.T @ d).to(t), "db": d.sum(0).to(t) if s["b"] is not None else None}


def _plain_muon(case, s):
    t, u = TYPES[case["dtype"]], s["g"].float()
    if case["call"] == "step":
        m = BETA * s["m"] + u
        u = u + BETA * m
    x = u / (torch.sqrt((u * u).sum((1, 2), keepdim=True)) + EPS)
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    if tall:
        x = x.transpose(1, 2).contiguous()
    if case["call"] == "step":
        return {"w": ((1 - LR * DECAY) * s["w"].float() - LR * _scale(case) * x).to(t), "m": m}
    return x.to(t)


def _plain_quantize(case, s):
    if case["by"] == "rows":
        y, scales = _codes(s["x"], "groups")
        return {"y": y, "scales": scales}
    y, scales = _codes(s["x"].t().contiguous(), "blocks")
    return {"y": y, "scales": scales}


def _plain_linear8(case, s):
    m, k, n = case["rows"], case["inputs"], case["outputs"]
    sx = s["sx"] if case["scales"] == "rows" else s["sx"].repeat_interleave(GROUP, 1)[:, :k]
    sw = s["sw"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    y = (s["x"].float() * sx) @ (s["w"].float() * sw).T
    if s["b"] is not None:
        y = y + s["b"].float()
    y = _act(case["act"], y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# The definitions, in 64 bits.
# ---------------------------------------------------------------------------
def _f(act, x):
    """f(x) by its definition."""
    if act == "relu":
        return x.clamp(min=0)
    if act == "tanh":
        return x.tanh()
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "gelu":  # x sigmoid(2 v), v = c (x + k x^3)
        return x * torch.sigmoid(2 * GELU_C * (x + GELU_K * x ** 3))
    return x


def _exact_loss(case, s):
    """The classes some at a time, so that 64 bits of the largest case fit."""
    x, label, n = s["x"].double(), s["labels"].long().unsqueeze(1), case["classes"]
    parts = range(0, n, 16384)

    def z(i):
        v = torch.mm(x, s["w"][:, i:i + 16384].double())
        return v if s["b"] is None else v + s["b"][i:i + 16384].double()

    lse = torch.stack([torch.logsumexp(z(i), 1) for i in parts]).logsumexp(0)
    if case["dir"] == "forward":
        at = (x * s["w"].t()[label[:, 0].clamp(min=0)].double()).sum(1)
        if s["b"] is not None:
            at = at + s["b"].double()[label[:, 0].clamp(min=0)]
        return {"loss": (lse - at).masked_fill(label[:, 0] < 0, 0.0), "lse": lse}
    g = s["dloss"].double().masked_fill(label[:, 0] < 0, 0.0).unsqueeze(1)
    dx, dw, db = torch.zeros_like(x), [], []
    for i in parts:
        p = torch.softmax(torch.cat([z(i), lse.unsqueeze(1)], 1), 1)
        p = p[:, :-1] / p[:, -1:]  # against lse, which stands for all classes
        hit = label - i
        inside = (hit >= 0) & (hit < p.shape[1])
        p.scatter_add_(1, hit.clamp(0, p.shape[1] - 1), -inside.double())
        p *= g
        dx += torch.mm(p, s["w"][:, i:i + 16384].double().t())
        dw.append(torch.mm(x.t(), p))
        db.append(p.sum(0))
    return {"dx": dx, "dw": torch.cat(dw, 1), "db": torch.cat(db) if s["b"] is not None else None}


def _exact_muon(case, s):
    m, x, w = [], [], []
    for i in range(case["batch"]):
        u = s["g"][i].double()
        if case["call"] == "step":
            m.append(BETA * s["m"][i].double() + u)
            u = u + BETA * m[-1]
        v = u / (torch.linalg.matrix_norm(u) + EPS)
        v = v.t() if case["rows"] > case["cols"] else v
        for _ in range(STEPS):  # X = (a I + b G + c G^2) X
            gram = torch.mm(v, v.t())
            poly = torch.addmm(gram, gram, gram, beta=COEFFICIENTS[1], alpha=COEFFICIENTS[2])
            poly.diagonal().add_(COEFFICIENTS[0])
            v = torch.mm(poly, v)
        x.append(v.t() if case["rows"] > case["cols"] else v)
        if case["call"] == "step":
            w.append(s["w"][i].double() * (1 - LR * DECAY) - x[-1] * (LR * _scale(case)))
    return {"w": torch.stack(w), "m": torch.stack(m)} if case["call"] == "step" else torch.stack(x)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "loss":
        return _exact_loss(case, s)
    if case["op"] == "muon":
        return _exact_muon(case, s)
    if case["op"] == "quantize":
        x = s["x"].double() if case["by"] == "rows" else s["x"].double().t()
        cut = list(x.split(GROUP, dim=1))
        if case["by"] == "rows":
            scales = torch.cat([torch.linalg.vector_norm(p, math.inf, dim=1, keepdim=True) for p in cut], 1) / E4M3_MAX
            each = scales
        else:
            scales = torch.stack([torch.stack([q.abs().max() for q in p.split(GROUP, dim=0)]) for p in cut], 1) / E4M3_MAX
            each = scales.repeat_interleave(GROUP, 0)[:x.shape[0]]
        return {"y": torch.cat([p / q for p, q in zip(cut, each.split(1, dim=1))], 1), "scales": scales}
    # sum over the blocks of k: scale of x, scale of W, and the product of the codes
    x, w, n = s["x"].double(), s["w"].double(), case["outputs"]
    y = torch.zeros(case["rows"], n, device="cuda", dtype=torch.float64)
    for b in range(s["sw"].shape[1]):
        at = slice(b * GROUP, (b + 1) * GROUP)
        sx = s["sx"][:, b if case["scales"] == "groups" else 0].double().unsqueeze(1)
        sw = s["sw"][:, b].double().repeat_interleave(GROUP)[:n]
        y += torch.mm(x[:, at], w[:, at].t()) * sx * sw
    if s["b"] is not None:
        y = y + s["b"].double()
    y = _f(case["act"], y)
    return y if s["residual"] is None else y + s["residual"].double()
