"""Measured cases of the serving and epilogue operators.

Three operators:

  whole / experts   the SwiGLU mixture-of-experts layer for a few tokens
                    (``moe_few_tokens``: router, top-k, experts, combine; ``moe_few_experts``:
                    the same with routing weights and indices already known)
  linear            act(x . W^T + bias) + residual, forward or forward and backward
  grouped           the same per expert over grouped rows, [E, N, K] weights and [E, N] biases

``run`` computes a case either in its plain form (elementary torch operations in fp32) or, when
``own`` is set, through the package's public entry points.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # The small layer of the test configuration (d = 512, 8 experts, fp32), one token:
        # latency counts.
        _moe("whole-1tok-small-fp32", "whole", "fp32", 1, 512, 8, 2, 1024, False),
        # Decoding one sequence with the benchmark layer (d = 4096, 64 experts, H = 11008).
        _moe("whole-1tok-bf16", "whole", "bf16", 1, 4096, 64, 2, 11008, False),
        # Decoding a batch of 16 sequences with the same layer, per-expert router bias.
        _moe("whole-16tok-bf16", "whole", "bf16", 16, 4096, 64, 2, 11008, True),
        # The fine-grained layer (d = 7168, 256 experts, top-8, H = 2048), a batch of 32, the
        # routing computed elsewhere: the largest weights and the most slots.
        _moe("experts-32tok-fine-bf16", "experts", "bf16", 32, 7168, 256, 8, 2048, False),
        # Odd sizes: 11 tokens, top-3 of 20 experts, tiles that end inside both weights.
        _moe("experts-11tok-odd-fp16", "experts", "fp16", 11, 1000, 20, 3, 1416, False),
        # A shared expert's first projection for one token: bias and activation.
        _lin("linear-1tok-bf16", "linear", "bf16", 1, 4096, 11008, "gelu_tanh", True, False, False),
        # The second projection of a small batch, added to the routed experts' output.
        _lin("linear-37tok-fp16", "linear", "fp16", 37, 7168, 4096, "none", True, True, False),
        # A prompt of 8192 tokens through a wide projection: the largest product.
        _lin("linear-8192tok-bf16", "linear", "bf16", 8192, 4096, 11008, "gelu", True, True, False),
        # A training step of a projection with every input's gradient, ragged row count.
        _lin("linear-train-4099tok-bf16", "linear", "bf16", 4099, 2048, 7168, "silu", True, True, True),
        # A small fp32 training step with sizes that are no multiple of anything.
        _lin("linear-train-333tok-fp32", "linear", "fp32", 333, 257, 130, "gelu", True, True, True),
        # Per-expert biases over ragged expert rows, training: 16 experts, some empty.
        _grp("grouped-train-8192row-bf16", "bf16", 8192, 16, 4096, 2048, "relu", True, False, True),
        # The rows of a few tokens over 64 experts: weights are nearly all of the bytes.
        _grp("grouped-96row-bf16", "bf16", 96, 64, 2048, 4096, "silu", True, False, False),
    ]


def _moe(name, op, dtype, tokens, d, experts, top_k, hidden, bias):
    c = {"op": op, "dtype": dtype, "tokens": tokens, "d": d, "experts": experts, "top_k": top_k,
         "hidden": hidden, "bias": bias}
    return {"name": name, **c} if name else c


def _lin(name, op, dtype, rows, k, n, act, bias, residual, train, experts=0):
    c = {"op": op, "dtype": dtype, "rows": rows, "k": k, "n": n, "act": act, "bias": bias,
         "residual": residual, "train": train, "experts": experts}
    return {"name": name, **c} if name else c


def _grp(name, dtype, rows, experts, k, n, act, bias, residual, train):
    return _lin(name, "grouped", dtype, rows, k, n, act, bias, residual, train, experts)


def _log(rng, lo, hi):
    """A whole number, spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, aligned):
    v = _log(rng, lo, hi)
    return max(8, v // 8 * 8) if aligned else v


def draw(rng):
    op = rng.choice(["whole", "experts", "linear", "linear", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    small = dtype == "fp32"  # fp32: the sizes of the test configuration and around it
    if op in ("whole", "experts"):
        while True:
            # 16-bit rows that are no multiple of 16 bytes only at small sizes
            odd = small or rng.random() < 0.15
            top = 1024 if odd else None
            e = _log(rng, 2, 64 if odd else 256)
            c = _moe(None, op, dtype, _log(rng, 1, 64), _size(rng, 128, top or 7168, not odd), e,
                     rng.randint(1, min(e, 8)), _size(rng, 128, top or 11008, not odd),
                     op == "whole" and rng.random() < 0.5)
            weights = 3 * c["experts"] * c["d"] * c["hidden"]
            if weights <= 8.6e9 and c["tokens"] * c["top_k"] * c["d"] * c["hidden"] <= 256 * 2048 * 7168:
                return c
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    bias, residual, train = rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.5
    while True:
        odd = small or rng.random() < 0.15
        top = 1024 if small else 2048 if odd else 11008
        rows = _log(rng, 1, 1024 if small else 8192)
        k, n = _size(rng, 64, top, not odd), _size(rng, 64, top, not odd)
        e = _log(rng, 2, 64) if op == "grouped" else 0
        if max(1, e) * n * k <= 6e8 and 2.0 * rows * n * k * (3 if train else 1) <= 7e11:
            return _lin(None, op, dtype, rows, k, n, act, bias, residual, train, e)


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1) + 17)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.empty(*shape, device="cuda", dtype=dt).normal_(0.0, std, generator=g)

    s = {"case": case}
    if case["op"] in ("whole", "experts"):
        t, d, e, h = case["tokens"], case["d"], case["experts"], case["hidden"]
        s["x"] = normal(t, d)
        s["w_gate"] = normal(e, h, d, std=0.02)
        s["w_up"] = normal(e, h, d, std=0.02)
        s["w_down"] = normal(e, d, h, std=0.02)
        if case["op"] == "whole":
            s["w_router"] = normal(e, d, std=0.02)
            s["router_bias"] = None
            if case["bias"]:
                s["router_bias"] = torch.randn(e, device="cuda", generator=g) * 0.1
        else:
            score = torch.randn(t, e, device="cuda", generator=g)
            top = torch.sort(score, dim=1, descending=True, stable=True)
            k = case["top_k"]
            s["indices"] = top.indices[:, :k].to(torch.int32).contiguous()
            s["weights"] = torch.softmax(top.values[:, :k], dim=1).contiguous()
        return s
    m, k, n, e = case["rows"], case["k"], case["n"], case["experts"]
    lead = (e,) if e else ()
    s["x"] = normal(m, k)
    s["w"] = normal(*lead, n, k, std=0.02)
    s["b"] = normal(*lead, n, std=0.5) if case["bias"] else None
    s["r"] = normal(m, n) if case["residual"] else None
    if case["train"]:
        s["dy"] = normal(m, n)
    if e:
        s["offsets"], s["most"] = _ragged(m, e, seed)
    return s


def _ragged(rows, experts, seed):
    """Row offsets of experts with uneven loads (about one in eight empty)."""
    g = torch.Generator().manual_seed(7919 * (seed + 1) + rows)
    load = torch.rand(experts, generator=g, dtype=torch.float64) + 0.25
    load[torch.rand(experts, generator=g) < 0.125] = 0.0
    if float(load.sum()) == 0.0:
        load[0] = 1.0
    ends = torch.round(torch.cumsum(load, 0) / load.sum() * rows).to(torch.int64)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), ends])
    most = int((offsets[1:] - offsets[:-1]).max())
    return offsets.to(torch.int32).cuda(), most


# --------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if op in ("whole", "experts"):
        return _own_moe(state) if own else _plain_moe(state)
    return _own_linear(state) if own else _plain_linear(state)


def _own_moe(s):
    import moe_ops_b200 as M

    c = s["case"]
    if c["op"] == "whole":
        return M.moe_few_tokens(s["x"], s["w_router"], s["w_gate"], s["w_up"], s["w_down"],
                                c["top_k"], router_bias=s["router_bias"])
    return M.moe_few_experts(s["x"], s["weights"], s["indices"], s["w_gate"], s["w_up"], s["w_down"])


def _own_linear(s):
    import moe_ops_b200 as M

    c = s["case"]

    def call(x, w, b, r):
        if c["experts"]:
            return M.grouped_linear(x, w, s["offsets"], bias=b, activation=c["act"], residual=r)
        return M.linear(x, w, bias=b, activation=c["act"], residual=r)

    if not c["train"]:
        return call(s["x"], s["w"], s["b"], s["r"])
    given = [s["x"], s["w"], s["b"], s["r"]]
    leaf = [v if v is None else v.detach().requires_grad_(True) for v in given]
    y = call(*leaf)
    grads = torch.autograd.grad(y, [v for v in leaf if v is not None], s["dy"])
    return [y.detach(), *grads]


def _plain_moe(s):
    c, x = s["case"], s["x"]
    if c["op"] == "whole":
        # which experts are picked is a comparison: the logits are formed in 64 bits
        logits = x.double() @ s["w_router"].double().t()
        if s["router_bias"] is not None:
            logits = logits + s["router_bias"].double()
        top = torch.sort(logits, dim=1, descending=True, stable=True)
        idx = top.indices[:, :c["top_k"]]
        p = top.values[:, :c["top_k"]]
        p = torch.exp(p - p[:, :1])
        p = (p / p.sum(dim=1, keepdim=True)).float()
    else:
        idx, p = s["indices"].long(), s["weights"].float()
    xf = x.float()
    gate = torch.matmul(s["w_gate"][idx].float(), xf[:, None, :, None])
    up = torch.matmul(s["w_up"][idx].float(), xf[:, None, :, None])
    h = gate / (1.0 + torch.exp(-gate)) * up
    del gate, up
    out = torch.matmul(s["w_down"][idx].float(), h)[..., 0]
    return (out * p[:, :, None]).sum(dim=1).to(x.dtype)


def _act(z, act):
    """The activation and its derivative."""
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        return z * sg, sg * (1.0 + z * (1.0 - sg))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 0.7071067811865476))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if act == "gelu_tanh":
        a = 0.7978845608028654
        th = torch.tanh(a * (z + 0.044715 * z * z * z))
        return (0.5 * z * (1.0 + th),
                0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * a * (1.0 + 0.134145 * z * z))
    return z, torch.ones_like(z)


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    b = None if s["b"] is None else s["b"].float()
    r = None if s["r"] is None else s["r"].float()
    e, m = c["experts"], c["rows"]
    if e:
        # rows laid out per expert, padded to the largest expert's
        row = torch.arange(m, device=x.device)
        g = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
        at = row - s["offsets"].long()[g]
        pad = x.new_zeros(e, s["most"], c["k"])
        pad[g, at] = x
        z = torch.bmm(pad, w.transpose(1, 2))[g, at]
        z = z if b is None else z + b[g]
    else:
        z = x @ w.t()
        z = z if b is None else z + b
    y, slope = _act(z, c["act"])
    y = (y if r is None else y + r).to(dt)
    if not c["train"]:
        return y
    dz = s["dy"].float() * slope
    if e:
        dpad = dz.new_zeros(e, s["most"], c["n"])
        dpad[g, at] = dz
        dx = torch.bmm(dpad, w)[g, at]
        dw = torch.bmm(dpad.transpose(1, 2), pad)
        db = dpad.sum(dim=1)
    else:
        dx, dw, db = dz @ w, dz.t() @ x, dz.sum(dim=0)
    grads = [dx.to(dt), dw.to(dt)]
    if b is not None:
        grads.append(db.to(dt))
    if r is not None:
        grads.append(s["dy"])
    return [y, *grads]


# --------------------------------------------------------------------- floor and truth
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("whole", "experts"):
        t, d, e, k, h = (case[x] for x in ("tokens", "d", "experts", "top_k", "hidden"))
        # experts that t tokens with k random picks each are expected to touch
        touched = e * (1.0 - (1.0 - k / e) ** t)
        bytes_ = touched * 3 * d * h * es + 2 * t * d * es
        flops = 6.0 * t * k * d * h
        if case["op"] == "whole":
            bytes_ += e * d * es
            flops += 2.0 * t * e * d
        else:
            bytes_ += t * k * 8
        return {"bytes": bytes_, "flops": flops}
    m, k, n, e = case["rows"], case["k"], case["n"], case["experts"]
    # grouped: about an eighth of the experts are empty, and no more than one per row is read
    live = min(max(1.0, 0.875 * e), m) if e else 1.0
    bytes_ = (m * k + live * n * k + m * n) * es
    bytes_ += (live * n * es if case["bias"] else 0) + (m * n * es if case["residual"] else 0)
    flops = 2.0 * m * k * n
    if case["train"]:
        # dy read; dx, dw, db written
        bytes_ += (m * n + m * k + max(1, e) * n * k) * es + (max(1, e) * n * es if case["bias"] else 0)
        flops *= 3
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("whole", "experts"):
        return _exact_moe(case, s)
    return _exact_linear(case, s)


def _exact_moe(case, s):
    """Expert by expert: every token that picked it, in 64 bits."""
    x = s["x"].double()
    if case["op"] == "whole":
        logits = torch.einsum("td,ed->te", x, s["w_router"].double())
        if s["router_bias"] is not None:
            logits += s["router_bias"].double()[None]
        left = logits.clone()
        picks = []
        for _ in range(case["top_k"]):
            best = left.max(dim=1, keepdim=True).values
            first = (left == best).to(torch.int8).argmax(dim=1)
            picks.append(first)
            left[torch.arange(left.shape[0], device=left.device), first] = -math.inf
        idx = torch.stack(picks, dim=1)
        p = torch.softmax(torch.gather(logits, 1, idx), dim=1)
    else:
        idx, p = s["indices"].long(), s["weights"].double()
    y = torch.zeros_like(x)
    for e in sorted(set(idx.flatten().tolist())):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        g = x[t] @ s["w_gate"][e].double().t()
        u = x[t] @ s["w_up"][e].double().t()
        o = (g * torch.sigmoid(g) * u) @ s["w_down"][e].double().t()
        y.index_add_(0, t, o * p[t, k][:, None])
    return y


def _exact_linear(case, s):
    """Forward and gradients by automatic differentiation of the definition in 64 bits."""
    leaf = [v if v is None else v.double().requires_grad_(case["train"])
            for v in (s["x"], s["w"], s["b"], s["r"])]
    x, w, b, r = leaf
    name = case["act"]
    f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[name]
    if case["experts"]:
        ends = s["offsets"].tolist()
        parts = []
        for e in range(case["experts"]):
            z = x[ends[e]:ends[e + 1]] @ w[e].t()
            parts.append(f(z if b is None else z + b[e]))
        y = torch.cat(parts)
    else:
        z = x @ w.t()
        y = f(z if b is None else z + b)
    y = y if r is None else y + r
    if not case["train"]:
        return y
    grads = torch.autograd.grad(y, [v for v in leaf if v is not None], s["dy"].double())
    return [y.detach(), *grads]
