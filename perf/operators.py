"""Timed cases of the 8-bit integer operators: token quantisation, the W8A8
linear product, and the W8A8 product grouped by expert.

`run` computes an operator in plain torch (32-bit arithmetic) or, with `own`
set, through the library's entry points. A case names the operator, its sizes
and its variant; `prepare` makes the inputs from a seed.
"""
import os
import sys

import torch

own = False

_api = None


def _framework():
    """The library's Python binding (imported on the first own pass only)."""
    global _api
    if _api is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grpc-unlimited-ocr_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import uocr_moe
        _api = uocr_moe
    return _api


def _quantize(name, rows, cols, dtype="f32", pad=0):
    return dict(name=name, op="quantize", rows=rows, cols=cols, dtype=dtype, pad=pad)


def _linear(name, m, n, k, out="f32", bias=False, residual=False):
    return dict(name=name, op="linear", m=m, n=n, k=k, out=out, bias=bias, residual=residual)


def _grouped(name, tokens, top_k, experts, n, k, gated, gather, out="bf16", skew=0.0):
    return dict(name=name, op="grouped", tokens=tokens, top_k=top_k, experts=experts, n=n, k=k, gated=gated,
                gather=gather, out=out, skew=skew)


def listed():
    return [
        # The hidden state of one decoded token in front of a projection: latency.
        _quantize("quantize, one token", 1, 2048),
        # The activations of a 4096-token page, columns of a wider bf16 buffer.
        _quantize("quantize, a page", 4096, 2048, "bf16", pad=64),
        # The attention output projection of one decoded token with its residual add: latency.
        _linear("linear, one token", 1, 2048, 2048, residual=True),
        # The vocabulary projection of one decoded token: a stream of weights.
        _linear("linear, one token to the vocabulary", 1, 102400, 2048),
        # A handful of tokens through a matrix of odd sizes.
        _linear("linear, odd sizes", 61, 1031, 1000, "bf16", bias=True),
        # The output projection of a 4096-token page with its residual add.
        _linear("linear, a page", 4096, 2048, 2048, residual=True),
        # Several pages through a wide projection: the arithmetic bound.
        _linear("linear, large", 8192, 8192, 4096, "bf16"),
        # The gate/up products of one decoded token's six experts.
        _grouped("experts gate/up, one token", 1, 6, 64, 1024, 2048, True, True),
        # The down products of a 16-token decode batch: most experts get one or two rows.
        _grouped("experts down, 16 tokens", 16, 6, 64, 2048, 1024, False, False),
        # Ragged groups of odd sizes, some of them empty.
        _grouped("experts, odd and ragged", 77, 2, 16, 203, 529, True, False, "f32", skew=1.5),
        # The down products of a 4096-token page.
        _grouped("experts down, a page", 4096, 6, 64, 2048, 1024, False, False),
        # The gate/up products of eight pages whose experts' popularity is skewed.
        _grouped("experts gate/up, eight pages", 32768, 6, 64, 1024, 2048, True, True, skew=1.2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "grouped", "grouped"])
    out = rng.choice(["f32", "bf16"])
    while True:
        if op == "quantize":
            c = dict(op=op, rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 64, 8192), dtype=out,
                     pad=rng.choice([0, 8, 24, 64, 5]))
            if c["rows"] * c["cols"] <= 1 << 26:
                return c
        elif op == "linear":
            c = dict(op=op, m=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 16384), k=_log_int(rng, 64, 8192), out=out,
                     bias=rng.random() < 0.3, residual=rng.random() < 0.3)
            if c["m"] * c["n"] * c["k"] <= 1 << 37:
                return c
        else:
            experts = _log_int(rng, 4, 128)
            c = dict(op=op, tokens=_log_int(rng, 1, 8192), top_k=rng.randint(1, min(8, experts)), experts=experts,
                     n=_log_int(rng, 64, 2048), k=_log_int(rng, 64, 2048), gated=rng.random() < 0.5,
                     gather=rng.random() < 0.5, out=out, skew=rng.choice([0.0, 0.6, 1.2]))
            if experts * c["n"] * c["k"] <= 1 << 27 and c["tokens"] * c["top_k"] * c["n"] * c["k"] <= 1 << 37:
                return c


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _pitch(k):
    return (k + 15) // 16 * 16


def _activations(gen, rows, cols):
    """N(0, 1) rows of different magnitude with a few larger channels, as hidden states have."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=gen, device="cuda") * 0.5)
    x[:, torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device="cuda")] *= 6.0
    return x


def _int8_rows(x):
    """Rows in int8 with a pitch of 16 bytes, and a scale for each row."""
    rows, cols = x.shape
    scales = x.abs().amax(1).clamp_min(1e-20) / 127.0
    q = torch.zeros(rows, _pitch(cols), dtype=torch.int8, device=x.device)[:, :cols]
    q.copy_(torch.round(x / scales[:, None]).clamp_(-127, 127))
    return q, scales


def _weights(gen, experts, n, k):
    q = torch.zeros(experts, n, _pitch(k), dtype=torch.int8, device="cuda")[:, :, :k]
    scales = torch.empty(experts, n, device="cuda")
    for e in range(experts):
        w, s = _int8_rows(torch.randn(n, k, generator=gen, device="cuda") * 0.02)
        q[e].copy_(w)
        scales[e].copy_(s)
    return q, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(gen, rows, cols + case["pad"]).to(_TYPES[case["dtype"]])[:, :cols]
        s["q"] = torch.zeros(rows, _pitch(cols), dtype=torch.int8, device="cuda")[:, :cols]
        s["scales"] = torch.zeros(rows, device="cuda")
        return s
    out = _TYPES[case["out"]]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"], s["x_scales"] = _int8_rows(_activations(gen, m, k))
        w, ws = _weights(gen, 1, n, k)
        s["w"], s["w_scales"] = w[0], ws[0]
        s["bias"] = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        s["residual"] = torch.randn(m, n, generator=gen, device="cuda").to(out) if case["residual"] else None
        s["y"] = torch.empty(m, n, dtype=out, device="cuda")
        return s
    tokens, top_k, experts, n, k = (case[v] for v in ("tokens", "top_k", "experts", "n", "k"))
    # Router scores with a popularity ~ (e + 1)^-skew; the rows in expert order, token order inside.
    scores = torch.randn(tokens, experts, generator=gen, device="cuda") * 0.7
    scores -= case["skew"] * torch.log(torch.arange(1, experts + 1, device="cuda"))
    ids = scores.topk(top_k, dim=1).indices.reshape(-1)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=experts)
    s["offsets"] = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    s["offsets"][1:] = counts.cumsum(0)
    s["counts"] = counts.tolist()
    rows = tokens * top_k
    s["row_index"] = (order // top_k).to(torch.int32) if case["gather"] else None
    s["x"], s["x_scales"] = _int8_rows(_activations(gen, tokens if case["gather"] else rows, k))
    s["w"], s["w_scales"] = _weights(gen, experts, n, k)
    s["w_up"], s["w_up_scales"] = _weights(gen, experts, n, k) if case["gated"] else (None, None)
    s["y"] = torch.empty(rows, n, dtype=out, device="cuda")
    return s


def _plain_quantize(s):
    x = s["x"].float()
    peak = x.abs().amax(1, keepdim=True)
    scales = torch.where(peak > 0, peak / 127.0, torch.ones_like(peak))
    return torch.round(x / scales).clamp(-127, 127) * scales, scales[:, 0]


def _plain_linear(s):
    y = (s["x"].float() @ s["w"].float().T) * s["x_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["y"].dtype)


def _plain_grouped(s):
    x, scales = s["x"].float(), s["x_scales"][:, None]
    if s["row_index"] is not None:
        x, scales = x[s["row_index"]], scales[s["row_index"]]
    rows, experts = x.shape[0], s["experts"]

    def product(w, w_scales):
        if rows <= experts:  # few rows: each with its own expert's matrix
            of = torch.searchsorted(s["offsets"], torch.arange(rows, device=x.device), right=True) - 1
            return torch.bmm(w[of].float(), x[:, :, None])[:, :, 0] * scales * w_scales[of]
        # Many rows: one product for each expert that has some.
        parts = zip(x.split(s["counts"]), w, w_scales)
        return torch.cat([(xe @ we.float().T) * se for xe, we, se in parts if xe.shape[0] > 0]) * scales

    y = product(s["w"], s["w_scales"])
    if s["w_up"] is not None:
        y = y / (1.0 + torch.exp(-y)) * product(s["w_up"], s["w_up_scales"])
    return y.to(s["y"].dtype)


def run(state):
    s = state
    if not own:
        return {"quantize": _plain_quantize, "linear": _plain_linear, "grouped": _plain_grouped}[s["op"]](s)
    api = _framework()
    if s["op"] == "quantize":
        api.quantize_tokens(s["x"], s["q"], s["scales"])
        return torch.mul(s["q"], s["scales"][:, None]), s["scales"]
    if s["op"] == "linear":
        api.linear_w8a8(s["x"], s["x_scales"], s["w"], s["w_scales"], s["y"], bias=s["bias"], residual=s["residual"])
    else:
        api.grouped_linear_w8a8(s["x"], s["x_scales"], s["w"], s["w_scales"], s["offsets"], s["y"],
                                row_index=s["row_index"], w_up=s["w_up"], w_up_scales=s["w_up_scales"])
    return s["y"]


def work(case):
    """Bytes: inputs once, outputs once (of the experts, only those that have rows, at their expected number).
    Operations: two for each multiply-add."""
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 4 * n + 4 * case["rows"], "flops": 3 * n}
    eb = 2 if case["out"] == "bf16" else 4
    n, k = case["n"], case["k"]
    if case["op"] == "linear":
        m = case["m"]
        io = m * k + n * k + 4 * (m + n) + m * n * eb * (2 if case["residual"] else 1)
        return {"bytes": io, "flops": 2 * m * n * k}
    rows, experts = case["tokens"] * case["top_k"], case["experts"]
    stacks = 2 if case["gated"] else 1
    used = min(rows, round(experts * (1.0 - (1.0 - case["top_k"] / experts) ** case["tokens"])))
    x_rows = case["tokens"] if case["gather"] else rows
    return {"bytes": x_rows * k + used * stacks * n * (k + 4) + rows * n * eb + 8 * rows + 4 * experts,
            "flops": 2 * rows * n * k * stacks}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double()
        step = x.abs().max(dim=1).values / 127.0
        step[step == 0] = 1.0
        q = torch.round(x / step[:, None]).clamp(min=-127, max=127)
        return q * step[:, None], step
    if case["op"] == "linear":
        y = s["w"].double() * s["w_scales"].double()[:, None]
        y = torch.mm(s["x"].double() * s["x_scales"].double()[:, None], y.t())
        y = y if s["bias"] is None else y + s["bias"].double()
        return y if s["residual"] is None else y + s["residual"].double()
    y = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e in range(case["experts"]):
        at = torch.arange(ends[e], ends[e + 1], device="cuda")
        rows = at if s["row_index"] is None else s["row_index"][at].long()
        x = s["x"][rows].double() * s["x_scales"][rows].double()[:, None]
        g = x @ (s["w"][e].double() * s["w_scales"][e].double()[:, None]).T
        if case["gated"]:
            g = g * torch.sigmoid(g) * (x @ (s["w_up"][e].double() * s["w_up_scales"][e].double()[:, None]).T)
        y[at] = g
    return y
