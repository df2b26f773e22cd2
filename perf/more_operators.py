"""Timed cases of the beam operators: the head rotation with its cache append,
the attention of sequences that share a prefix, the selection over beams and
vocabulary, and the reordering of their states.

`run` computes an operator in plain torch (32-bit arithmetic, 64 where a
comparison or an angle needs it) or, with `own` set, through the library's
entry points. A case names the operator, its sizes and its variant; `prepare`
makes the inputs from a seed.
"""
import math
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


def _rotate(name, rows, heads, kv_heads, dim, rotary, capacity, dtype="f32", norm=False, interleaved=False, far=0,
            caches=1):
    return dict(name=name, op="rotate", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                capacity=capacity, dtype=dtype, norm=norm, interleaved=interleaved, far=far, caches=caches)


def _attention(name, prefixes, prefix, sequences, heads, kv_heads, dim, own_keys, rows_each=1, ancestry=False):
    return dict(name=name, op="attention", prefixes=prefixes, prefix=prefix, sequences=sequences, heads=heads,
                kv_heads=kv_heads, dim=dim, own_keys=own_keys, rows_each=rows_each, ancestry=ancestry)


def _select(name, batch, beams, select, vocab, dtype="f32", finished=False):
    return dict(name=name, op="select", batch=batch, beams=beams, select=select, vocab=vocab, dtype=dtype,
                finished=finished)


def _reorder(name, layers, groups, beams, segments, units, width):
    return dict(name=name, op="reorder", layers=layers, groups=groups, beams=beams, segments=segments, units=units,
                width=width)


def listed():
    return [
        # The queries and keys of four beams' new tokens behind a page, appended to the beams' caches: latency.
        _rotate("rotate, four beams", 4, 16, 4, 128, 128, 1024, caches=4),
        # A page's rows into the prefix cache, heads normalised, half of each head rotated, far positions.
        _rotate("rotate, a page with norms", 4096, 10, 10, 128, 64, 4096, "bf16", norm=True, interleaved=True,
                far=1000000),
        # Eight pages of fp32 projections into their caches.
        _rotate("rotate, eight pages", 32768, 16, 4, 128, 128, 4096, norm=True, caches=8),
        # One step of four beams over a page: latency and one read of the page's keys.
        _attention("attention, four beams on a page", 1, 4096, 4, 16, 4, 128, 300, ancestry=True),
        # One step of eight beams on each of sixteen pages: a stream of keys.
        _attention("attention, sixteen pages of eight beams", 16, 4096, 128, 16, 4, 128, 512, ancestry=True),
        # Instructions of different lengths on one page, heads of 64, odd sizes.
        _attention("attention, odd and ragged", 1, 1001, 7, 9, 3, 64, 61, rows_each=37),
        # Instructions of different lengths on one page: the arithmetic bound.
        _attention("attention, prompts on a page", 1, 4096, 24, 16, 4, 128, 160, rows_each=160),
        # Many sequences behind one long document, a token each.
        _attention("attention, many on a document", 1, 32768, 128, 16, 4, 128, 256),
        # The next tokens of four beams on one page: latency.
        _select("select, four beams", 1, 4, 4, 102400),
        # Sixteen pages of eight beams, some of them finished, with room to set finished ones aside.
        _select("select, sixteen pages", 16, 8, 16, 102400, finished=True),
        # The beams' token histories on a page: latency.
        _reorder("reorder, histories", 1, 1, 4, 1, 1024, 4),
        # The keys of eight beams' own tokens in every layer.
        _reorder("reorder, caches", 24, 4, 8, 4, 512, 256),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["rotate", "attention", "attention", "select", "reorder"])
    while True:
        if op == "rotate":
            caches = _log_int(rng, 1, 32)
            each = _log_int(rng, 1, 8192)
            kv = rng.randint(1, 8)
            dim = rng.choice([64, 80, 96, 128, 192])
            c = _rotate("", caches * each, kv * rng.randint(1, 4), kv, dim, rng.choice([dim, dim // 2, 32]),
                        each + rng.randint(0, 64), rng.choice(["f32", "bf16"]), rng.random() < 0.5,
                        rng.random() < 0.5, rng.choice([0, 5000, 1000000]), caches)
            if c["rows"] * (c["heads"] + 2 * kv) * dim <= 32768 * 24 * 128:
                break
        elif op == "attention":
            prefixes = _log_int(rng, 1, 16)
            kv = rng.randint(1, 8)
            rows_each = rng.choice([1, 1, _log_int(rng, 2, 200)])
            own_keys = _log_int(rng, max(rows_each, 4), 1024)
            c = _attention("", prefixes, _log_int(rng, 1, 32768), prefixes * _log_int(rng, 1, 64),
                           kv * rng.randint(1, 6), kv, rng.choice([64, 128, 128]), own_keys, rows_each,
                           rows_each == 1 and rng.random() < 0.5)
            cost = work(c)
            scores = c["sequences"] * c["rows_each"] * c["heads"] * (c["prefix"] + own_keys)
            if cost["flops"] <= 8e10 and cost["bytes"] <= 4e8 and scores <= 1 << 28:
                break
        elif op == "select":
            c = _select("", _log_int(rng, 1, 32), rng.randint(1, 16), rng.randint(1, 32), _log_int(rng, 100, 200000),
                        rng.choice(["f32", "bf16"]), rng.random() < 0.5)
            if c["batch"] * c["beams"] * c["vocab"] <= 128 * 102400 and c["select"] <= c["vocab"]:
                break
        else:
            c = _reorder("", _log_int(rng, 1, 32), _log_int(rng, 1, 16), rng.randint(2, 32), rng.randint(1, 8),
                         _log_int(rng, 1, 1024), rng.choice([4, 36, 128, 256]))
            if c["layers"] * c["groups"] * c["beams"] * c["segments"] * c["units"] * c["width"] <= 1 << 28:
                break
    del c["name"]
    return c


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_THETA = 1e4


def _activations(gen, *shape):
    """N(0, 1) with a few larger channels, as projections have."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    x[..., torch.randint(0, shape[-1], (max(1, shape[-1] // 64),), generator=gen, device="cuda")] *= 4.0
    return x


def _own_lens(case):
    """Own keys of each sequence, and its query rows: spread over the upper three quarters of the range."""
    n, longest, rows = case["sequences"], case["own_keys"], case["rows_each"]
    lens = [max(1, longest - (37 * i) % max(1, 3 * longest // 4)) for i in range(n)]
    rows = [max(1, rows - (53 * i) % max(1, 3 * rows // 4)) for i in range(n)]
    return [max(a, b) for a, b in zip(lens, rows)], rows


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    bf16 = torch.bfloat16
    if case["op"] == "rotate":
        rows, heads, kv, dim = (case[v] for v in ("rows", "heads", "kv_heads", "dim"))
        dt = _TYPES[case["dtype"]]
        s["q"] = _activations(gen, rows, heads, dim).to(dt)
        both = _activations(gen, rows, 2 * kv, dim).to(dt)  # k and v as one projection leaves them
        s["k"], s["v"] = both[:, :kv], both[:, kv:]
        each = rows // case["caches"]
        s["cache_rows"] = (torch.arange(rows, device="cuda") // each).to(torch.int32)
        first = int(torch.randint(0, case["capacity"] - each + 1, (1,), generator=gen, device="cuda"))
        s["slots"] = (torch.arange(rows, device="cuda") % each + first).to(torch.int32)
        s["positions"] = s["slots"] + case["far"]
        s["inv_freq"] = (1.0 / _THETA ** (torch.arange(case["rotary"] // 2, dtype=torch.float64) * 2
                                          / case["rotary"])).float().cuda()
        s["q_norm"] = torch.rand(dim, generator=gen, device="cuda") + 0.5 if case["norm"] else None
        s["k_norm"] = torch.rand(dim, generator=gen, device="cuda") + 0.5 if case["norm"] else None
        s["q_out"] = torch.empty(rows, heads, dim, dtype=bf16, device="cuda")
        s["k_cache"] = torch.zeros(case["caches"], kv, case["capacity"], dim, dtype=bf16, device="cuda")
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        return s
    if case["op"] == "attention":
        prefixes, n, heads, kv, dim = (case[v] for v in ("prefixes", "sequences", "heads", "kv_heads", "dim"))
        lens, rows = _own_lens(case)
        order = torch.randperm(n, generator=gen, device="cuda").tolist()
        lens, rows = [lens[i] for i in order], [rows[i] for i in order]
        s["lens_list"], s["rows_list"] = lens, rows
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["row_offsets"] = None
        if case["rows_each"] > 1:
            s["row_offsets"] = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
            s["row_offsets"][1:] = torch.tensor(rows, device="cuda").cumsum(0)
        s["prefix_lens"] = torch.full((prefixes,), case["prefix"], dtype=torch.int32, device="cuda")
        shape, cap = (prefixes, kv, case["prefix"], dim), case["own_keys"]
        s["prefix_k"] = _activations(gen, *shape).to(bf16)
        s["prefix_v"] = torch.randn(*shape, generator=gen, device="cuda").to(bf16)
        s["k"] = _activations(gen, n, kv, cap, dim).to(bf16)
        s["v"] = torch.randn(n, kv, cap, dim, generator=gen, device="cuda").to(bf16)
        s["q"] = torch.randn(sum(rows), heads, dim, generator=gen, device="cuda").to(bf16)
        s["ancestry"] = None
        if case["ancestry"]:  # each key with one of the beams of the same page, in runs as a search leaves them
            beams = n // prefixes
            runs = torch.randint(0, beams, (n, cap // 16 + 1), generator=gen, device="cuda").repeat_interleave(16, 1)
            base = torch.arange(n, device="cuda") // beams * beams
            s["ancestry"] = (runs[:, :cap] + base[:, None]).to(torch.int32).contiguous()
        s["out"] = torch.empty(sum(rows), heads, dim, dtype=bf16, device="cuda")
        s["lse"] = torch.empty(sum(rows), heads, device="cuda")
        return s
    if case["op"] == "select":
        batch, beams, select = case["batch"], case["beams"], case["select"]
        logits = torch.randn(batch * beams, case["vocab"], generator=gen, device="cuda") * 2.5
        s["logits"] = logits.to(_TYPES[case["dtype"]])
        s["scores"] = -torch.rand(batch, beams, generator=gen, device="cuda") * 20.0
        s["finished"], s["eos"] = None, -1
        if case["finished"]:
            s["finished"] = (torch.rand(batch, beams, generator=gen, device="cuda") < 0.25).to(torch.int32)
            s["finished"][:, 0] = 0  # a search in which every beam of a page has ended is over
            s["eos"] = 1
        s["tokens"] = torch.empty(batch, select, dtype=torch.int32, device="cuda")
        s["parents"] = torch.empty_like(s["tokens"])
        s["new_finished"] = torch.empty_like(s["tokens"])
        s["new_scores"] = torch.empty(batch, select, device="cuda")
        return s
    layers, groups, beams = case["layers"], case["groups"], case["beams"]
    rows, units = groups * beams, case["units"]
    s["state"] = torch.randint(-30000, 30000, (layers, rows, case["segments"], units, case["width"] // 2),
                               generator=gen, device="cuda", dtype=torch.int16)
    # The first half of each page's beams (in a random order) survive in place; the others become copies of them.
    kept = max(1, beams // 2)
    parents = torch.empty(groups, beams, dtype=torch.int32, device="cuda")
    for g in range(groups):
        order = torch.randperm(beams, generator=gen, device="cuda")
        parents[g, order[:kept]] = order[:kept].to(torch.int32)
        pick = torch.arange(beams - kept, device="cuda") % kept
        parents[g, order[kept:]] = order[:kept][pick].to(torch.int32)
    s["parents"] = parents.reshape(rows)
    s["counts"] = torch.full((rows,), units - units // 8, dtype=torch.int32, device="cuda")
    return s


def _plain_rotate(s):
    rot, dim = s["rotary"], s["dim"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()  # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotated(x, gain):
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain
        y = x.clone()
        if s["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
        return y.to(torch.bfloat16)

    rows, slots = s["cache_rows"].long(), s["slots"].long()
    s["k_cache"][rows, :, slots] = rotated(s["k"], s["k_norm"])
    s["v_cache"][rows, :, slots] = s["v"].to(torch.bfloat16)
    return rotated(s["q"], s["q_norm"]), s["k_cache"], s["v_cache"]


def _own_cache(s, cache):
    """[sequences, kv_heads, capacity, dim]: each sequence's own keys or values, gathered where beams share them."""
    if s["ancestry"] is None:
        return cache
    at = torch.arange(cache.shape[2], device="cuda")
    return cache[s["ancestry"].long(), :, at[None, :]].transpose(1, 2)


def _plain_attention(s):
    heads, kv, dim, n = s["heads"], s["kv_heads"], s["dim"], s["sequences"]
    group, scale, per = heads // kv, s["dim"] ** -0.5, s["sequences"] // s["prefixes"]
    keys, values = _own_cache(s, s["k"]).float(), _own_cache(s, s["v"]).float()
    q = s["q"].float().view(-1, kv, group, dim).transpose(0, 1)  # [kv, rows, group, dim]
    out = torch.empty(q.shape, device="cuda")
    lse = torch.empty(q.shape[:3], device="cuda")
    at = torch.arange(keys.shape[2], device="cuda")
    one = s["row_offsets"] is None
    starts = list(range(n + 1)) if one else [0] + torch.tensor(s["rows_list"]).cumsum(0).tolist()
    for p in range(s["prefixes"]):
        lo, hi, of = starts[p * per], starts[(p + 1) * per], slice(p * per, (p + 1) * per)
        # The prefix once for all of its rows.
        sp = torch.matmul(q[:, lo:hi].reshape(kv, -1, dim), s["prefix_k"][p].float().transpose(1, 2)) * scale
        sp = sp.view(kv, hi - lo, group, -1)
        if one:
            so = torch.matmul(q[:, lo:hi].transpose(0, 1), keys[of].transpose(2, 3)) * scale
            so = torch.where(at < s["lens"][of, None, None, None], so, -math.inf).transpose(0, 1)
        else:
            so = torch.full((kv, hi - lo, group, keys.shape[2]), -math.inf, device="cuda")
            for b in range(p * per, (p + 1) * per):
                i, j, rows = starts[b] - lo, starts[b + 1] - lo, s["rows_list"][b]
                part = torch.matmul(q[:, lo + i:lo + j].reshape(kv, -1, dim), keys[b].transpose(1, 2)) * scale
                limit = s["lens_list"][b] - rows + 1 + torch.arange(rows, device="cuda")
                so[:, i:j] = torch.where(at < limit[:, None, None], part.view(kv, rows, group, -1), -math.inf)
        peak = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
        sp, so = torch.exp(sp - peak), torch.exp(so - peak)
        total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
        lse[:, lo:hi] = (peak + torch.log(total))[..., 0]
        o = torch.matmul(sp.view(kv, -1, sp.shape[3]), s["prefix_v"][p].float()).view(kv, hi - lo, group, dim)
        if one:
            o = o + torch.matmul(so.transpose(0, 1), values[of]).transpose(0, 1)
        else:
            for b in range(p * per, (p + 1) * per):
                i, j = starts[b] - lo, starts[b + 1] - lo
                part = torch.matmul(so[:, i:j].reshape(kv, -1, so.shape[3]), values[b])
                o[:, i:j] += part.view(kv, j - i, group, dim)
        out[:, lo:hi] = o / total
    return (out.transpose(0, 1).reshape(-1, heads, dim).to(torch.bfloat16), lse.transpose(0, 1).reshape(-1, heads))


def _plain_select(s):
    batch, beams, select, vocab = s["batch"], s["beams"], s["select"], s["vocab"]
    logits = s["logits"].float()
    peak = logits.amax(1, keepdim=True)
    # Candidates of different beams are compared in 64 bits; the sums of 32-bit exponentials are taken there too.
    total = torch.exp(logits - peak).double().sum(1, keepdim=True)
    scores = s["scores"].reshape(-1, 1).double()
    cand = scores + (logits.double() - (peak.double() + torch.log(total)))
    if s["finished"] is not None:
        done = s["finished"].reshape(-1, 1) != 0
        cand = torch.where(done, -math.inf, cand)
        cand[:, s["eos"]] = torch.where(done, scores, cand[:, s["eos"]:s["eos"] + 1])[:, 0]
    # The first of equal candidates comes first: a stable order of each beam's best, then of all beams'.
    few = min(vocab, 4 * select + 64)
    best, token = cand.topk(few, dim=1)
    token, by_token = token.sort(dim=1)
    best, order = best.gather(1, by_token).sort(dim=1, descending=True, stable=True)
    token = token.gather(1, order)
    best, token = best[:, :select].reshape(batch, -1), token[:, :select].reshape(batch, -1)
    best, order = best.sort(dim=1, descending=True, stable=True)
    best, order = best[:, :select], order[:, :select]
    tokens = token.gather(1, order).to(torch.int32)
    parents = (order // min(select, vocab)).to(torch.int32)
    finished = tokens == s["eos"]
    if s["finished"] is not None:
        finished = finished | (s["finished"].gather(1, parents.long()) != 0)
    return tokens, parents, best.float(), finished.to(torch.int32)


def _plain_reorder(s):
    state, beams = s["state"], s["beams"]
    rows = torch.arange(state.shape[1], device="cuda") // beams * beams + s["parents"]
    held = torch.arange(state.shape[3], device="cuda") < s["counts"][rows, None]
    state.copy_(torch.where(held[None, :, None, :, None], state[:, rows], state))
    return state


def run(state):
    s = state
    if not own:
        return {"rotate": _plain_rotate, "attention": _plain_attention, "select": _plain_select,
                "reorder": _plain_reorder}[s["op"]](s)
    api = _framework()
    if s["op"] == "rotate":
        api.rotate_heads(s["q"], s["k"], s["v"], s["inv_freq"], s["positions"], s["q_out"], s["k_cache"], s["v_cache"],
                         q_norm=s["q_norm"], k_norm=s["k_norm"], cache_rows=s["cache_rows"], slots=s["slots"],
                         interleaved=s["interleaved"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    if s["op"] == "attention":
        api.prefix_attention(s["q"], s["prefix_k"], s["prefix_v"], s["prefix_lens"], s["k"], s["v"], s["lens"],
                             s["out"], ancestry=s["ancestry"], row_offsets=s["row_offsets"], lse=s["lse"])
        return s["out"], s["lse"]
    if s["op"] == "select":
        api.beam_select(s["logits"], s["scores"], s["tokens"], s["parents"], s["new_scores"],
                        finished=s["finished"], new_finished=s["new_finished"], eos=s["eos"])
        return s["tokens"], s["parents"], s["new_scores"], s["new_finished"]
    api.reorder_states(s["state"], s["parents"], s["beams"], counts=s["counts"])
    return s["state"]


def work(case):
    """Bytes: inputs once, outputs once. Operations: two for each multiply-add (attention: the products' alone)."""
    if case["op"] == "rotate":
        n = case["rows"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 2 * n + 12 * case["rows"],
                "flops": n * (7 if case["norm"] else 3)}
    if case["op"] == "attention":
        lens, rows = _own_lens(case)
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        seen = sum(r * case["prefix"] + r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, rows))
        return {"bytes": (case["prefixes"] * case["prefix"] + sum(lens)) * kv * dim * 4
                + sum(rows) * heads * (4 * dim + 4) + (4 * sum(lens) if case["ancestry"] else 0),
                "flops": 4 * seen * heads * dim}
    if case["op"] == "select":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 16 * case["batch"] * case["select"],
                "flops": 3 * n}
    kept = max(1, case["beams"] // 2)
    moved = case["beams"] - kept
    unit = case["layers"] * case["groups"] * case["segments"] * (case["units"] - case["units"] // 8) * case["width"]
    return {"bytes": (min(kept, moved) + moved) * unit, "flops": 0}


def _exact_rotate(s):
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["inv_freq"].double()))[:, None, :]
    rot = s["rotary"]

    def heads(x, gain):
        x = x.double()
        if gain is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / s["dim"] + 1e-6) * gain.double()
        head, tail = x[..., :rot], x[..., rot:]
        if s["interleaved"]:
            z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
            head = torch.view_as_real(z).reshape(head.shape)
        else:
            z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, tail], -1)

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    where = (s["cache_rows"].long(), slice(None), s["slots"].long())
    k_cache[where] = heads(s["k"], s["k_norm"])
    v_cache[where] = s["v"].double()
    return heads(s["q"], s["q_norm"]), k_cache, v_cache


def _exact_attention(s):
    group, per = s["heads"] // s["kv_heads"], s["sequences"] // s["prefixes"]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["lse"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b in range(s["sequences"]):
        rows, length, p = s["rows_list"][b], s["lens_list"][b], b // per
        for h in range(s["kv_heads"]):
            if s["ancestry"] is None:
                k, v = s["k"][b, h, :length], s["v"][b, h, :length]
            else:
                cell = (s["ancestry"][b, :length].long(), h, torch.arange(length, device="cuda"))
                k, v = s["k"][cell], s["v"][cell]
            k = torch.cat([s["prefix_k"][p, h], k]).double()
            v = torch.cat([s["prefix_v"][p, h], v]).double()
            q = s["q"][row:row + rows, h * group:(h + 1) * group].double()
            z = torch.einsum("rgd,kd->rgk", q, k) / math.sqrt(s["dim"])
            key = torch.arange(k.shape[0], device="cuda")
            last = k.shape[0] - rows + torch.arange(rows, device="cuda")
            z = z.masked_fill((key[None, :] > last[:, None])[:, None, :], -math.inf)
            out[row:row + rows, h * group:(h + 1) * group] = torch.einsum("rgk,kd->rgd", torch.softmax(z, -1), v)
            lse[row:row + rows, h * group:(h + 1) * group] = torch.logsumexp(z, -1)
        row += rows
    return out, lse


def _exact_select(s):
    batch, beams, select, vocab = s["batch"], s["beams"], s["select"], s["vocab"]
    z = torch.log_softmax(s["logits"].double(), 1).view(batch, beams, vocab) + s["scores"].double()[:, :, None]
    if s["finished"] is not None:
        for b, k in (s["finished"] != 0).nonzero().tolist():
            z[b, k] = -math.inf
            z[b, k, s["eos"]] = s["scores"][b, k].double()
    z = z.view(batch, -1)
    value, flat = z.sort(dim=1, descending=True, stable=True)
    value, flat = value[:, :select], flat[:, :select]
    tokens, parents = flat % vocab, flat // vocab
    finished = tokens == s["eos"]
    if s["finished"] is not None:
        finished |= torch.gather(s["finished"], 1, parents) != 0
    return tokens.to(torch.int32), parents.to(torch.int32), value, finished.to(torch.int32)


def exact(case, seed):
    if case["op"] == "reorder":
        return None  # whole numbers, moved and not computed
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "attention": _exact_attention, "select": _exact_select}[case["op"]](s)
