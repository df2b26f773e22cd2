"""Attention behind shared prefixes on the GPU against a plain 64-bit form.

Tolerance. With exact bf16 inputs a score's products are exact and its sum of
`dim` terms is off by at most dim * 2^-23 of the terms' magnitudes (the tensor
cores may cut instead of round): d = scale * sum |q k| * dim * 2^-23, plus 2^-22
|s| for the change to base 2; a weight is then off by the factor exp(2 d) and
2^-21 of the exponential, and by half a step of bf16, 2^-8, as the operand of
the second product, whose sum over n keys (and the sum of the weights, and the
joins' factors) is off by (n + 64) * 2^-23 of the magnitudes. So with A = sum p |v|
the output is off by A * (2^-8 + 2 d + (n + 64) * 2^-22), and by its own rounding,
2^-8 of itself; lse by d + (n + 64) * 2^-22 + 2^-22 |lse|.
"""
import math

import pytest

import uocr_moe as M

pytestmark = pytest.mark.gpu


def gen_of(*key):
    import torch
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)) + 1)


def plain(c):
    """(out, lse, tolerance of out, of lse) in 64 bits; rows of no sequence are NaN."""
    import torch
    q, k, v = c["q"].double(), c["k"], c["v"]
    rows, heads, dim = q.shape
    kv = k.shape[1]
    n_seq, prefixes = c["lens"].numel(), c["prefix_lens"].numel()
    offsets = list(range(n_seq + 1)) if c["row_offsets"] is None else c["row_offsets"].tolist()
    out, lse, tol, tol_lse = (torch.full(s, math.nan, dtype=torch.float64, device="cuda")
                              for s in ((rows, heads, dim), (rows, heads), (rows, heads, dim), (rows, heads)))
    scale = c["scale"]
    for b in range(n_seq):
        p, r0, r1, n = b // (n_seq // prefixes), offsets[b], offsets[b + 1], int(c["lens"][b])
        plen = int(c["prefix_lens"][p])
        of = torch.full((n,), b, device="cuda") if c["ancestry"] is None else c["ancestry"][b, :n].long()
        at = torch.arange(n, device="cuda")
        limit = n - (r1 - r0) + 1 + torch.arange(r1 - r0, device="cuda")
        seen = torch.cat([torch.ones(r1 - r0, plen, dtype=torch.bool, device="cuda"), at < limit[:, None]], 1)
        for h in range(heads):
            g = h // (heads // kv)
            kk = torch.cat([c["prefix_k"][p, g, :plen], k[of, g, at]]).double()
            vv = torch.cat([c["prefix_v"][p, g, :plen], v[of, g, at]]).double()
            qq = q[r0:r1, h]
            s = torch.where(seen, scale * qq @ kk.T, -math.inf)
            size = torch.where(seen, abs(scale) * qq.abs() @ kk.abs().T, 0.0)
            d = (size.amax(1) if s.shape[1] else torch.zeros(r1 - r0, device="cuda")).double() * (dim * 2.0 ** -23 + 2.0 ** -22)
            top = s.amax(1, keepdim=True) if s.shape[1] else torch.full((r1 - r0, 1), -math.inf, device="cuda").double()
            w = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            keys = (seen.sum(1) + 64) * 2.0 ** -22
            out[r0:r1, h] = w @ vv
            lse[r0:r1, h] = (torch.log(total) + top)[:, 0]
            tol[r0:r1, h] = (w @ vv.abs()) * (2.0 ** -8 + 2 * d + keys)[:, None] + 2.0 ** -8 * out[r0:r1, h].abs()
            tol_lse[r0:r1, h] = d + keys + 2.0 ** -22 * lse[r0:r1, h].abs()
    return out, lse, tol, tol_lse


def make(prefix_lens, lens, heads, kv, dim, rows=None, beams=False, prefix_capacity=None, capacity=None, first_row=0,
         rows_behind=0, spread=1.0, seed=0):
    """rows: query rows of each sequence (None: one each, without offsets)."""
    import torch
    g = gen_of(len(prefix_lens), sum(prefix_lens), sum(lens), heads, kv, dim, seed)
    bf16, i32 = torch.bfloat16, torch.int32
    pcap = max(prefix_lens) + 3 if prefix_capacity is None else prefix_capacity
    cap = max(lens) + 5 if capacity is None else capacity
    n = len(lens)

    def values(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * spread).to(bf16)

    c = dict(prefix_k=values(len(prefix_lens), kv, pcap, dim), prefix_v=values(len(prefix_lens), kv, pcap, dim),
             k=values(n, kv, cap, dim), v=values(n, kv, cap, dim), ancestry=None, row_offsets=None, scale=dim ** -0.5)
    # What lies behind the lengths is no number.
    for p, length in enumerate(prefix_lens):
        c["prefix_k"][p, :, length:] = math.nan
        c["prefix_v"][p, :, length:] = math.inf
    if beams:
        per = n // len(prefix_lens)
        base = torch.arange(n, device="cuda")[:, None] // per * per
        c["ancestry"] = (torch.randint(0, per, (n, cap), generator=g, device="cuda") + base).to(i32)
        for b in range(n):
            c["ancestry"][b, lens[b]:] = 1 << 30
    else:
        for b, length in enumerate(lens):
            c["k"][b, :, length:] = math.nan
            c["v"][b, :, length:] = math.nan
    c["prefix_lens"] = torch.tensor(prefix_lens, dtype=i32, device="cuda")
    c["lens"] = torch.tensor(lens, dtype=i32, device="cuda")
    total = n if rows is None else first_row + sum(rows) + rows_behind
    if rows is not None:
        c["row_offsets"] = torch.tensor([first_row + sum(rows[:i]) for i in range(n + 1)], dtype=i32, device="cuda")
    c["q"] = values(total, heads, dim)
    c["out"] = torch.full((total, heads, dim), 33.0, dtype=bf16, device="cuda")
    c["lse"] = torch.full((total, heads), 44.0, device="cuda")
    return c


def check(c, call=True):
    import torch
    if call:
        M.prefix_attention(**c)
        M.ops_check()
    out, lse, tol, tol_lse = plain(c)
    none = out.isnan()
    assert (c["out"][none] == 33.0).all() and (c["lse"][none[..., 0]] == 44.0).all()
    live = ~none[..., 0]
    got, want = c["out"][live].double(), out[live]
    over = (got - want).abs() - tol[live]
    assert not over.isnan().any() and (over.numel() == 0 or over.max().item() <= 0), over.max().item()
    empty = live & (lse == -math.inf)
    assert torch.equal(c["lse"] == -math.inf, empty) and (c["out"][empty] == 0).all()
    some = live & ~empty
    over = (c["lse"][some].double() - lse[some]).abs() - tol_lse[some]
    assert not over.isnan().any() and (over.numel() == 0 or over.max().item() <= 0), over.max().item()


@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 128), (10, 10, 128), (8, 1, 64), (9, 3, 64), (14, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("prefix_lens,lens", [
    ([4096], [300, 17, 1, 255]), ([1], [1]), ([700, 0, 63], [5, 0, 9, 64, 65, 1]), ([0, 0], [0, 3]),
    ([128, 129], [0, 0, 0, 0]), ([1000], [1] * 33)])
def test_one_token_each(cuda, prefix_lens, lens, heads, kv, dim):
    check(make(prefix_lens, lens, heads, kv, dim))


@pytest.mark.parametrize("prefix_lens,lens,heads,kv,dim", [
    ([4096], [300] * 4, 16, 4, 128), ([100, 300, 5], [37] * 12, 8, 2, 64), ([2500, 2500], [64, 1, 65, 200] * 4, 4, 4, 128)])
def test_beams_that_share_ancestors(cuda, prefix_lens, lens, heads, kv, dim):
    check(make(prefix_lens, lens, heads, kv, dim, beams=True))


@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 128), (9, 3, 64), (2, 2, 128), (12, 2, 64)])
@pytest.mark.parametrize("prefix_lens,lens,rows", [
    ([1001], [61, 30, 9, 100], [37, 30, 1, 80]),
    ([64, 500], [5, 2, 0, 200], [5, 7, 3, 120]),       # rows before their sequence's keys: some see the prefix alone
    ([0, 0], [4, 3, 0, 9], [6, 3, 2, 1]),              # and some nothing
    ([333], [50, 20, 70], [0, 20, 0]),                 # sequences without rows
    ([2000], [160] * 9, [160] * 9), ([0], [700], [700])])
def test_rows_of_any_number(cuda, prefix_lens, lens, rows, heads, kv, dim):
    check(make(prefix_lens, lens, heads, kv, dim, rows=rows))


@pytest.mark.parametrize("first,behind", [(0, 7), (3, 0), (5, 70)])
def test_rows_outside_the_sequences_stay(cuda, first, behind):
    check(make([300], [40, 8, 3], 8, 2, 128, rows=[20, 8, 1], first_row=first, rows_behind=behind))


@pytest.mark.parametrize("sequences", [64, 100])
def test_many_sequences_on_one_prefix(cuda, sequences):
    check(make([5000], [1 + i % 40 for i in range(sequences)], 16, 4, 128))


@pytest.mark.parametrize("heads,kv,rows", [(8, 2, None), (24, 2, None), (8, 2, [3, 20, 1])])
def test_without_room_for_keys(cuda, heads, kv, rows):
    """Capacities of zero: of the prefixes, of the own keys, of both."""
    check(make([0], [5, 70, 9], heads, kv, 128, rows=rows, prefix_capacity=0))
    check(make([40], [0, 0, 0], heads, kv, 128, rows=rows, capacity=0))
    check(make([0], [0, 0, 0], heads, kv, 128, rows=rows, prefix_capacity=0, capacity=0))


def test_a_long_prefix(cuda):
    check(make([33001], [3, 9], 8, 2, 128))


def test_more_keys_than_the_lengths_say(cuda):
    check(make([70, 5], [3, 9, 1, 0], 8, 2, 128, prefix_capacity=9000, capacity=2000))


@pytest.mark.parametrize("spread", [6.0, 0.0])
def test_peaked_and_flat_scores(cuda, spread):
    check(make([900, 40], [33, 80, 7, 1], 8, 2, 128, spread=spread))


def test_scores_that_rise_along_the_keys(cuda):
    """The running maximum moves at every key."""
    import torch
    c = make([3000], [200, 100], 4, 2, 64)
    ramp = torch.linspace(-4, 4, 3000, device="cuda")
    c["q"].fill_(1.0)
    c["prefix_k"][0, :, :3000] = ramp[:, None].to(torch.bfloat16)
    check(c)


def test_infinite_and_nan_inputs_stay_in_their_rows(cuda):
    import torch
    c = make([200], [20, 30, 40], 4, 2, 128, rows=[4, 5, 6])
    c["q"][6] = math.nan                 # a row of the second sequence
    c["v"][2, 1, 39] = math.inf          # the last own value of the third: its last row's alone
    M.prefix_attention(**c)
    got = c["out"].float()
    assert got[6].isnan().all() and not got[:6].isnan().any() and not got[7:14].isnan().any()
    assert got[14, :2].isfinite().all() and got[14, 2:].isinf().all()
    assert got[:6].isfinite().all() and got[7:14].isfinite().all()


def test_scale_and_strides(cuda):
    import torch
    c = make([513, 77], [90, 3, 0, 45], 6, 2, 64, rows=[9, 3, 2, 45])
    c["scale"] = 0.37

    def spread(t, axes):  # the same values inside a larger buffer
        shape = [s + 8 * (a in axes) for a, s in enumerate(t.shape)]
        wide = torch.full(shape, math.nan, dtype=t.dtype, device="cuda")
        view = wide[tuple(slice(0, s) for s in t.shape)]
        view.copy_(t)
        return view
    for name in ("prefix_k", "prefix_v", "k", "v"):
        c[name] = spread(c[name].transpose(0, 1).contiguous(), (1, 2)).transpose(0, 1)
    c["q"], c["out"] = spread(c["q"], (1,)), spread(c["out"], (1,))
    check(c)


def test_offsets_above_32_bits(cuda):
    """A cache of more than 2^32 bytes and 2^31 elements."""
    import torch
    kv, dim, cap = 2, 128, 1100
    caches = 8000  # 2.25e9 elements each
    n = 3
    g = gen_of(caches)
    k = torch.empty(caches, kv, cap, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    table = torch.tensor([caches - 1, 0, caches - 7], device="cuda")
    for t in (k, v):
        for row in table.tolist():
            t[row].copy_(torch.randn(kv, cap, dim, generator=g, device="cuda"))
    c = make([100], [1000, 20, 333], 8, kv, dim, capacity=cap)
    c["k"], c["v"] = k, v
    c["ancestry"] = table.to(torch.int32)[:, None].expand(n, cap).contiguous()
    check(c)


@pytest.mark.parametrize("what", ["prefix_lens", "lens", "ancestry", "row_offsets"])
def test_bad_lengths_offsets_and_ancestors_are_reported(cuda, what):
    import torch
    for value in (1 << 30, -5):
        c = make([200, 100], [20, 30, 10, 5], 4, 2, 128, rows=[3, 3, 3, 3], beams=True)
        if what == "ancestry":
            c[what][1, 7] = value
        else:
            c[what][1] = value
        M.prefix_attention(**c)
        with pytest.raises(M.UocrError) as e:
            M.ops_check()
        assert e.value.code == 5 and "prefix_attention" in str(e.value)
        M.ops_check()
        if what in ("prefix_lens", "lens"):  # taken as the nearest in range
            c[what][1] = 0 if value < 0 else c["prefix_k" if what == "prefix_lens" else "k"].shape[2]
            if value < 0:
                check(c)


def test_runs_are_bitwise_repeatable_on_streams_and_from_graphs(cuda):
    import torch
    c = make([3000, 100], [120, 7, 60, 200], 16, 4, 128, beams=True)
    check(c)
    want, want_lse = c["out"].clone(), c["lse"].clone()
    d = make([500], [30, 90, 1], 8, 2, 64, rows=[30, 5, 1], seed=3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):  # two calls at once, with workspaces of their own
        c["out"].fill_(1.0)
        torch.cuda.synchronize()
        M.prefix_attention(**c, stream=side)
        M.prefix_attention(**d)
        torch.cuda.synchronize()
        assert torch.equal(c["out"], want) and torch.equal(c["lse"], want_lse)
    check(d, call=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.prefix_attention(**c)
    # A replay takes the lengths as they are then.
    c["lens"].copy_(torch.tensor([121, 8, 61, 201], device="cuda"))
    c["prefix_lens"][1] = 102
    c["prefix_k"][1, :, 100:102] = 0.5
    c["prefix_v"][1, :, 100:102] = 0.25
    c["ancestry"].clamp_(max=3)
    graph.replay()
    torch.cuda.synchronize()
    check(c, call=False)


def test_the_lse_joins_parts_of_a_prefix(cuda):
    """Two halves of a prefix, joined by their lse, are the whole."""
    import torch
    c = make([1000], [0, 0, 0], 8, 2, 128, prefix_capacity=1000)
    check(c)
    parts = []
    for half in (slice(0, 400), slice(400, 1000)):
        d = dict(c, prefix_k=c["prefix_k"][:, :, half].contiguous(), prefix_v=c["prefix_v"][:, :, half].contiguous(),
                 prefix_lens=torch.tensor([half.stop - half.start], dtype=torch.int32, device="cuda"),
                 out=torch.empty_like(c["out"]), lse=torch.empty_like(c["lse"]))
        M.prefix_attention(**d)
        parts.append((d["out"].double(), d["lse"].double()))
    (a, la), (b, lb) = parts
    joined = torch.logaddexp(la, lb)
    assert (joined - c["lse"].double()).abs().max() < 1e-4
    both = a * (la - joined).exp()[..., None] + b * (lb - joined).exp()[..., None]
    _, _, tol, _ = plain(c)
    # each half and the whole within their tolerances: the halves' add up to at most the whole's of |a| and |b|
    assert ((both - c["out"].double()).abs() <= 3 * tol + 2.0 ** -7 * (a.abs() + b.abs())).all()


# ---- many rows of many prefixes, and keys in parts

@pytest.mark.parametrize("dim", [64, 128])
def test_many_prefixes_with_many_rows(cuda, dim):
    lengths = [(37 * i) % 700 if i % 5 else 0 for i in range(40)]
    check(make(lengths, [(11 * i) % 90 for i in range(200)], 8, 2, dim))


@pytest.mark.parametrize("dim", [64, 128])
def test_many_prefixes_with_more_rows_than_a_tile(cuda, dim):
    rows = [50 + i % 3 if i % 7 else 0 for i in range(70)]
    lens = [n + (5 * i) % 60 for i, n in enumerate(rows)]
    check(make([(53 * i) % 400 for i in range(35)], lens, 8, 2, dim, rows=rows))


@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 128), (8, 2, 64), (12, 1, 128)])
@pytest.mark.parametrize("rows", [[90, 2, 2], [2, 1, 0], [0, 0, 96], [600, 0, 1], [1, 129, 300]])
def test_prefixes_with_unlike_rows(cuda, rows, heads, kv, dim):
    check(make([1000, 50, 2700], [max(n, 40) for n in rows], heads, kv, dim, rows=rows, first_row=2, rows_behind=3))


@pytest.mark.parametrize("what", ["prefix_lens", "lens", "ancestry", "row_offsets"])
def test_bad_values_with_many_rows_are_reported(cuda, what):
    import torch
    for value in (1 << 30, -5):
        c = make([200, 100], [20, 30, 10, 5], 8, 2, 128, rows=[30, 40, 10, 30], beams=True)
        if what == "ancestry":
            c[what][1, 7] = value
        else:
            c[what][1] = value
        M.prefix_attention(**c)
        with pytest.raises(M.UocrError) as e:
            M.ops_check()
        assert e.value.code == 5 and "prefix_attention" in str(e.value)
        M.ops_check()
        if what in ("prefix_lens", "lens") and value < 0:
            c[what][1] = 0
            check(c)


@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_scales_that_are_not_positive(cuda, scale):
    c = make([600, 90], [40, 70, 20, 33], 8, 2, 128, rows=[40, 30, 20, 1])
    c["scale"] = scale
    check(c)


@pytest.mark.parametrize("rows", [None, [40, 50, 30, 64]])
def test_heads_and_sequences_that_share_memory(cuda, rows):
    c = make([300, 200], [60, 70, 30, 90], 8, 2, 64, rows=rows)
    for name in ("prefix_k", "prefix_v"):
        c[name] = c[name][:, :1].expand(-1, 2, -1, -1)
    for name in ("k", "v"):
        c[name] = c[name][:, 1:].expand(-1, 2, -1, -1)
    check(c)


@pytest.mark.parametrize("length", [64, 128, 129, 200, 257, 300, 511])
def test_infinite_values_stay_infinite(cuda, length):
    """One visible value after another is infinite: so are its rows, and no other."""
    for key in sorted({0, length // 3, length // 2, length - 2, length - 1}):
        c = make([length, 90], [60, 70], 8, 2, 128, rows=[60, 70])
        c["prefix_v"][0, 1, key] = -math.inf
        M.prefix_attention(**c)
        got = c["out"].float()
        assert (got[:60, 4:] == -math.inf).all() and got[:60, :4].isfinite().all() and got[60:].isfinite().all()


def test_nan_rows_of_many_stay_alone(cuda):
    import torch
    c = make([900, 300], [60, 70], 8, 2, 128, rows=[60, 70])
    c["q"][17] = math.nan
    c["prefix_v"][1, :, 11] = math.inf  # the second prefix's rows alone
    M.prefix_attention(**c)
    got = c["out"].float()
    others = [r for r in range(60) if r != 17]
    assert got[17].isnan().all() and got[others].isfinite().all() and got[60:].isinf().all()


@pytest.mark.parametrize("beams", [False, True])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (12, 12, 64), (24, 2, 64)])
@pytest.mark.parametrize("prefix_lens,lens", [([100], [3000, 10, 0, 600]), ([0, 70], [1, 2000]), ([300], [5000])])
def test_long_own_keys(cuda, prefix_lens, lens, heads, kv, dim, beams):
    check(make(prefix_lens, lens, heads, kv, dim, beams=beams))


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (9, 1, 64)])
def test_long_own_keys_of_several_rows(cuda, heads, kv, dim):
    check(make([400, 1], [2000, 3, 900, 700], heads, kv, dim, rows=[5, 6, 0, 33]))
    check(make([400], [2500], heads, kv, dim, rows=[150], beams=True))


def test_a_prefix_for_each_of_many_sequences(cuda):
    check(make([(17 * i) % 300 for i in range(140)], [(29 * i) % 900 for i in range(140)], 4, 1, 64, capacity=905))
    check(make([(17 * i) % 300 for i in range(300)], [(29 * i) % 90 for i in range(300)], 4, 2, 128))


@pytest.mark.parametrize("heads,kv", [(24, 2), (16, 4), (8, 1)])
def test_many_beams_with_and_without_own_keys(cuda, heads, kv):
    check(make([500, 0], [0, 3, 90, 64, 65, 0, 1, 200] * 10, heads, kv, 128, beams=True))


def test_many_rows_on_a_stream_and_from_a_graph(cuda):
    import torch
    c = make([900, 0, 300], [60, 70, 40], 8, 2, 128, rows=[60, 70, 33])
    d = make([500], [1000, 7], 8, 2, 64, seed=5)
    check(c)
    want, side = c["out"].clone(), torch.cuda.Stream()
    for _ in range(4):
        c["out"].fill_(33.0)
        torch.cuda.synchronize()
        M.prefix_attention(**c, stream=side)
        M.prefix_attention(**d)
        torch.cuda.synchronize()
        assert torch.equal(c["out"], want)
    check(d, call=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.prefix_attention(**c)
    c["prefix_lens"].copy_(torch.tensor([0, 500, 301], device="cuda"))
    for name in ("prefix_k", "prefix_v"):
        c[name][1, :, :500] = 0.5
        c[name][2, :, 300] = 0.25
    c["row_offsets"].copy_(torch.tensor([0, 20, 90, 163], device="cuda"))
    c["lens"].copy_(torch.tensor([20, 70, 45], device="cuda"))
    for name in ("k", "v"):
        c[name].nan_to_num_(0.125)
    graph.replay()
    torch.cuda.synchronize()
    check(c, call=False)


# ---- scores of any magnitude

def level_case(level, rows, lengths, dim, scale_log=8):
    """Rows of sequences behind prefixes; a row's scores are exact in fp32: sums of products of powers of two, most of
    them `level` * 2^-8, and of some keys, the row's greatest, all the same."""
    import torch
    c = make(lengths, [40 + 7 * i for i in range(len(rows))], 8, 2, dim, rows=rows)
    c["scale"] = 2.0 ** scale_log
    # score = scale * q . k = scale * dim * q * k
    unit = level / (c["scale"] * dim)
    q = 2.0 ** 8
    c["q"].fill_(q)
    for name in ("prefix_k", "k"):
        t = c[name]
        real = t[..., 0].isfinite()
        t[real] = 0.0
        index = torch.arange(t.shape[2], device="cuda")
        best = (index % 5 == 3).expand(t.shape[:3]) & real
        # positive levels: the best keys alone have them; negative ones: all keys, the best half as far down
        t[real] = 0.0 if level > 0 else 2.0 * unit / q
        t[best] = unit / q
    return c


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("level", [2.0 ** 12, 2.0 ** 26, 2.0 ** 31, 2.0 ** 34, 2.0 ** 60, -2.0 ** 12, -2.0 ** 26,
                                   -2.0 ** 33, -2.0 ** 34, -2.0 ** 60])
@pytest.mark.parametrize("rows,lengths", [([60, 70], [300, 200]), ([9, 11], [300, 90]), ([600, 3], [1000, 128]),
                                          ([2, 1], [700, 130])])
def test_scores_of_any_magnitude(cuda, level, rows, lengths, dim):
    """Many keys with a row's greatest score share its weight, however large the score is and however many rows there are."""
    import torch
    c = level_case(level, rows, lengths, dim)
    M.prefix_attention(**c)
    M.ops_check()
    per, r0 = len(rows) // len(lengths), 0
    for b, n in enumerate(rows):
        plen, own = lengths[b // per], int(c["lens"][b])
        for j in range(n):
            seen = max(0, own - (n - 1 - j))
            pick = torch.arange(plen, device="cuda") % 5 == 3
            mine = torch.arange(seen, device="cuda") % 5 == 3
            if j not in (0, n // 2, n - 1) or not (pick.any() or mine.any()):
                continue
            for h in (0, 7):
                v = torch.cat([c["prefix_v"][b // per, h // 4, :plen][pick], c["v"][b, h // 4, :seen][mine]]).double()
                want = v.mean(0)
                # n equal weights, 1 or (a key that two tiles have) 1/2 each: exact in bf16; their fp32 sums, and the result's rounding
                tol = (v.shape[0] + 64) * 2.0 ** -22 * v.abs().mean(0) + 2.0 ** -8 * want.abs() + 1e-30
                got = c["out"][r0 + j, h].double()
                assert ((got - want).abs() <= tol).all(), (b, j, h, (got - want).abs().max().item())
                lse = level + math.log(v.shape[0])
                assert abs(c["lse"][r0 + j, h].item() - lse) <= 2.0 ** -21 * abs(lse)
        r0 += n


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [[60, 70], [300, 9], [2, 1]])
@pytest.mark.parametrize("levels", [[-2.0 ** 34, 1.0], [1.0, -2.0 ** 34], [-2.0 ** 40, -2.0 ** 34, -2.0 ** 33, -2.0 ** 12, -2.0 ** 11, 1.0],
                                    [-2.0 ** 12, -2.0 ** 10, 1.0, -2.0 ** 36], [-2.0 ** 60, -2.0 ** 60, -2.0 ** 11, 1.0]])
def test_scores_that_come_from_afar(cuda, levels, rows, dim):
    """Keys with ordinary scores before, behind and between keys far below them, 150 of each in turn: those have no weight."""
    import torch
    c = make([1000, 515], [40, 50], 8, 2, dim, rows=rows)
    c["scale"] = 1.0
    c["q"].zero_()
    c["q"][..., 0] = 1.0
    ordinary = []  # of each prefix, the keys that count, and those that do without them: the highest level's
    for p, n in enumerate([1000, 515]):
        level = torch.tensor(levels, device="cuda")[torch.arange(n, device="cuda") // 150 % len(levels)]
        t = c["prefix_k"][p, :, :n]
        t.copy_(torch.where((level == 1.0)[None, :, None], t, level[None, :, None].to(t.dtype)))
        ordinary.append((level == 1.0, level == level.max()))
    M.prefix_attention(**c)
    M.ops_check()
    r0 = 0
    for b, n in enumerate(rows):
        own = int(c["lens"][b])
        for j in (0, n // 2, n - 1):
            seen = max(0, own - (n - 1 - j))
            for h in (0, 7):
                g, (at, highest) = h // 4, ordinary[b]
                plen = at.numel()
                at = at if at.any() or seen > 0 else highest
                s = torch.cat([c["prefix_k"][b, g, :plen, 0][at], c["k"][b, g, :seen, 0]]).double()
                v = torch.cat([c["prefix_v"][b, g, :plen][at], c["v"][b, g, :seen]]).double()
                w = torch.softmax(s, 0)
                # The scores are single products with 1, exact. A weight is rounded to bf16 and off by the rounding of a
                # shift of up to 1024 (2^-14 of an exponent) and 2^-20 else; then the sums, and the result's rounding.
                tol = (w @ v.abs()) * (2.0 ** -8 + 2.0 ** -13 + (s.numel() + 64) * 2.0 ** -22) + 2.0 ** -8 * (w @ v).abs()
                got = c["out"][r0 + j, h].double()
                assert ((got - w @ v).abs() <= tol).all(), (b, j, h, ((got - w @ v).abs() - tol).max().item())
                lse = torch.logsumexp(s, 0).item()
                assert abs(c["lse"][r0 + j, h].item() - lse) <= 2.0 ** -13 + (s.numel() + 64) * 2.0 ** -22 + 2.0 ** -21 * abs(lse)
        r0 += n


def test_a_scale_too_small_for_its_inverse(cuda):
    c = make([600, 90], [40, 70, 20, 33], 8, 2, 128, rows=[40, 30, 20, 1])
    for scale in (1e-38, 1e-39, 1e-44):
        c["scale"] = scale
        check(c)


@pytest.mark.parametrize("heads,keys", [(1, 32800), (32, 16000)])
def test_row_offsets_that_name_rows_many_times_over(cuda, heads, keys):
    """The sum of what they name is more than 2^32 units of work, for the kernels of few and of many rows: reported, and
    nothing outside the rows is written."""
    import torch
    n, dim, bf16, i32 = 16384, 64, torch.bfloat16, torch.int32
    memory = torch.randn(keys + n, dim, generator=gen_of(heads, keys), device="cuda").to(bf16)
    prefix = torch.as_strided(memory, (n, 1, keys, dim), (0 if heads == 1 else dim, keys * dim, dim, 1))
    none = torch.empty(n, 1, 0, dim, dtype=bf16, device="cuda")
    whole = torch.full((n + 2, heads, dim), 33.0, dtype=bf16, device="cuda")
    q = torch.randn(n, heads, dim, generator=gen_of(heads), device="cuda").to(bf16)
    offsets = torch.zeros(n + 1, dtype=i32, device="cuda")
    offsets[1::2] = n
    c = dict(q=q, prefix_k=prefix, prefix_v=prefix, prefix_lens=torch.full((n,), keys, dtype=i32, device="cuda"), k=none,
             v=none, lens=torch.zeros(n, dtype=i32, device="cuda"), out=whole[1:-1], row_offsets=offsets)
    M.prefix_attention(**c)
    with pytest.raises(M.UocrError) as e:
        M.ops_check()
    assert e.value.code == 5 and "rows" in str(e.value)
    assert (whole[0] == 33.0).all() and (whole[-1] == 33.0).all()
    # The same call in order, a row each behind a few keys.
    offsets.copy_(torch.arange(n + 1, device="cuda"))
    c["prefix_lens"].fill_(70)
    M.prefix_attention(**c)
    M.ops_check()
    for row in (0, 1, 8191, n - 1):
        k = prefix[row, 0, :70].double()
        w = torch.softmax(q[row].double() @ k.T * dim ** -0.5, -1)
        tol = (w @ k.abs()) * (2.0 ** -8 + 2.0 ** -12) + 2.0 ** -8 * (w @ k).abs()  # see above; 134 keys, |s| below 40
        assert ((whole[1 + row].double() - w @ k).abs() <= tol).all()
