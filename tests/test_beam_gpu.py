"""The rotation of heads, the selection of beams and the reordering of states on
the GPU against plain 64-bit forms.

Tolerances. Rotation: the sum of n <= 256 squares is off by at most n * 2^-24 of
itself, its root by half of that; rsqrt, the mean, the products with gain,
cosine and sine and the magnitude add 8 roundings of 2^-24 and the 2 ulp of
rsqrt and of sine and cosine; the angle, reduced to a turn in 64 bits, is off by
2^-25 turns, 2^-22.3 of a full amplitude. 2^-15 of the pair's amplitude covers
them; then half a step of bf16, 2^-8 of the value. Selection: a thread sums 16
exponentials of 2^-22 + |x| 2^-23 relative error (weighted by exp(x), at most
2^-21 of the sum) a round, adds at most 8 rounds here with a factor each, and 13
more additions and 2 factors make the block's sum: the log of the sum is off by
50 * 2^-24, the score besides by 2^-24 of itself. Reordering moves bits.
"""
import math

import pytest

import uocr_moe as M

pytestmark = pytest.mark.gpu


def gen_of(*key):
    import torch
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)) + 1)


# ---- rotate_heads

def rotated(x, gain, inv_freq, positions, interleaved, eps, magnitude):
    """(values, amplitudes) in 64 bits."""
    import torch
    x = x.double()
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    rot = 2 * inv_freq.numel()
    angle = (positions.double()[:, None] * inv_freq.double())[:, None, :]
    c, s = magnitude * angle.cos(), magnitude * angle.sin()
    y, size = x.clone(), x.abs()
    at = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    size[..., at[0]] = size[..., at[1]] = abs(magnitude) * (a.abs() + b.abs())
    return y, size


def close(got, want, size):
    over = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + 2.0 ** -15 * size + 1e-38)
    assert not over.isnan().any() and (over.numel() == 0 or over.max().item() <= 0.0), over.max().item()


def run_rotate(rows, heads, kv, dim, rot, dtype="float32", norm="both", interleaved=False, far=0, caches=None,
               pad=0, magnitude=1.0, shift=0, own_places=True):
    import torch
    g = gen_of(rows, heads, kv, dim, rot)
    dt = getattr(torch, dtype)

    def make(h):  # rows of a wider buffer, `shift` elements from its start
        wide = torch.randn(rows, shift + h * dim + pad, generator=g, device="cuda").to(dt)
        return torch.as_strided(wide, (rows, h, dim), (wide.shape[1], dim, 1), shift)

    q, k, v = make(heads), make(kv), make(kv)
    caches = rows if caches is None else caches
    cap = -(-rows // caches) + 3
    order = torch.randperm(caches * cap, generator=g, device="cuda")[:rows]
    places, slots = (order // cap).to(torch.int32), (order % cap).to(torch.int32)
    positions = slots + far if own_places else slots
    inv = (1.0 / 1e4 ** (torch.arange(rot // 2, device="cuda").double() * 2 / max(rot, 1))).float()
    gains = {n: torch.rand(dim, generator=g, device="cuda") + 0.5 if norm in (n, "both") else None for n in "qk"}
    kc = torch.full((caches, kv, cap, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    vc = torch.full_like(kc, 8.0)
    out = torch.full((rows, heads * dim + pad), 9.0, dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(out, (rows, heads, dim), (out.shape[1], dim, 1))
    M.rotate_heads(q, k, v, inv, positions, view, kc, vc, q_norm=gains["q"], k_norm=gains["k"], cache_rows=places,
                   slots=slots if own_places else None, eps=1e-5, magnitude=magnitude, interleaved=interleaved)
    args = (inv, positions, interleaved, 1e-5, magnitude)
    close(view, *rotated(q, gains["q"], *args))
    assert (out[:, heads * dim:] == 9.0).all()
    at = (places.long(), slice(None), slots.long())
    close(kc[at], *rotated(k, gains["k"], *args))
    assert torch.equal(vc[at], v.to(torch.bfloat16))
    written = torch.zeros(caches, cap, dtype=torch.bool, device="cuda")
    written[places.long(), slots.long()] = True
    assert (kc.transpose(1, 2)[~written] == 7.0).all() and (vc.transpose(1, 2)[~written] == 8.0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rot", [(16, 4, 128, 128), (10, 10, 128, 64), (3, 1, 64, 64), (5, 5, 80, 32),
                                              (7, 7, 96, 96), (2, 2, 256, 256), (9, 3, 8, 8), (33, 11, 192, 72),
                                              (4, 2, 128, 0)])
def test_rotate_heads(cuda, dtype, interleaved, heads, kv, dim, rot):
    run_rotate(5, heads, kv, dim, rot, dtype, interleaved=interleaved)


@pytest.mark.parametrize("kw", [dict(rows=1), dict(rows=1000, caches=3), dict(norm="q"), dict(norm="k"), dict(norm=""),
                                dict(far=3000000), dict(far=-50000), dict(pad=5), dict(pad=8, dtype="bfloat16"),
                                dict(pad=3, shift=1, dtype="bfloat16"), dict(shift=3, pad=1), dict(magnitude=1.4),
                                dict(own_places=False, caches=1)])
def test_rotate_heads_forms(cuda, kw):
    run_rotate(**{**dict(rows=9, heads=8, kv=2, dim=128, rot=64), **kw})


def test_rotate_heads_in_place_and_without_keys(cuda):
    import torch
    g = gen_of(3)
    q = torch.randn(6, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    inv, _ = M.rope_frequencies(64)
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    none = torch.empty(6, 0, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.empty(6, 0, 8, 64, dtype=torch.bfloat16, device="cuda")
    want = rotated(q, None, inv.cuda(), pos, False, 0.0, 1.0)
    M.rotate_heads(q, none, none, inv.cuda(), pos, q, cache, cache)
    close(q, *want)


@pytest.mark.parametrize("place,slot", [(4, 0), (-1, 0), (0, 8), (0, -1)])
def test_rotate_heads_reports_places_that_do_not_exist(cuda, place, slot):
    import torch
    x = torch.ones(2, 1, 64, device="cuda")
    cache = torch.zeros(4, 1, 8, 64, dtype=torch.bfloat16, device="cuda")
    vcache, out = torch.zeros_like(cache), torch.empty(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    M.rotate_heads(x, x, x, torch.ones(32, device="cuda"), torch.zeros(2, **i32), out, cache, vcache,
                   cache_rows=torch.tensor([1, place], **i32), slots=torch.tensor([2, slot], **i32))
    with pytest.raises(M.UocrError) as e:
        M.ops_check()
    assert e.value.code == 5 and "row 1" in str(e.value)
    assert (out == 1).all() and (vcache[1, 0, 2] == 1).all() and vcache.sum() == 64
    M.ops_check()


# ---- beam_select

def selected(logits, scores, finished, eos, select):
    """[batch, select] of (value, flat index), best first, in 64 bits; and [batch, beams, vocab] values."""
    import torch
    batch, beams = scores.shape
    z = logits.double().view(batch, beams, -1)
    z = torch.where(z.isnan(), -math.inf, z)
    z = torch.log_softmax(z, -1) + scores.double()[..., None]
    z = torch.where(z.isnan(), -math.inf, z)
    if finished is not None:
        done = finished != 0
        z[done] = -math.inf
        z[..., max(eos, 0)] = torch.where(done, scores.double(), z[..., max(eos, 0)])
    value, at = z.reshape(batch, -1).sort(dim=1, descending=True, stable=True)
    pad = max(0, select - at.shape[1])
    value = torch.nn.functional.pad(value, (0, pad), value=-math.inf)
    at = torch.nn.functional.pad(at, (0, pad))
    return value[:, :select], at[:, :select], z


def check_select(logits, scores, select, finished=None, eos=-1):
    import torch
    batch, beams = scores.shape
    vocab = logits.shape[1]
    tokens = torch.full((batch, select), -7, dtype=torch.int32, device="cuda")
    parents, flags = torch.full_like(tokens, -7), torch.full_like(tokens, -7)
    new = torch.full((batch, select), math.nan, device="cuda")
    M.beam_select(logits, scores, tokens, parents, new, finished=finished, new_finished=flags, eos=eos)
    value, at, z = selected(logits, scores, finished, eos, select)
    dead = value == -math.inf
    assert torch.equal(new == -math.inf, dead)
    tol = torch.where(dead, 0.0, 50 * 2.0 ** -24 + 2.0 ** -23 * value.abs())
    assert ((new.double() - value).abs() <= tol)[~dead].all()
    tok, par = at % vocab, at // vocab
    tok[dead], par[dead] = max(eos, 0), 0
    # The same candidates in the same order, but where two beams' scores are closer than the scores' own error.
    same = (tokens == tok) & (parents == par)
    if not same.all():
        own = z[torch.arange(batch, device="cuda")[:, None], parents.long(), tokens.long()]
        assert ((own - value).abs() <= 2 * tol)[~same].all() and not (~same & dead).any()
    done = dead | (tokens == eos)
    if finished is not None:
        done |= finished.gather(1, parents.long()) != 0
    assert torch.equal(flags != 0, done)
    flat = parents.long() * vocab + tokens
    for b in range(batch):
        live = flat[b][~dead[b]]
        assert live.unique().numel() == live.numel()
    return tokens, parents, new


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch,beams,select,vocab", [
    (1, 1, 1, 1), (1, 1, 32, 40), (1, 4, 4, 102400), (3, 2, 5, 129), (2, 8, 16, 4096), (1, 32, 32, 5001), (5, 3, 7, 8192),
    (2, 5, 31, 33333), (40, 8, 8, 20001), (1, 2, 3, 1 << 20)])
def test_beam_select(cuda, dtype, batch, beams, select, vocab):
    import torch
    g = gen_of(batch, beams, select, vocab)
    logits = (torch.randn(batch * beams, vocab, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    check_select(logits, -10 * torch.rand(batch, beams, generator=g, device="cuda"), select)


def test_beam_select_ties_go_to_the_lower_beam_and_token(cuda):
    import torch
    tokens, parents, _ = check_select(torch.zeros(6, 10000, device="cuda"), torch.zeros(2, 3, device="cuda"), 32)
    assert torch.equal(tokens, torch.arange(32, dtype=torch.int32, device="cuda").expand(2, 32)) and (parents == 0).all()
    logits = torch.zeros(3, 9000, device="cuda")
    logits[:, 8000:8003] = 5.0
    tokens, parents, _ = check_select(logits, torch.zeros(1, 3, device="cuda"), 7)
    assert tokens[0].tolist() == [8000, 8001, 8002] * 2 + [8000] and parents[0].tolist() == [0] * 3 + [1] * 3 + [2]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_beam_select_takes_both_zeros_for_equal(cuda, dtype):
    import torch
    logits = torch.full((2, 9000), -5.0, device="cuda", dtype=getattr(torch, dtype))
    logits[:, 100:130], logits[:, 110:8000:7] = -0.0, 0.0
    tokens, parents, _ = check_select(logits, torch.zeros(1, 2, device="cuda"), 20)
    assert tokens[0].tolist() == list(range(100, 120)) and (parents == 0).all()
    scores = torch.tensor([[-0.0, 0.0, -0.0]], device="cuda")
    finished = torch.ones(1, 3, dtype=torch.int32, device="cuda")
    _, parents, _ = check_select(torch.zeros(3, 50, device="cuda"), scores, 3, finished, 7)
    assert parents[0].tolist() == [0, 1, 2]


@pytest.mark.parametrize("score", [-1e9, -1e30])
def test_beam_select_of_scores_that_hide_the_logits(cuda, score):
    """Within a beam the logits' order stays; equal scores of two beams go to the lower one."""
    import torch
    logits = torch.randn(3, 30000, generator=gen_of(9), device="cuda")
    logits[2] = logits[1]
    scores = torch.tensor([[score * 2, score, score]], device="cuda")
    tokens, parents, new = (torch.empty(1, 32, dtype=d, device="cuda") for d in (torch.int32, torch.int32, torch.float32))
    M.beam_select(logits, scores, tokens, parents, new)
    assert (new == score).all()
    if score == -1e30:  # all of a beam's scores are one 64-bit value
        want = logits[1].sort(descending=True, stable=True)[1][:32]
        assert (parents == 1).all() and torch.equal(tokens[0].long(), want)
    else:
        want = logits[1].sort(descending=True, stable=True)[1][:16]
        assert torch.equal(parents[0].long(), torch.tensor([1, 2] * 16, device="cuda"))
        assert torch.equal(tokens[0].long(), want.repeat_interleave(2))


@pytest.mark.parametrize("order", ["rising", "falling", "steps"])
@pytest.mark.parametrize("select", [1, 32])
def test_beam_select_of_sorted_logits(cuda, order, select):
    """Large values side by side: whole threads' and warps' worth of them above the others."""
    import torch
    x = torch.linspace(-20, 20, 70000, device="cuda")
    x = x.flip(0) if order == "falling" else torch.floor(x) if order == "steps" else x
    check_select(torch.stack([x, x.roll(777)]).contiguous(), torch.tensor([[-1.0, -1.5]], device="cuda"), select)


def test_beam_select_finished_dead_and_bad_rows(cuda):
    import torch
    g = gen_of(8)
    logits = torch.randn(12, 5000, generator=g, device="cuda")
    scores = -torch.rand(2, 6, generator=g, device="cuda") * 4
    finished = torch.zeros(2, 6, dtype=torch.int32, device="cuda")
    finished[0, 1], finished[1, 0], finished[1, 5] = 1, -3, 1
    scores[0, 2], scores[1, 3] = -math.inf, math.nan
    scores[1, 5] = -math.inf
    logits[0, 100:4000] = math.nan
    logits[3] = -math.inf
    logits[4, 77] = math.inf
    logits[6] = math.nan  # of a finished beam
    logits[11, :] = -math.inf
    for eos in (-1, 0, 4999):
        check_select(logits, scores, 8, finished, eos)
        check_select(logits, scores, 32, finished, eos)


def test_beam_select_when_candidates_run_out(cuda):
    import torch
    scores = torch.tensor([[-1.0, -math.inf, -2.0], [-math.inf] * 3], device="cuda")
    finished = torch.tensor([[1, 0, 0], [0, 1, 0]], dtype=torch.int32, device="cuda")
    logits = torch.full((6, 50), -math.inf, device="cuda")
    logits[2, 7] = 0.5
    tokens, parents, new = check_select(logits, scores, 5, finished, 3)
    assert tokens[0].tolist() == [3, 7, 3, 3, 3] and parents[0].tolist() == [0, 2, 0, 0, 0]
    assert new[0, :2].tolist() == [-1.0, -2.0] and (new[1] == -math.inf).all()


@pytest.mark.parametrize("dtype,pad,shift", [("float32", 3, 0), ("bfloat16", 5, 0), ("float32", 4, 1),
                                             ("bfloat16", 8, 1)])
def test_beam_select_of_rows_at_any_address(cuda, dtype, pad, shift):
    import torch
    wide = torch.randn(6, shift + 7001 + pad, generator=gen_of(pad, shift), device="cuda").to(getattr(torch, dtype))
    check_select(wide[:, shift:shift + 7001], torch.zeros(2, 3, device="cuda"), 6)


def test_beam_select_on_a_stream_and_from_a_graph(cuda):
    import torch
    g = gen_of(77)
    logits = torch.randn(8, 60000, generator=g, device="cuda")
    scores = -torch.rand(2, 4, generator=g, device="cuda")
    tokens = torch.empty(2, 4, dtype=torch.int32, device="cuda")
    parents, new = torch.empty_like(tokens), torch.empty(2, 4, device="cuda")
    want = check_select(logits, scores, 4)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    M.beam_select(logits, scores, tokens, parents, new, stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((tokens, parents, new), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.beam_select(logits, scores, tokens, parents, new)
    logits.copy_(torch.randn(8, 60000, generator=g, device="cuda"))
    want = check_select(logits, scores, 4)
    for _ in range(3):
        new.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((tokens, parents, new), want))


# ---- reorder_states

def reordered(state, parents, beams, counts):
    """state [layers, rows, segments, units, width]."""
    import torch
    want, units = state.clone(), state.shape[3]
    for r in range(state.shape[1]):
        p = r // beams * beams + int(parents[r])
        n = units if counts is None else int(counts[p])
        want[:, r, :, :n] = state[:, p, :, :n]
    return want


@pytest.mark.parametrize("counted", [False, True])
@pytest.mark.parametrize("layers,groups,beams,segments,units,width,dtype", [
    (1, 1, 1, 1, 5, 1, "int32"), (1, 1, 4, 1, 1000, 1, "int32"), (2, 3, 5, 2, 33, 128, "bfloat16"),
    (3, 2, 8, 4, 17, 64, "bfloat16"), (2, 2, 16, 1, 100, 3, "bfloat16"), (1, 3, 32, 2, 65, 16, "float32"),
    (2, 1, 31, 1, 77, 7, "uint8"), (1, 2, 9, 3, 13, 20, "uint8"), (4, 1, 17, 1, 1, 1, "uint8")])
def test_reorder_states(cuda, layers, groups, beams, segments, units, width, dtype, counted):
    import torch
    g = gen_of(layers, groups, beams, segments, units, width)
    rows = groups * beams
    state = torch.randint(0, 100, (layers, rows, segments, units, width), generator=g, device="cuda").to(
        getattr(torch, dtype))
    parents = torch.randint(0, beams, (rows,), generator=g, device="cuda", dtype=torch.int32)
    parents[:beams] = torch.arange(beams, device="cuda").roll(1)  # one group is a single cycle
    counts = torch.randint(0, units + 1, (rows,), generator=g, device="cuda",
                           dtype=torch.int32) if counted else None
    want = reordered(state, parents, beams, counts)
    M.reorder_states(state, parents, beams, counts=counts)
    M.ops_check()
    assert torch.equal(state, want)


def test_reorder_states_of_strided_states(cuda):
    import torch
    g = gen_of(5)
    whole = torch.randint(0, 1000, (3, 8, 2, 40, 8), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.tensor([3, 0, 0, 1], dtype=torch.int32, device="cuda")
    want = whole.clone()
    want[:, 1:5, :, 5:25] = reordered(whole[:, 1:5, :, 5:25], parents, 4, None)
    M.reorder_states(whole[:, 1:5, :, 5:25], parents, 4)
    assert torch.equal(whole, want)
    table = torch.randint(0, 1000, (8, 51), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.tensor([1, 1, 0, 3, 2, 2, 3, 0], dtype=torch.int32, device="cuda")
    counts = torch.full((8,), 30, dtype=torch.int32, device="cuda")
    want = reordered(table[None, :, None, :, None], parents, 4, counts)[0, :, 0, :, 0]
    M.reorder_states(table, parents, 4, counts=counts)
    assert torch.equal(table, want)


def test_reorder_states_reports_bad_parents_and_counts(cuda):
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    state = torch.arange(6, **i32)[:, None].expand(6, 10).contiguous()
    M.reorder_states(state, torch.tensor([1, 3, -1, 2, 0, 1], **i32), 3)
    with pytest.raises(M.UocrError) as e:
        M.ops_check()
    assert e.value.code == 5 and "parent" in str(e.value)
    assert state[:, 0].tolist() == [1, 1, 2, 5, 3, 4]
    state = torch.arange(4, **i32)[:, None].expand(4, 10).contiguous()
    M.reorder_states(state, torch.tensor([1, 0, 3, 2], **i32), 4, counts=torch.tensor([11, -1, 4, 4], **i32))
    with pytest.raises(M.UocrError) as e:
        M.ops_check()
    assert e.value.code == 5 and "units" in str(e.value)
    assert state[0].tolist() == [0] * 10 and state[1].tolist() == [0] * 10
    assert state[2].tolist() == [3] * 4 + [2] * 6


# ---- many rows

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,rot", [(16, 4, 128, 128), (10, 10, 128, 64), (3, 1, 64, 64), (5, 5, 80, 32),
                                              (2, 2, 256, 256), (9, 3, 8, 8), (4, 2, 128, 0), (30, 30, 64, 64),
                                              (28, 1, 128, 96)])
def test_rotate_heads_of_many_rows(cuda, dtype, interleaved, heads, kv, dim, rot):
    run_rotate(4001, heads, kv, dim, rot, dtype, interleaved=interleaved, caches=13)


@pytest.mark.parametrize("kw", [dict(norm="q"), dict(norm="k"), dict(norm=""), dict(far=3000000), dict(pad=8, dtype="bfloat16"),
                                dict(pad=4), dict(pad=5), dict(pad=7, shift=1, dtype="bfloat16"), dict(shift=4, pad=4),
                                dict(own_places=False, caches=1), dict(rows=2368), dict(rows=2367), dict(rows=20000, caches=5),
                                dict(norm="", magnitude=1.4, dtype="bfloat16")])
def test_rotate_heads_of_many_rows_forms(cuda, kw):
    run_rotate(**{**dict(rows=5003, heads=8, kv=2, dim=128, rot=64, caches=7), **kw})


def test_rotate_heads_of_many_rows_in_place_and_without_keys(cuda):
    import torch
    rows = 9001
    q = torch.randn(rows, 4, 64, generator=gen_of(3), device="cuda").to(torch.bfloat16)
    inv, _ = M.rope_frequencies(64)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    none = torch.empty(rows, 0, 64, dtype=torch.bfloat16, device="cuda")
    cache = torch.empty(rows, 0, 8, 64, dtype=torch.bfloat16, device="cuda")
    want = rotated(q, None, inv.cuda(), pos, False, 0.0, 1.0)
    M.rotate_heads(q, none, none, inv.cuda(), pos, q, cache, cache)
    close(q, *want)


def test_rotate_heads_of_many_rows_reports_places_that_do_not_exist(cuda):
    import torch
    rows = 6000
    x = torch.ones(rows, 1, 64, device="cuda")
    cache = torch.zeros(4, 1, 2000, 64, dtype=torch.bfloat16, device="cuda")
    vcache, out = torch.zeros_like(cache), torch.empty(rows, 1, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(rows, dtype=torch.int32, device="cuda")
    places, slots = at // 2000, at % 2000
    good = torch.ones(rows, dtype=torch.bool, device="cuda")
    for row, place, slot in ((7, 4, 0), (2500, -1, 5), (4444, 1, 2000), (5999, 3, -1)):
        places[row], slots[row], good[row] = place, slot, False
    M.rotate_heads(x, x, x, torch.ones(32, device="cuda"), torch.zeros_like(at), out, cache, vcache,
                   cache_rows=places, slots=slots)
    with pytest.raises(M.UocrError) as e:
        M.ops_check()
    assert e.value.code == 5
    want = torch.zeros(4, 2000, device="cuda")
    want[places[good].long(), slots[good].long()] = 1
    assert (out == 1).all() and torch.equal(vcache[:, 0].float(), want[..., None].expand(4, 2000, 64))
    assert torch.equal(cache, vcache)
    M.ops_check()


@pytest.mark.parametrize("rows", [5, 7000])
def test_rotate_heads_on_a_stream_and_from_a_graph(cuda, rows):
    import torch
    g = gen_of(rows, 21)
    q, k, v = (torch.randn(rows, h, 128, generator=g, device="cuda") for h in (8, 2, 2))
    inv, _ = M.rope_frequencies(128)
    inv = inv.cuda()
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    kc = torch.zeros(1, 2, 2 * rows, 128, dtype=torch.bfloat16, device="cuda")
    vc, out = torch.zeros_like(kc), torch.empty(rows, 8, 128, dtype=torch.bfloat16, device="cuda")
    places = torch.zeros_like(pos)

    def verify():
        close(out, *rotated(q, None, inv, pos, False, 1e-6, 1.0))
        close(kc[0, :, pos.long()].transpose(0, 1), *rotated(k, None, inv, pos, False, 1e-6, 1.0))
        assert torch.equal(vc[0, :, pos.long()].transpose(0, 1), v.to(torch.bfloat16))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    M.rotate_heads(q, k, v, inv, pos, out, kc, vc, cache_rows=places, stream=side)
    torch.cuda.synchronize()
    verify()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.rotate_heads(q, k, v, inv, pos, out, kc, vc, cache_rows=places)
    pos += rows // 2
    q.mul_(1.5)
    v.neg_()
    graph.replay()
    torch.cuda.synchronize()
    verify()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch,beams,select,vocab", [(4, 32, 32, 102400), (150, 3, 8, 8193), (1, 32, 32, 1 << 20),
                                                      (500, 1, 1, 4097), (64, 16, 32, 20000)])
def test_beam_select_of_large_groups(cuda, dtype, batch, beams, select, vocab):
    import torch
    g = gen_of(batch, beams, select, vocab, 3)
    logits = (torch.randn(batch * beams, vocab, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    scores = -10 * torch.rand(batch, beams, generator=g, device="cuda")
    for b in range(0, batch, 20):  # in pieces: the plain form holds several copies in 64 bits
        of = slice(b, min(b + 20, batch))
        check_select(logits[of.start * beams:of.stop * beams], scores[of].contiguous(), select)
    tokens = torch.empty(batch, select, dtype=torch.int32, device="cuda")
    parents, new = torch.empty_like(tokens), torch.empty(batch, select, device="cuda")
    M.beam_select(logits, scores, tokens, parents, new)
    for b in (0, batch // 2, batch - 1):
        one = check_select(logits[b * beams:(b + 1) * beams], scores[b:b + 1].contiguous(), select)
        # A group's parts depend on how many rows the call has, and with them a sum's last bits.
        assert (new[b] - one[2][0]).abs().max() <= 50 * 2.0 ** -23 + 2.0 ** -22 * new[b].abs().max()


def test_reorder_states_on_a_stream_and_from_a_graph(cuda):
    import torch
    g = gen_of(31)
    state = torch.randint(0, 1000, (2, 8, 2, 50, 64), generator=g, device="cuda", dtype=torch.int32)
    parents = torch.tensor([3, 0, 0, 1, 1, 2, 3, 0], dtype=torch.int32, device="cuda")
    counts = torch.tensor([50, 3, 0, 49, 20, 21, 1, 50], dtype=torch.int32, device="cuda")
    want = reordered(state, parents, 4, counts)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    M.reorder_states(state, parents, 4, counts=counts, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(state, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.reorder_states(state, parents, 4, counts=counts)
    for turn in range(3):
        parents.copy_(torch.randint(0, 4, (8,), generator=g, device="cuda"))
        counts.copy_(torch.randint(0, 51, (8,), generator=g, device="cuda"))
        want = reordered(state, parents, 4, counts)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(state, want)


# ---- logits of any magnitude

def check_any_logits(logits, scores, select):
    """check_select for logits so large that log_softmax may not form the maximum plus the sum's log in one number; a
    score that float32 holds as -inf is no candidate."""
    import torch
    batch, beams = scores.shape
    vocab = logits.shape[1]
    tokens = torch.full((batch, select), -7, dtype=torch.int32, device="cuda")
    parents, flags = torch.full_like(tokens, -7), torch.full_like(tokens, -7)
    new = torch.full((batch, select), math.nan, device="cuda")
    M.beam_select(logits, scores, tokens, parents, new, new_finished=flags)
    z = logits.double().view(batch, beams, vocab)
    z = z - z.amax(-1, keepdim=True)
    z = z - z.exp().sum(-1, keepdim=True).log() + scores.double()[..., None]
    z = torch.where(z.float() == -math.inf, -math.inf, z)
    # Within a beam the logits' order stays where scores cannot tell them apart: equal logits alone do here.
    value, at = z.reshape(batch, -1).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :select], at[:, :select]
    dead = value == -math.inf
    assert torch.equal(new == -math.inf, dead) and torch.equal(flags != 0, dead)
    tol = torch.where(dead, 0.0, 50 * 2.0 ** -24 + 2.0 ** -23 * value.abs())
    assert ((new.double() - value).abs() <= tol)[~dead].all()
    tok, par = at % vocab, at // vocab
    tok[dead], par[dead] = 0, 0
    same = (tokens == tok) & (parents == par)
    own = z[torch.arange(batch, device="cuda")[:, None], parents.long(), tokens.long()]
    assert ((own - value).abs() <= 2 * tol)[~same].all() and not (~same & dead).any()
    flat = parents.long() * vocab + tokens
    for b in range(batch):
        live = flat[b][~dead[b]]
        assert live.unique().numel() == live.numel()


MASKS = [-1e10, -1e20, -1e30, "lowest"]


def mask_of(mask, dtype):
    import torch
    return torch.finfo(dtype).min if mask == "lowest" else mask


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("where", ["threads", "warps", "rounds", "tail", "head", "all but a few", "all but one", "all"])
@pytest.mark.parametrize("vocab", [20001, 102400])
def test_beam_select_of_masked_logits(cuda, dtype, mask, where, vocab):
    """Tokens masked by a large finite value: over whole threads, warps, rounds and parts of a row."""
    import torch
    dt = getattr(torch, dtype)
    logits = (torch.randn(6, vocab, generator=gen_of(vocab, len(where)), device="cuda") * 3).to(dt)
    at = torch.arange(vocab, device="cuda")
    side = 16 // logits.element_size()  # elements of a thread side by side
    thread = at // side % 256
    masked = {"threads": thread % 3 == 1, "warps": thread // 32 % 2 == 0, "rounds": at // 4096 % 2 == 0,
              "tail": at >= vocab - 9001, "head": at < vocab - 100, "all but a few": at % (vocab // 90) != 5,
              "all but one": at != 777, "all": at >= 0}[where]
    logits[:, masked] = mask_of(mask, dt)
    logits[4] = (torch.randn(vocab, generator=gen_of(vocab), device="cuda") * 3).to(dt)  # a row without a mask
    scores = -torch.rand(2, 3, generator=gen_of(5), device="cuda")
    check_any_logits(logits, scores, 8)
    check_any_logits(logits, scores, 32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("level", [3e38, 1e30, 1e10, 2.0 ** 33, -2.0 ** 33, -1e20, -3e38])
def test_beam_select_of_large_logits(cuda, dtype, level):
    """Rows about one large value, and rows with one such value above or below ordinary ones."""
    import torch
    dt = getattr(torch, dtype)
    g = gen_of(11)
    logits = torch.randn(6, 9001, generator=g, device="cuda") * 3
    logits[:2] = level * (1 + torch.randint(0, 3, (2, 9001), generator=g, device="cuda") * 2.0 ** -6)
    logits[2:4, 4321] = level
    logits[4, 100:8000] = level
    logits[5, ::2], logits[5, 1::2] = level, torch.finfo(dt).min
    check_any_logits(logits.to(dt), -torch.rand(2, 3, generator=g, device="cuda"), 8)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_beam_select_takes_a_score_that_rounds_to_minus_infinity_for_none(cuda, dtype):
    import torch
    dt = getattr(torch, dtype)
    logits = torch.full((1, 5000), torch.finfo(dt).min, device="cuda", dtype=dt)
    logits[0, 70] = 3e38
    check_any_logits(logits, torch.zeros(1, 1, device="cuda"), 3)
    tokens, parents, flags = (torch.empty(1, 3, dtype=torch.int32, device="cuda") for _ in range(3))
    new = torch.empty(1, 3, device="cuda")
    M.beam_select(logits, torch.zeros(1, 1, device="cuda"), tokens, parents, new, new_finished=flags, eos=9)
    assert tokens[0].tolist() == [70, 9, 9] and new[0].tolist() == [0.0, -math.inf, -math.inf] and flags[0].tolist() == [0, 1, 1]
