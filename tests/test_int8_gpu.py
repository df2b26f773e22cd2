"""The 8-bit integer operators on the GPU against plain 64-bit forms.

Tolerances. The products' int32 sums are exact; what remains is the epilogue
in fp32: the sum to float and two scales (3 roundings, each at most 2^-24 of
the value), then one rounding for each term added, at most 2^-24 of the sum of
the magnitudes: 6 * 2^-24 of (|product| + |bias| + |residual|) covers them.
bf16 outputs add half a unit in the last of 8 bits, 2^-9 of the value (taken as
2^-8). The gated form multiplies two such values by g's logistic: relative
2^-24 * (20 + 4 |g|), since d log(silu)/dg <= 1 + 1/|g| turns g's own relative
error into at most (1 + |g|) times it, plus 1e-36 where exp(-g) overflows. The
quantiser is compared for equality with the same IEEE operations on the CPU.
"""
import numpy as np
import pytest

import uocr_moe as M

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def padded(t, pitch):
    """t [rows, cols] inside rows of `pitch` elements, the rest filled with a value that would show."""
    import torch
    wide = torch.full((t.shape[0], pitch), 77, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def pitch16(k, extra=0):
    return (k + 15) // 16 * 16 + extra


def ints(gen, rows, cols, extra=0):
    import torch
    q = torch.randint(-128, 128, (rows, cols), generator=gen, device="cuda", dtype=torch.int8)
    return padded(q, pitch16(cols, extra))


def scales(gen, n):
    import torch
    return torch.rand(n, generator=gen, device="cuda") * 0.01 + 1e-3


def gen_of(*key):
    import torch
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def check(y, want, size, bf16, g=None):
    y, want = y.double(), want.double()
    tol = 6 * EPS * size if g is None else EPS * (20 + 4 * g.abs()) * size + 1e-36
    if bf16:
        tol = tol + 2.0 ** -8 * want.abs()
    over = (y - want).abs() - tol
    assert not over.isnan().any() and over.max().item() <= 0.0, f"{over.max().item():.3e} above the tolerance"


# ---- quantize_tokens

def quantized(x):
    """The rule in numpy's IEEE fp32: (q, scales)."""
    x = np.asarray(x, dtype=np.float32)
    q, s = np.zeros(x.shape, np.int8), np.ones(x.shape[0], np.float32)
    for r, row in enumerate(x):
        if not np.isfinite(row).all():
            s[r] = np.nan
            continue
        peak = np.abs(row).max() if row.size else np.float32(0)
        if peak > 0:
            s[r] = max(np.float32(peak) * (np.float32(1) / np.float32(127)), np.finfo(np.float32).tiny)
        q[r] = np.clip(np.rint(row / s[r]), -127, 127)
    return q, s


def run_quantize(x, extra=0):
    import torch
    rows, cols = x.shape
    q = torch.full((rows, pitch16(cols, extra)), 99, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), -1.0, device="cuda")
    M.quantize_tokens(x, q[:, :cols], s)
    return q, s


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,cols,pad,shift", [
    (1, 1, 0, 0), (1, 2048, 0, 0), (3, 7, 0, 0), (9, 8, 8, 0), (33, 63, 1, 0), (17, 2047, 3, 1), (300, 1024, 64, 0),
    (5, 2049, 0, 0), (4, 16384, 0, 0), (2, 16391, 9, 0), (3, 40000, 0, 1)])
def test_quantize_tokens(cuda, dtype, rows, cols, pad, shift):
    import torch
    g = gen_of(rows, cols)
    wide = torch.randn(rows, cols + pad + shift, generator=g, device="cuda") * torch.exp(
        torch.randn(rows, 1, generator=g, device="cuda") * 4)
    x = wide.to(getattr(torch, dtype))[:, shift:shift + cols]  # shift: rows that do not start at 16 bytes
    q, s = run_quantize(x, 16)
    want_q, want_s = quantized(x.float().cpu().numpy())
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q[:, :cols].cpu().numpy(), want_q)
    assert (q[:, cols:] == 99).all()


@pytest.mark.parametrize("cols", [100, 4096, 20000])
def test_quantize_tokens_odd_rows(cuda, cols):
    import torch
    x = torch.randn(10, cols, generator=gen_of(cols), device="cuda")
    x[0] = 0.0
    x[1, cols // 2] = float("inf")
    x[2, cols - 1] = float("nan")
    x[3] *= 1e-44                       # subnormal
    x[4, 0] = 3.4028234e38              # the largest float
    x[5] = -x[5].abs()
    x[6] = 0.0
    x[6, cols - 1] = -1e-30
    x[7] = -float("inf")
    x[8] = torch.arange(cols, device="cuda") % 255 - 127.0  # ties of peak 127 * 0.5 among them
    x[8] *= 0.5
    q, s = run_quantize(x)
    want_q, want_s = quantized(x.cpu().numpy())
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q[:, :cols].cpu().numpy(), want_q)


def test_quantize_tokens_agrees_with_quantize_q8(cuda):
    import torch
    x = torch.randn(64, 2048, generator=gen_of(5), device="cuda").to(torch.bfloat16)
    q, s = run_quantize(x)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    M.quantize_q8(x, q2, s2)
    # s: a product here and a quotient there, one bit apart at most; then q differs by a tie's side at most
    assert ((s - s2).abs() <= s * 2.0 ** -23).all() and (q.int() - q2.int()).abs().max() <= 1


# ---- linear_w8a8

def linear_case(m, n, k, bf16, bias, residual, extra=0):
    import torch
    g = gen_of(m, n, k)
    dt = torch.bfloat16 if bf16 else torch.float32
    x, w = ints(g, m, k, extra), ints(g, n, k, 0)
    xs, ws = scales(g, m), scales(g, n)
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    r = padded(torch.randn(m, n, generator=g, device="cuda").to(dt), n + extra) if residual else None
    y = torch.full((m, n + extra), 55.0, dtype=dt, device="cuda")
    M.linear_w8a8(x, xs, w, ws, y[:, :n], bias=b, residual=r)
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    size = want.abs()
    if bias:
        want, size = want + b.double(), size + b.double().abs()
    if residual:
        want, size = want + r.double(), size + r.double().abs()
    check(y[:, :n], want, size, bf16)
    assert (y[:, n:] == 55.0).all()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("n,k,bf16,bias,residual,extra", [
    (256, 512, False, False, False, 0), (203, 529, True, True, False, 16), (1031, 1000, False, True, True, 1 * 16),
    (512, 2048, True, False, True, 0)])
def test_linear_w8a8(cuda, m, n, k, bf16, bias, residual, extra):
    linear_case(m, n, k, bf16, bias, residual, extra)


@pytest.mark.parametrize("m", [1, 13, 40, 200])
@pytest.mark.parametrize("n,k", [(1, 64), (2, 1), (15, 15), (16, 16), (17, 17), (255, 127), (257, 128), (64, 129),
                                 (31, 4113), (5000, 64)])
def test_linear_w8a8_edges(cuda, m, n, k):
    linear_case(m, n, k, False, False, False)
    linear_case(m, n, k, True, True, True, 16)


@pytest.mark.parametrize("m,n,k", [(1, 102400, 256), (1024, 2048, 2048), (2500, 1024, 640), (700, 4100, 300)])
def test_linear_w8a8_large(cuda, m, n, k):
    linear_case(m, n, k, True, True, False)


@pytest.mark.parametrize("m", [33, 64, 100, 129, 300, 500, 1000])
@pytest.mark.parametrize("n,k", [(70, 8000), (300, 2049), (1030, 4113), (2048, 4096), (4100, 5000)])
def test_linear_w8a8_long_k_of_few_tiles(cuda, m, n, k):
    linear_case(m, n, k, False, True, True, 16)
    linear_case(m, n, k, True, False, m % 2 == 0)


@pytest.mark.parametrize("m,bf16", [(40, False), (40, True), (500, False), (700, True)])
def test_linear_w8a8_long_k_is_repeatable(cuda, m, bf16):
    import torch
    g = gen_of(m, bf16)
    n, k = 600, 6000
    x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
    b = torch.randn(n, generator=g, device="cuda")
    y = [torch.empty(m, n, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda") for _ in range(20)]
    for out in y:
        M.linear_w8a8(x, xs, w, ws, out, bias=b)
    # The sums are exact and the rest is rounded alike: rows taken alone are the same bits.
    few = torch.empty_like(y[0][:5])
    M.linear_w8a8(x[:5], xs[:5], w, ws, few, bias=b)
    assert torch.equal(few, y[0][:5])
    for out in y[1:]:
        assert torch.equal(out, y[0])


@pytest.mark.parametrize("m", [1, 20, 150])
def test_linear_w8a8_longest_sums(cuda, m):
    """Rows of the largest width and magnitude: the sums come within 2^14 of 2^31."""
    import torch
    k, n = 131071, 40
    x = padded(torch.full((m, k), -128, dtype=torch.int8, device="cuda"), pitch16(k))
    w = padded(torch.full((n, k), -128, dtype=torch.int8, device="cuda"), pitch16(k))
    w[1::2] = 127
    y = torch.empty(m, n, device="cuda")
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    M.linear_w8a8(x, one_m, w, one_n, y)
    want = x.double() @ w.double().T
    check(y, want, want.abs(), False)


@pytest.mark.parametrize("m", [1, 12, 77])
def test_linear_w8a8_residual_in_place_and_repeatable(cuda, m):
    import torch
    g = gen_of(m)
    n, k = 320, 768
    x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
    h = torch.randn(m, n, generator=g, device="cuda")
    apart = torch.empty_like(h)
    M.linear_w8a8(x, xs, w, ws, apart, residual=h)
    again = torch.empty_like(h)
    M.linear_w8a8(x, xs, w, ws, again, residual=h)
    M.linear_w8a8(x, xs, w, ws, h, residual=h)
    assert torch.equal(apart, h) and torch.equal(apart, again)


@pytest.mark.parametrize("m", [3, 100])
def test_linear_w8a8_scales_carry_nan_and_inf(cuda, m):
    import torch
    g = gen_of(m)
    x, w, xs, ws = ints(g, m, 64), ints(g, 48, 64), scales(g, m), scales(g, 48)
    x[0] = 0
    xs[0], xs[1], ws[5] = float("nan"), 0.0, float("inf")
    y = torch.empty(m, 48, device="cuda")
    M.linear_w8a8(x, xs, w, ws, y)
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    assert y[0].isnan().all()
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())


@pytest.mark.parametrize("m", [3, 70])
def test_linear_w8a8_distances_past_32_bits(cuda, m):
    """Rows further apart than 2^31 elements and bytes, in x, the residual and y."""
    import torch
    g = gen_of(9)
    n, k = 24, 48
    far = (1 << 31) // (m - 1) // 16 * 16 + 64
    x = torch.empty(far * (m - 1) + k, dtype=torch.int8, device="cuda").as_strided((m, k), (far, 1))
    x.copy_(torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8))
    buf = torch.empty(far * (m - 1) + n, dtype=torch.bfloat16, device="cuda")
    y = buf.as_strided((m, n), (far, 1))
    y.copy_(torch.randn(m, n, generator=g, device="cuda"))
    r = y.double()
    w, xs, ws = ints(g, n, k), scales(g, m), scales(g, n)
    M.linear_w8a8(x, xs, w, ws, y, residual=y)
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    check(y, want + r, want.abs() + r.abs(), True)


@pytest.mark.parametrize("m", [1, 64, 400])
def test_linear_w8a8_on_another_stream_and_in_a_graph(cuda, m):
    import torch
    g = gen_of(m)
    n, k = 640, 1024
    x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
    y = torch.zeros(m, n, device="cuda")
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    M.linear_w8a8(x, xs, w, ws, y, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check(y, want, want.abs(), False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        M.linear_w8a8(x, xs, w, ws, y)
    x.copy_(torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8))
    graph.replay()
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    check(y, want, want.abs(), False)


# ---- grouped_linear_w8a8

def grouped_case(counts, n, k, bf16=True, gated=False, gather=False, first=0, after=0, tokens=None, extra=0):
    import torch
    g = gen_of(sum(counts), n, k, len(counts))
    dt = torch.bfloat16 if bf16 else torch.float32
    groups, used = len(counts), sum(counts)
    rows = first + used + after
    offsets = torch.tensor(np.cumsum([first] + list(counts)), dtype=torch.int32, device="cuda")
    x_rows = (tokens or max(1, rows // 2)) if gather else rows
    x, xs = ints(g, x_rows, k, extra), scales(g, x_rows)
    idx = torch.randint(0, x_rows, (rows,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    w, ws = ints(g, groups * n, k), scales(g, groups * n)
    u, us = (ints(g, groups * n, k), scales(g, groups * n)) if gated else (None, None)
    y = torch.full((rows, n + extra), 55.0, dtype=dt, device="cuda")
    if gated:  # gates of the size a network has, some far out
        ws *= 0.3
    M.grouped_linear_w8a8(x, xs, w, ws, offsets, y[:, :n], row_index=idx, w_up=u, w_up_scales=us)
    M.ops_check()
    at = np.cumsum([first] + list(counts))
    for e in range(groups):
        lo, hi = int(at[e]), int(at[e + 1])
        src = torch.arange(lo, hi, device="cuda") if idx is None else idx[lo:hi].long()
        part = slice(e * n, (e + 1) * n)
        p = (x[src].double() @ w[part].double().T) * xs[src].double()[:, None] * ws[part].double()
        if gated:
            up = (x[src].double() @ u[part].double().T) * xs[src].double()[:, None] * us[part].double()
            want = p * torch.sigmoid(p) * up
            if hi > lo:
                check(y[lo:hi, :n], want, want.abs(), bf16, g=p)
        elif hi > lo:
            check(y[lo:hi, :n], p, p.abs(), bf16)
    assert (y[:first] == 55.0).all() and (y[first + used:] == 55.0).all() and (y[:, n:] == 55.0).all()


RAGGED = [
    [1], [0, 1, 0], [6], [1, 1, 1, 1, 1, 1], [0, 0, 9, 0, 17, 1, 0], [8, 9, 16, 17, 33], [64, 1, 0, 65, 128, 129, 0],
    [0] * 40 + [3] + [0] * 23, [2] * 128, [300, 0, 5, 700], [1] * 3 + [0] * 500 + [2] * 9]


@pytest.mark.parametrize("counts", RAGGED, ids=lambda c: f"{len(c)}groups_{sum(c)}rows")
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_ragged(cuda, counts, gated, gather):
    n, k = (96, 160) if len(counts) < 100 else (48, 64)
    grouped_case(counts, n, k, True, gated, gather)
    grouped_case(counts, n + 7, k + 9, False, gated, gather, first=3, after=5, extra=16)


@pytest.mark.parametrize("gated,gather", [(True, True), (False, False)])
@pytest.mark.parametrize("counts", [[1, 0, 1, 1, 0, 1, 1, 1], [40, 2, 0, 130], [1000, 0, 1, 500]])
def test_grouped_model_sizes(cuda, counts, gated, gather):
    grouped_case(counts, 1024, 2048, True, gated, gather)
    grouped_case(counts, 2048, 1024, False, gated, gather)


@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_gather_of_few_tokens(cuda, tokens, gated):
    grouped_case([tokens, 0, tokens * 30, 1, 7], 200, 272, True, gated, True, tokens=tokens)


@pytest.mark.parametrize("scale", [1.0, 300])
def test_grouped_bad_offsets_are_reported_and_skipped(cuda, scale):
    import torch
    g = gen_of(3)
    base = int(8 * scale)
    rows, n, k = base, 64, 64
    x, xs, w, ws = ints(g, rows, k), scales(g, rows), ints(g, 4 * n, k), scales(g, 4 * n)
    for bad, good in (([0, 2, rows + 1, rows, rows], 0), ([0, rows, rows - 2, rows - 2, rows - 2], 0),
                      ([-1, 0, rows, rows, rows], 1)):
        y = torch.full((rows, n), 55.0, device="cuda")
        M.grouped_linear_w8a8(x, xs, w, ws, torch.tensor(bad, dtype=torch.int32, device="cuda"), y)
        with pytest.raises(M.UocrError) as e:
            M.ops_check()
        assert e.value.code == 5 and "group" in str(e.value)
        lo, hi = bad[good], bad[good + 1]
        part = slice(good * n, (good + 1) * n)
        want = (x[lo:hi].double() @ w[part].double().T) * xs[lo:hi].double()[:, None] * ws[part].double()
        check(y[lo:hi], want, want.abs(), False)
        assert (y[hi:] == 55.0).all()
    M.ops_check()


@pytest.mark.parametrize("rows", [12, 900])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_bad_row_index_is_reported_and_zero(cuda, rows, gated):
    import torch
    g = gen_of(4)
    n, k = 64, 64
    x, xs, w, ws = ints(g, 10, k), scales(g, 10), ints(g, 2 * n, k), scales(g, 2 * n)
    u, us = (w, ws) if gated else (None, None)
    idx = torch.randint(0, 10, (rows,), generator=g, device="cuda", dtype=torch.int32)
    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    want = torch.empty(rows, n, device="cuda")
    M.grouped_linear_w8a8(x, xs, w, ws, offsets, want, row_index=idx, w_up=u, w_up_scales=us)
    M.ops_check()
    for value in (-1, 10, 2 ** 31 - 1, -2 ** 31):
        broken = idx.clone()
        broken[rows // 2 + 1] = value
        y = torch.full((rows, n), 55.0, device="cuda")
        M.grouped_linear_w8a8(x, xs, w, ws, offsets, y, row_index=broken, w_up=u, w_up_scales=us)
        with pytest.raises(M.UocrError) as e:
            M.ops_check()
        assert e.value.code == 5 and "row" in str(e.value)
        assert (y[rows // 2 + 1] == 0).all()
        keep = torch.arange(rows, device="cuda") != rows // 2 + 1
        assert torch.equal(y[keep], want[keep])


def test_grouped_one_group_is_the_linear_product(cuda):
    import torch
    for m in (1, 30, 260):
        g = gen_of(m)
        n, k = 130, 400
        x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
        a, b = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        M.linear_w8a8(x, xs, w, ws, a)
        M.grouped_linear_w8a8(x, xs, w, ws, torch.tensor([0, m], dtype=torch.int32, device="cuda"), b)
        assert torch.equal(a, b)


def test_binding_refuses_wrong_shapes(cuda):
    import torch
    g = gen_of(1)
    x, w, xs, ws = ints(g, 4, 32), ints(g, 6, 32), scales(g, 4), scales(g, 6)
    y = torch.empty(4, 6, device="cuda")
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    for call in (lambda: M.linear_w8a8(x, xs, w, ws, torch.empty(4, 5, device="cuda")),
                 lambda: M.linear_w8a8(x, ws, w, ws, y),
                 lambda: M.linear_w8a8(x, xs, ints(g, 6, 16), ws, y),
                 lambda: M.linear_w8a8(x, xs, w, ws, y.T.contiguous().T),
                 lambda: M.linear_w8a8(x, xs, w, ws, y, residual=y.bfloat16()),
                 lambda: M.linear_w8a8(x, xs, w, ws, y.half()),
                 lambda: M.grouped_linear_w8a8(x, xs, w, ws, off.long(), y),
                 lambda: M.grouped_linear_w8a8(x, xs, w, ws, off, y, row_index=off),
                 lambda: M.grouped_linear_w8a8(x, xs, w[:5], ws, off, y),
                 lambda: M.quantize_tokens(x.float(), x, ws)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("rows,n,k", [(1, 1, 5), (1, 33, 40), (4, 1, 16), (3, 2, 1), (300, 1, 33)])
def test_lone_rows_and_columns(cuda, rows, n, k):
    """Single rows and columns, whose strides say nothing: plain, and grouped in either layout of the weights."""
    import torch
    g = gen_of(rows, n, k)
    x, w, xs, ws = ints(g, rows, k), ints(g, n, k), scales(g, rows), scales(g, n)
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    y = torch.empty(rows, n, device="cuda")
    M.linear_w8a8(x, xs, w, ws, y)
    check(y, want, want.abs(), False)
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    for stack in (w, torch.as_strided(w, (1, n, k), (n * w.stride(0), w.stride(0), 1))):
        z = torch.empty(rows, n, device="cuda")
        M.grouped_linear_w8a8(x, xs, stack, ws, off, z)
        assert torch.equal(y, z)
    two = ints(g, 2 * n, k)
    off = torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda")
    z = torch.empty(rows, n, device="cuda")
    M.grouped_linear_w8a8(x, xs, torch.as_strided(two, (2, n, k), (n * two.stride(0), two.stride(0), 1)),
                          scales(g, 2 * n), off, z)
    M.ops_check()
