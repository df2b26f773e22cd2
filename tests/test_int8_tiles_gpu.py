"""The W8A8 products where a pair of SMs works through several tiles: what a
tile leaves behind for the next one (staging buffers, accumulators, residual
slots, the tiles worked out ahead). Sizes are chosen for 74 pairs, one wave of
which is 74 tiles of 256 (gated: 128) channels by up to 256 tokens; K is short,
so that a tile's stores are still under way when the next tile is ready.

Against the plain 64-bit form with test_int8_gpu's tolerances, and repeated
calls against each other bit for bit."""
import pytest

import uocr_moe as M
from test_int8_gpu import check, gen_of, grouped_case, ints, scales

pytestmark = pytest.mark.gpu


def dense(m, n, k, dtype, bias=False, residual=False, repeats=6):
    import torch
    g = gen_of(m, n, k)
    x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    r = torch.randn(m, n, generator=g, device="cuda").to(dtype) if residual else None
    ys = [torch.full((m, n), 55.0, dtype=dtype, device="cuda") for _ in range(repeats)]
    for y in ys:  # one after another: a call's first tiles follow the last ones of the call before
        M.linear_w8a8(x, xs, w, ws, y, bias=b, residual=r)
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    size = want.abs()
    for term in (b, r):
        if term is not None:
            want, size = want + term.double(), size + term.double().abs()
    check(ys[0], want, size, dtype is torch.bfloat16)
    for y in ys[1:]:
        assert torch.equal(y, ys[0])


# 161 tiles whose last units are partial, in the one half of the epilogue's warps (80 rows: 16 left over for the first
# half; 100: 4 for the second; 129: 1) or none (64, 256).
@pytest.mark.parametrize("m", [64, 80, 100, 129, 161, 256])
@pytest.mark.parametrize("n", [160 * 256 + 8, 160 * 256 + 3])
def test_dense_bf16_of_many_ragged_tiles(cuda, m, n):
    import torch
    dense(m, n, 64, torch.bfloat16)


def test_dense_bf16_residual_of_many_ragged_tiles(cuda):
    import torch
    dense(100, 160 * 256 + 8, 64, torch.bfloat16, bias=True, residual=True)


RAGGED = {
    "80_each": [80] * 64,
    "33_to_127": [33 + (37 * i) % 95 for i in range(64)],
    "some_empty": [0 if i % 5 == 3 else 1 + (53 * i) % 300 for i in range(48)],
}


@pytest.mark.parametrize("counts", list(RAGGED))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_bf16_of_many_ragged_tiles(cuda, counts, gated, gather):
    grouped_case(RAGGED[counts], 1032 if gated else 2056, 64, True, gated, gather)


# fp32 tiles: residual slots that go from one tile to the next (rows at 16 bytes: by TMA, two units ahead), or none.
@pytest.mark.parametrize("m", [33, 64, 100, 129, 300])
@pytest.mark.parametrize("n", [160 * 256 + 8, 160 * 256 + 3])
@pytest.mark.parametrize("residual", [False, True])
def test_dense_fp32_of_many_ragged_tiles(cuda, m, n, residual):
    import torch
    dense(m, n, 64, torch.float32, bias=n % 2 == 1, residual=residual)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_dense_residual_in_place_of_many_ragged_tiles(cuda, dtype):
    import torch
    m, n, k = 100, 160 * 256 + 8, 64
    g = gen_of(m, n)
    x, w, xs, ws = ints(g, m, k), ints(g, n, k), scales(g, m), scales(g, n)
    h = torch.randn(m, n, generator=g, device="cuda").to(getattr(torch, dtype))
    apart = torch.empty_like(h)
    M.linear_w8a8(x, xs, w, ws, apart, residual=h)
    M.linear_w8a8(x, xs, w, ws, h, residual=h)
    assert torch.equal(apart, h)


# More than 32 tiles a pair: the tiles are worked out 32 at a time, here in a second batch too.
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_dense_of_more_tiles_than_a_batch(cuda, dtype):
    import torch
    dense(70, 2500 * 256 + 8, 32, getattr(torch, dtype), residual=True, repeats=2)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_grouped_of_more_tiles_than_a_batch(cuda, bf16, gated):
    counts = [0 if i % 50 == 7 else 5 + (11 * i) % 40 for i in range(300)]
    grouped_case(counts, 1160 if gated else 2312, 64, bf16, gated, gated)


@pytest.mark.parametrize("bf16", [False, True])
def test_grouped_tiles_of_unaligned_rows(cuda, bf16):
    grouped_case(RAGGED["33_to_127"], 1031, 65, bf16, True, True, first=2, after=3)
    grouped_case(RAGGED["33_to_127"], 2051, 65, bf16, False, True, first=2, after=3)
