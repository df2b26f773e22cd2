"""The W8A8 products where a pair of SMs works through several tiles: what a
tile leaves behind for the next one (staging buffers, accumulators, residual
slots, the tiles worked out ahead). Sizes are chosen for 74 pairs, one wave of
which is 74 tiles of 256 (gated: 128) channels by up to 256 tokens; K is short,
so that a tile's stores are still under way when the next tile is ready.

Against the plain 64-bit form with test_int8_gpu's tolerances, and repeated
calls against each other bit for bit."""
import numpy as np
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
