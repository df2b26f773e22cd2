"""Operands written by the launch right in front of a product, which may start
before that launch has ended: the product sees the new values. The same operands
multiplied after a synchronisation give the bits to compare with."""
import pytest

import uocr_moe as M
from test_int8_gpu import gen_of, pitch16

pytestmark = pytest.mark.gpu


def rows8(rows, k):
    import torch
    return torch.zeros(rows, pitch16(k), dtype=torch.int8, device="cuda")[:, :k], torch.zeros(rows, device="cuda")


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (6, 2048, 256), (24, 600, 2000), (60, 300, 4000), (500, 1024, 256),
                                   (3000, 512, 64)])
@pytest.mark.parametrize("last", ["x", "w"])
def test_linear_after_its_operands(cuda, m, n, k, last):
    import torch
    g = gen_of(m, n, k)
    (xq, xs), (wq, ws) = rows8(m, k), rows8(n, k)
    for _ in range(5):
        x, w = (torch.randn(r, k, generator=g, device="cuda") for r in (m, n))
        y, want = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        torch.cuda.synchronize()
        for name in ("w", "x") if last == "x" else ("x", "w"):
            M.quantize_tokens(*((x, xq, xs) if name == "x" else (w, wq, ws)))
        M.linear_w8a8(xq, xs, wq, ws, y)
        torch.cuda.synchronize()
        M.linear_w8a8(xq, xs, wq, ws, want)
        assert torch.equal(y, want)


@pytest.mark.parametrize("rows", [20, 700])
@pytest.mark.parametrize("last", ["x", "w", "up"])
def test_grouped_after_its_operands(cuda, rows, last):
    import torch
    groups, n, k = 8, 200, 320
    g = gen_of(rows, groups)
    parts = {name: rows8(rows if name == "x" else groups * n, k) for name in ("x", "w", "up")}
    offsets = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
    index = torch.empty(rows, dtype=torch.int32, device="cuda")
    for _ in range(5):
        src = {name: torch.randn(p[0].shape, generator=g, device="cuda") for name, p in parts.items()}
        at = torch.randint(0, rows + 1, (groups + 1,), generator=g, device="cuda").sort().values.int()
        at[0], at[-1] = 0, rows
        perm = torch.randperm(rows, generator=g, device="cuda").int()
        y, want = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
        torch.cuda.synchronize()
        offsets.copy_(at)
        index.copy_(perm)
        for name in sorted(parts, key=lambda name: name == last):
            M.quantize_tokens(src[name], *parts[name])

        def product(out):
            M.grouped_linear_w8a8(*parts["x"], *parts["w"], offsets, out, row_index=index, w_up=parts["up"][0],
                                  w_up_scales=parts["up"][1])
        product(y)
        torch.cuda.synchronize()
        product(want)
        assert torch.equal(y, want)
    M.ops_check()
