"""The grouped W8A8 product with a row index on a stream that is not torch's
current one: its workspace belongs to the stream that uses it, and calls on two
streams that share no tensor do not disturb each other."""
import pytest

import uocr_moe as M
from test_int8_gpu import check, gen_of, ints, scales

pytestmark = pytest.mark.gpu

ROWS, TOKENS, GROUPS, N, K = 16384, 512, 8, 96, 1024
WORKSPACE = ROWS * K


def inputs(seed):
    import torch
    g = gen_of(seed)
    at = torch.linspace(0, ROWS, GROUPS + 1).to(torch.int32).cuda()
    return dict(x=ints(g, TOKENS, K), x_scales=scales(g, TOKENS), w=ints(g, GROUPS * N, K),
                w_scales=scales(g, GROUPS * N), offsets=at, y=torch.full((ROWS, N), 55.0, device="cuda"),
                row_index=torch.randint(0, TOKENS, (ROWS,), generator=g, device="cuda", dtype=torch.int32))


def check_outputs(a):
    at = a["offsets"].tolist()
    for e in range(GROUPS):
        lo, hi, part = at[e], at[e + 1], slice(e * N, (e + 1) * N)
        src = a["row_index"][lo:hi].long()
        want = (a["x"][src].double() @ a["w"][part].double().T) * a["x_scales"][src].double()[:, None]
        want = want * a["w_scales"][part].double()
        check(a["y"][lo:hi], want, want.abs(), False)


@pytest.mark.parametrize("handle", [False, True])
def test_workspace_is_the_stream_s_own(cuda, handle):
    """Blocks of another stream's pool may still be in use there when the allocator hands them out."""
    import torch
    a = inputs(1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

    def held():
        return sum(s["total_size"] for s in torch.cuda.memory_snapshot() if s["stream"] == side.cuda_stream)
    before = held()
    M.grouped_linear_w8a8(**a, stream=side.cuda_stream if handle else side)
    assert held() >= before + WORKSPACE
    torch.cuda.synchronize()
    check_outputs(a)


def test_calls_on_two_streams(cuda):
    import torch
    a, b = inputs(2), inputs(3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(8):
        M.grouped_linear_w8a8(**a)
        M.grouped_linear_w8a8(**b, stream=side)
    torch.cuda.synchronize()
    check_outputs(a)
    check_outputs(b)


def test_captured_with_the_stream_given(cuda):
    import torch
    a = inputs(4)
    M.grouped_linear_w8a8(**a)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        M.grouped_linear_w8a8(**a, stream=side)
    a["y"].fill_(55.0)
    graph.replay()
    torch.cuda.synchronize()
    check_outputs(a)
