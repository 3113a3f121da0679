"""The status watch must not disturb a stream capture that starts while one of its checks is pending."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_capture_while_a_status_check_is_pending():
    from tmq_b200 import ops
    x = torch.randint(-127, 128, (4, 128), dtype=torch.int8, device="cuda")
    w = torch.randint(-1, 2, (64, 128), dtype=torch.int8, device="cuda")
    wt = ops.prepack(ops.compactify_ternary(w), 64, ops.FMT_I8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.ternary_gemm_i8(x, wt, 64)
        watch = ops._watch[x.device.index]
        while not watch.pending:                  # at most one round of launches
            ops.ternary_gemm_i8(x, wt, 64)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = ops.ternary_gemm_i8(x, wt, 64)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y.cpu().long(), x.cpu().long() @ w.cpu().long().t())
    ops.check_gemm_status()
