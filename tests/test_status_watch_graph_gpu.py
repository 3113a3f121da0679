"""The status watch beside stream captures and on a device with a failure: what is due while a graph is captured is done by the
next call outside it, and a failure is raised by the first call behind its copy."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def product():
    from tmq_b200 import ops
    x = torch.randint(-127, 128, (4, 128), dtype=torch.int8, device="cuda")
    w = torch.randint(-1, 2, (64, 128), dtype=torch.int8, device="cuda")
    wt = ops.prepack(ops.compactify_ternary(w), 64, ops.FMT_I8)
    call = lambda: ops.ternary_gemm_a8(x, wt, 64, out_dtype=torch.float32)
    call()
    torch.cuda.synchronize()
    yield call, ops._watch[x.device.index], x.cpu().double() @ w.cpu().double().t()
    ops.check_gemm_status()


@pytest.mark.parametrize("pending", [False, True])
def test_a_captured_launch_on_which_a_copy_falls_due(product, pending):
    call, watch, want = product
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        watch.due = watch.launches + 1
        if pending:
            call()
            assert watch.pending
            side.synchronize()                                 # landed, not yet looked at
            watch.due = watch.launches + 1
        else:
            watch.pending = False
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = call()
        assert watch.due <= watch.launches                     # still to be done
        assert not watch.pending
        watch.word.value = 123
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert watch.word.value == 123                         # no copy in the graph
        call()
        assert watch.pending and watch.due > watch.launches
    torch.cuda.synchronize()
    assert watch.word.value == 0
    assert torch.equal(y.cpu().double(), want)


def test_the_call_behind_a_landed_copy_raises(product):
    from tmq_b200 import _lib, ops
    call, watch, want = product
    ops.gemm_status_word("cuda").fill_(-4)
    watch.pending = False
    watch.due = watch.launches + 1
    call()
    torch.cuda.synchronize()
    with pytest.raises(_lib.TmqError):
        call()
    assert torch.equal(call().cpu().double(), want)
