"""Launches that let the next one start early, in front of skinny launches that take their result as scale or bias, directly and
with another skinny launch between.  The chains run as graphs (launches close together), on inputs that change from replay to
replay, and have to give what the same calls give with the device idle before each of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

N, K = 4096, 1024


@pytest.fixture(scope="module")
def ops():
    from tmq_b200 import ops
    yield ops
    ops.check_gemm_status()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ternary(seed, *shape):
    return torch.randint(-1, 2, shape, generator=gen(seed), dtype=torch.int8, device="cuda")


def prepacked(ops, w, fmt):
    return ops.prepack(ops.compactify_ternary(w), w.shape[0], fmt)


def producers(ops):
    """name -> (input, call that writes an fp32 vector of N numbers from it)"""
    w = ternary(1, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    wts = torch.stack([wt, wt])
    off = torch.tensor([0, 500, 1500], device="cuda")
    codes = lambda m: torch.zeros(m, K, dtype=torch.int8, device="cuda")
    out = lambda m: torch.zeros(m, N, device="cuda")
    made = {}
    x, q, s = torch.zeros(N, 8 * K, dtype=torch.bfloat16, device="cuda"), torch.zeros(N, 8 * K, dtype=torch.int8, device="cuda"), out(1)[0]
    made["quantize_rows"] = (x, lambda x=x, q=q, s=s: ops.quantize_rows(x, out=(q, s))[1])
    for name, m, call in (("token", 1, lambda x, y: ops.ternary_gemm_a8(x, wt, N, out_dtype=torch.float32, out=y)),
                          ("packed", 1500, lambda x, y: ops.ternary_gemm_a8(x, wt, N, out_dtype=torch.float32, out=y)),
                          ("int8", 1500, lambda x, y: ops.gemm_i8(x, w, out_dtype=torch.float32, out=y)),
                          ("grouped", 1500, lambda x, y: ops.ternary_gemm_grouped(x, wts, N, off, out_dtype=torch.float32, out=y)),
                          ("grouped int8", 1500, lambda x, y: ops.gemm_i8_grouped(x, torch.stack([w, w]), off,
                                                                                  out_dtype=torch.float32, out=y))):
        x, y = codes(m), out(m)
        made[name] = (x, lambda x=x, y=y, call=call: call(x, y)[-1])
    return made


@pytest.mark.parametrize("between", [0, 1, 2])
@pytest.mark.parametrize("name", ["quantize_rows", "token", "packed", "int8", "grouped", "grouped int8"])
def test_result_as_scale_and_bias_of_a_skinny_launch(ops, name, between):
    x, produce = producers(ops)[name]
    wt = prepacked(ops, ternary(2, N, K), ops.FMT_BF16)
    other = prepacked(ops, ternary(3, N, K), ops.FMT_BF16)
    h = torch.randn(3, K, generator=gen(4), device="cuda").to(torch.bfloat16)

    def chain(pause):
        v = produce()
        pause()
        for _ in range(between):
            ops.ternary_gemm(h, other, N, path="gemv")
            pause()
        y = ops.ternary_gemm(h, wt, N, v, v, out_dtype=torch.float32, path="gemv")
        pause()
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(lambda: None)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ys = [chain(lambda: None) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(6):
        if x.dtype == torch.int8:
            x.copy_(torch.randint(-127, 128, x.shape, generator=gen(seed), dtype=torch.int8, device="cuda"))
        else:
            x.copy_(torch.randn(x.shape, generator=gen(seed), device="cuda") * (seed + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in ys]
        want = chain(torch.cuda.synchronize)
        assert float(want.abs().max()) > 0
        assert all(torch.equal(y, want) for y in got), seed
