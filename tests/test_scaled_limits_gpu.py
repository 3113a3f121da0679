"""The 8-bit and grouped products at their edges: results and rows beyond 2^31 elements, calls on two streams at once, a set
status word, and the same product by every route giving the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tmq_b200 import ops
    yield ops
    ops.check_gemm_status()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ternary(seed, *shape):
    return torch.randint(-1, 2, shape, generator=gen(seed), dtype=torch.int8, device="cuda")


def codes(seed, *shape):
    return torch.randint(-127, 128, shape, generator=gen(seed), dtype=torch.int8, device="cuda")


def prepacked(ops, w, fmt):
    if w.dim() == 3:
        return torch.stack([prepacked(ops, e, fmt) for e in w.unbind(0)])
    return ops.prepack(ops.compactify_ternary(w), w.shape[0], fmt)


def test_results_beyond_32_bit_offsets(ops):
    M, N, K = 70001, 32768, 32                     # 2.29e9 results
    x, w = codes(1, M, K), ternary(2, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    y = ops.ternary_gemm_a8(x, wt, N)              # sums below 2^12: exact in bf16 only up to 2^8, so scaled rows are compared
    for m in (0, 65535, 65536, 65537, M - 1):
        ref = (x[m].double() @ w.double().t()).to(torch.bfloat16)
        assert torch.equal(y[m], ref), m
    off = torch.tensor([0, 10, 65600, M], device="cuda", dtype=torch.int64)
    ws = torch.stack([w, -w, w])
    g = ops.ternary_gemm_grouped(x, prepacked(ops, ws, ops.FMT_I8), N, off, out=y)
    for m, e in ((9, 0), (10, 1), (65599, 1), (65600, 2), (M - 1, 2)):
        assert torch.equal(g[m], (x[m].double() @ ws[e].double().t()).to(torch.bfloat16)), m


def test_quantised_rows_beyond_32_bit_offsets(ops):
    M, K = 140001, 16384                           # 2.29e9 codes
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    for i in range(0, M, 20000):
        x[i:i + 20000].normal_(generator=gen(i))
    q, s = ops.quantize_rows(x)
    for m in (0, 131071, 131072, M - 1):
        xd = x[m].double()
        assert torch.equal(q[m], (127.0 * xd / xd.abs().max()).round().to(torch.int8)), m
        assert s[m].cpu() == xd.abs().max().float().cpu() / torch.tensor(127.0)


def test_two_streams_at_once(ops):
    N, K, E = 1000, 1032, 5
    w, we = ternary(3, N, K), ternary(4, E, N, K)
    wt, wts = prepacked(ops, w, ops.FMT_I8), prepacked(ops, we, ops.FMT_I8)
    xs = [codes(10 + i, 200, K) for i in range(2)]
    rs = [torch.rand(200, generator=gen(20 + i), device="cuda") for i in range(2)]
    offs = [torch.tensor([0, 3, 3, 120, 130, 200], device="cuda"), torch.tensor([0, 64, 65, 66, 67, 200], device="cuda")]

    def work(i):
        return (ops.ternary_gemm_a8(xs[i], wt, N, rs[i]), ops.ternary_gemm_a8(xs[i][:3], wt, N, rs[i][:3]),
                ops.ternary_gemm_a8(xs[i].float(), wt, N), ops.ternary_gemm_grouped(xs[i], wts, N, offs[i], rs[i]))

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for results in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(results, want[i]))


def test_every_route_gives_the_same_bits(ops):
    """Rows of one product do not depend on how many of them a call has, nor on who quantised them, nor on the grouping."""
    N, K = 700, 1500
    x = torch.randn(300, K, generator=gen(1), device="cuda").to(torch.bfloat16)
    w = ternary(2, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    wd = torch.nn.functional.pad(w, (0, -K % 16))[:, :K]
    sc, bi = torch.rand(N, generator=gen(3), device="cuda"), torch.randn(N, generator=gen(4), device="cuda")
    q, s = ops.quantize_rows(x)
    whole = ops.ternary_gemm_a8(q, wt, N, s, sc, bi, out_dtype=torch.float32)
    for m in (1, 2, 5, 8, 9, 33, 64, 65, 130, 257, 300):
        for y in (ops.ternary_gemm_a8(x[:m], wt, N, scale=sc, bias=bi, out_dtype=torch.float32),
                  ops.ternary_gemm_a8(q[:m], wt, N, s[:m], sc, bi, out_dtype=torch.float32),
                  ops.gemm_i8(x[:m], wd, scale=sc, bias=bi, out_dtype=torch.float32),
                  ops.gemm_i8(q[:m], wd, s[:m], sc, bi, out_dtype=torch.float32)):
            assert torch.equal(y, whole[:m]), m
    off = torch.tensor([0, 7, 7, 150, 300], device="cuda", dtype=torch.int32)
    y = ops.ternary_gemm_grouped(q, torch.stack([wt] * 4), N, off, s, sc.expand(4, N), bi.expand(4, N), out_dtype=torch.float32)
    assert torch.equal(y, whole)
    y = ops.gemm_i8_grouped(q, torch.nn.functional.pad(w, (0, -K % 16)).expand(4, N, -1).contiguous()[..., :K], off, s,
                            sc.expand(4, N), bi.expand(4, N), out_dtype=torch.float32)
    assert torch.equal(y, whole)


def test_a_set_status_word_leaves_results_alone(ops):
    from tmq_b200 import _lib
    N, K = 300, 640
    x, w = codes(1, 40, K), ternary(2, N, K)
    wt8, wt16 = prepacked(ops, w, ops.FMT_I8), prepacked(ops, w, ops.FMT_BF16)
    off = torch.tensor([3, 20, 38], device="cuda")
    out = torch.full((40, N), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.check_gemm_status()
    calls = [lambda: ops.ternary_gemm_a8(x, wt8, N, out=out), lambda: ops.ternary_gemm_a8(x[:2], wt8, N, out=out[:2]),
             lambda: ops.ternary_gemm_a8(x.float(), wt8, N, out=out), lambda: ops.gemm_i8(x, w, out=out),
             lambda: ops.ternary_gemm_grouped(x, torch.stack([wt8, wt8]), N, off, out=out),
             lambda: ops.ternary_gemm_grouped(x.to(torch.bfloat16), torch.stack([wt16, wt16]), N, off, out=out),
             lambda: ops.gemm_i8_grouped(x, torch.stack([w, w]), off, out=out)]
    for call in calls:
        ops.gemm_status_word(x.device).fill_(-4)
        try:
            call()
        except _lib.TmqError:                      # the watch may find it first
            ops.gemm_status_word(x.device).fill_(-4)
            call()
        with pytest.raises(_lib.TmqError):
            ops.check_gemm_status()
        assert (out == 7).all()
    assert torch.equal(ops.ternary_gemm_a8(x, wt8, N, out_dtype=torch.float32).double(), x.double() @ w.double().t())
