"""8-bit row quantisation and the products with token and channel scales, plain and grouped by expert, against plain
64-bit implementations.

Tolerances (u = 2^-24, half a step of fp32; h = half a step of the output type):
  8-bit products: acc is an exact integer; int -> fp32, times row scale, fused times channel scale plus bias: at most
  3 u |acc rs sc| + u |y| before the output rounding of h |y|; asserted as 4 u |acc rs sc| + (h + 2 u) |y| plus the
  smallest subnormal of the output type.
  bf16 products: the tensor core adds 16 products per step to a running fp32 sum and may drop the bits below it: at most
  2^-22 of the largest magnitude in play per step, which sum_k |x w| bounds: (K / 16 + 1) 2^-22 sum|x w| |sc|.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    from tmq_b200 import ops
    yield ops
    ops.check_gemm_status()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ternary(seed, *shape):
    return torch.randint(-1, 2, shape, generator=gen(seed), dtype=torch.int8)


def codes(seed, *shape):
    return torch.randint(-128, 128, shape, generator=gen(seed), dtype=torch.int16).to(torch.int8)


def prepacked(ops, w, fmt):
    """[.., N, K] codes on the host -> prepacked weights on the device (a stack for three dimensions)"""
    if w.dim() == 3:
        return torch.stack([prepacked(ops, e, fmt) for e in w.unbind(0)])
    return ops.prepack(ops.compactify_ternary(w.cuda()), w.shape[0], fmt)


def quantized(x):
    """The definition: codes decided in 64 bits (the quotient of two fp32 numbers cannot come closer than 2^-33 to a
    border that it does not hit, far above the rounding of a 64-bit division)."""
    xd = x.double()
    amax = xd.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0])
    bad = ~torch.isfinite(xd).all(1)
    safe = torch.where((amax > 0) & ~bad, amax, torch.ones_like(amax))
    q = torch.where(bad[:, None], torch.zeros_like(xd), xd) * 127.0 / safe[:, None]
    q = torch.where((amax == 0)[:, None], torch.zeros_like(q), q)
    scale = amax.float() / torch.tensor(127.0)
    scale[bad] = float("nan")
    return q.round().to(torch.int8), scale


def check(y, acc, rs, sc, bi, extra=None):
    """acc: exact sums in 64 bits (host)"""
    prod = acc * rs.double()[:, None] * sc.double()
    ref = prod + (0 if bi is None else bi.double())
    h = torch.finfo(y.dtype).eps / 2
    tol = 4 * 2.0 ** -24 * prod.abs() + (h + 2.0 ** -23) * ref.abs() + TINY[y.dtype]
    if extra is not None:
        tol = tol + extra
    got = y.double().cpu()
    assert got.shape == ref.shape
    over = (got - ref).abs() - tol
    assert float(over.max()) <= 0, (float(over.max()), int(over.argmax()))


# ---------------------------------------------------------------------------------------------------------- quantisation

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 4096), (3, 15), (2, 16), (5, 17), (7, 255), (4, 4100), (3, 5003), (2, 20011),
                                 (1300, 520), (1200, 1027), (1, 40000)])
def test_quantize_rows(ops, M, K, dtype):
    x = (torch.randn(M, K, generator=gen(M * 31 + K)) * torch.exp(torch.randn(M, 1, generator=gen(K)))).to(DTYPES[dtype])
    q, s = ops.quantize_rows(x.cuda())
    eq, es = quantized(x)
    assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu(), es)
    assert q.stride(0) % 16 == 0 or M == 1
    whole = q.as_strided((M, (K + 15) // 16 * 16), (q.stride(0), 1))
    assert not whole[:, K:].any()                                     # the padding the products may read


def test_quantize_rows_on_the_borders(ops):
    """Quotients that are exact ties (round half to even), one step beside them, and extreme magnitudes."""
    rows = []
    for amax in (127.0, 254.0, 1.0, 3.0, 2.0 ** -140, 2.0 ** -120, 3.0e38, 1e-44):
        a = np.float32(amax)
        n = np.arange(-126, 126)
        exact = (n + 0.5) * float(a) / 127.0
        mid = exact.astype(np.float32)
        rows.append(np.concatenate([[a], mid, np.nextafter(mid, np.float32(np.inf)), np.nextafter(mid, np.float32(-np.inf))]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    x = torch.minimum(torch.maximum(x, -x[:, :1]), x[:, :1])
    q, s = ops.quantize_rows(x.cuda())
    eq, es = quantized(x)
    assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu(), es)


def test_quantize_rows_zero_and_non_finite_rows(ops):
    x = torch.randn(6, 77, generator=gen(1))
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 76] = float("inf")
    x[4, 0] = float("-inf")
    q, s = ops.quantize_rows(x.cuda())
    eq, es = quantized(x)
    assert torch.equal(q.cpu(), eq)
    assert torch.equal(torch.isnan(s.cpu()), torch.tensor([False, False, True, True, True, False]))
    assert s[1] == 0 and s[0].item() == es[0].item() and s[5].item() == es[5].item()


def test_quantize_rows_strides_and_out(ops):
    base = torch.randn(9, 201, generator=gen(2)).cuda()
    for x in (base[:, 3:180], base[::2], base.t(), base[:1].expand(5, 201), base[4:4]):
        q, s = ops.quantize_rows(x)
        eq, es = quantized(x.cpu())
        assert torch.equal(q.cpu(), eq) and torch.equal(s.cpu(), es)
    hold = torch.full((9, 230), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(9, device="cuda")
    q, s = ops.quantize_rows(base, out=(hold[:, 5:206], scale))
    eq, es = quantized(base.cpu())
    assert torch.equal(hold[:, 5:206].cpu(), eq) and torch.equal(scale.cpu(), es)
    assert (hold[:, :5] == 99).all() and (hold[:, 206:] == 99).all()


# ---------------------------------------------------------------------------------------------------------- products

SHAPES = [(1, 1, 1), (1, 128, 64), (1, 11008, 4096), (2, 1000, 2051), (3, 130, 72), (8, 256, 1024), (9, 200, 4100),
          (16, 4096, 512), (17, 129, 300), (24, 1000, 640), (33, 200, 192), (64, 128, 2304), (65, 127, 129), (100, 520, 576),
          (128, 1531, 333), (129, 128, 64), (256, 256, 1024), (300, 520, 577), (517, 1531, 2051), (1000, 40, 16)]


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_products_from_codes(ops, M, N, K, dense):
    x, w = codes(M + K, M, K), (codes if dense else ternary)(N + K, N, K)
    rs = torch.rand(M, generator=gen(K)) * 0.05
    sc = torch.rand(N, generator=gen(N)) * 0.1 - 0.05
    bi = torch.randn(N, generator=gen(M)) if M % 2 else None
    acc = x.double() @ w.double().t()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        rs_t = rs if dtype != torch.float16 else rs / K          # fp16 results stay finite
        if dense:
            wp = torch.nn.functional.pad(w, (0, -K % 16)).cuda()[:, :K]
            y = ops.gemm_i8(x.cuda(), wp, rs_t.cuda(), sc.cuda(), None if bi is None else bi.cuda(), out_dtype=dtype)
        else:
            y = ops.ternary_gemm_a8(x.cuda(), prepacked(ops, w, ops.FMT_I8), N, rs_t.cuda(), sc.cuda(),
                                    None if bi is None else bi.cuda(), out_dtype=dtype)
        assert y.dtype == dtype
        check(y, acc, rs_t, sc, bi)
    ops.check_gemm_status()


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("M,N,K", [(710, 2024, 700), (900, 1700, 1500), (400, 14000, 700), (2404, 1058, 930), (517, 11008, 1100),
                                   (1000, 11008, 300), (1747, 2100, 1007)])
def test_products_with_rows_dealt_evenly(ops, M, N, K, dense):
    """Sizes whose row tiles are neither 32, 64, 128 nor 256 rows high (80, 96, 112, 160, 176, 208, 224)."""
    test_products_from_codes(ops, M, N, K, dense)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 11008, 4096), (1, 77, 5), (2, 300, 1027), (4, 1000, 8192), (5, 640, 512), (8, 129, 2051),
                                   (12, 500, 700), (40, 300, 260), (200, 260, 515)])
def test_products_from_floating_point(ops, M, N, K, dtype):
    """Quantised by the call: the same numbers as quantising first."""
    x = (torch.randn(M, K, generator=gen(M + N)) * 3).to(DTYPES[dtype])
    w = ternary(K, N, K)
    sc = torch.rand(N, generator=gen(N)) * 0.1
    bi = torch.randn(N, generator=gen(M))
    wt = prepacked(ops, w, ops.FMT_I8)
    q, rs = quantized(x)
    y = ops.ternary_gemm_a8(x.cuda(), wt, N, scale=sc.cuda(), bias=bi.cuda(), out_dtype=torch.float32)
    check(y, q.double() @ w.double().t(), rs, sc, bi)
    wd = torch.nn.functional.pad(w, (0, -K % 16)).cuda()[:, :K]
    y = ops.gemm_i8(x.cuda(), wd, scale=sc.cuda(), bias=bi.cuda(), out_dtype=torch.float32)
    check(y, q.double() @ w.double().t(), rs, sc, bi)


@pytest.mark.parametrize("M", [1, 3, 20, 150])
def test_products_non_finite_rows_stay_alone(ops, M):
    N, K = 200, 300
    x = torch.randn(M, K, generator=gen(3))
    x[M // 2, 7] = float("nan")
    w = ternary(4, N, K)
    y = ops.ternary_gemm_a8(x.cuda(), prepacked(ops, w, ops.FMT_I8), N, out_dtype=torch.float32).cpu()
    assert torch.isnan(y[M // 2]).all()
    rest = [m for m in range(M) if m != M // 2]
    if rest:
        q, rs = quantized(x[rest])
        check(y[rest], q.double() @ w.double().t(), rs, torch.ones(N), None)


def test_products_without_scales_and_extreme_sums(ops):
    """Every operand at its largest magnitude: the int32 sums reach 2^14 K and stay exact."""
    K = 131071
    x = torch.full((2, K), -128, dtype=torch.int8)
    x[1] = 127
    w = torch.full((3, K), -128, dtype=torch.int8)
    w[1] = 127
    w[2, ::2] = 1
    wp = torch.nn.functional.pad(w, (0, -K % 16)).cuda()[:, :K]
    y = ops.gemm_i8(x.cuda(), wp, out_dtype=torch.float32)
    check(y, x.double() @ w.double().t(), torch.ones(2), torch.ones(3), None)
    t = ternary(9, 5, K)
    y = ops.ternary_gemm_a8(x.cuda(), prepacked(ops, t, ops.FMT_I8), 5, out_dtype=torch.float32)
    check(y, x.double() @ t.double().t(), torch.ones(2), torch.ones(5), None)


@pytest.mark.parametrize("M", [1, 7, 40, 200])
def test_products_strides_and_out(ops, M):
    N, K = 136, 272
    big = codes(5, M + 1, K + 37).cuda()
    w = ternary(6, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    rs = torch.rand(M, generator=gen(7))
    acc = lambda x: x.cpu().double() @ w.double().t()
    one = torch.ones(N)
    wide = torch.full((M, N + 50), 7.0, device="cuda")
    for x in (big[:M, 5:5 + K], big[1:M + 1, :K], codes(8, K, M).cuda().t(), codes(8, 1, K).cuda().expand(M, K)):
        for lo in (0, 8, 3):                                           # vector stores, vector stores, element stores
            wide.fill_(7.0)
            out = wide[:, lo:lo + N]
            y = ops.ternary_gemm_a8(x, wt, N, rs.cuda(), out_dtype=torch.float32, out=out)
            assert y.data_ptr() == out.data_ptr()
            check(y, acc(x), rs, one, None)
            assert (wide[:, :lo] == 7).all() and (wide[:, lo + N:] == 7).all()
    assert ops.ternary_gemm_a8(big[:0, :K], wt, N, out_dtype=torch.float32).shape == (0, N)


# ---------------------------------------------------------------------------------------------------------- grouped

def boundaries(counts, lead=0):
    return torch.tensor([lead] + [lead + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32)


GROUPS = [[5], [0, 3], [1, 1, 1, 1], [0, 0, 0], [64, 0, 65, 1], [7, 300, 0, 2], [130, 129, 257, 31], [1, 0, 700],
          [3] * 40 + [0] * 30, [2, 0, 1] * 50]


@pytest.mark.parametrize("form", ["ternary_i8", "ternary_bf16", "int8"])
@pytest.mark.parametrize("N,K", [(130, 72), (256, 1040), (33, 200), (130, 128), (200, 640), (64, 64)])
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}x{sum(c)}")
def test_grouped(ops, counts, N, K, form):
    E, T = len(counts), sum(counts)
    lead, tail = (2, 3) if len(counts) % 2 else (0, 0)                 # rows outside every group
    M = T + lead + tail
    off = boundaries(counts, lead)
    w = (codes if form == "int8" else ternary)(K, E, N, K)
    sc = torch.rand(E, N, generator=gen(N)) * 0.1
    bi = torch.randn(E, N, generator=gen(K)) if E % 2 else None
    dtype = torch.float32 if N == 130 else torch.bfloat16
    if form == "ternary_bf16":
        x, rs = torch.randn(M, K, generator=gen(T)).to(torch.bfloat16), None
    else:
        x, rs = codes(T, M, K), torch.rand(M, generator=gen(T)) * 0.05
    dev = lambda t: None if t is None else t.cuda()
    off_d = off.cuda() if E % 3 else off.long().cuda()
    kw = dict(scales=dev(sc), biases=dev(bi), out_dtype=dtype)
    if form == "int8":
        wp = torch.nn.functional.pad(w, (0, -K % 16)).cuda()[..., :K]
        call = lambda **o: ops.gemm_i8_grouped(x.cuda(), wp, off_d, row_scale=dev(rs), **kw, **o)
    else:
        wt = prepacked(ops, w, ops.FMT_BF16 if form == "ternary_bf16" else ops.FMT_I8)
        call = lambda **o: ops.ternary_gemm_grouped(x.cuda(), wt, N, off_d, row_scale=dev(rs), **kw, **o)
    kept = torch.full((M, N), 3.0, dtype=dtype, device="cuda")
    for y, rest in ((call(), 0.0), (call(out=kept), 3.0)):
        assert (y[:lead] == rest).all() and (y[M - tail:] == rest).all()
        for e, c in enumerate(counts):
            rows = slice(int(off[e]), int(off[e + 1]))
            if not c:
                continue
            xe, we = x[rows].double(), w[e].double()
            extra = None
            if form == "ternary_bf16":
                extra = (K / 16 + 1) * 2.0 ** -22 * (xe.abs() @ we.abs().t()) * sc[e].double().abs()
            check(y[rows], xe @ we.t(), torch.ones(c) if rs is None else rs[rows], sc[e], None if bi is None else bi[e], extra)
    ops.check_gemm_status()


def test_grouped_bad_boundaries_stay_inside(ops):
    """Boundaries out of range or out of order: clamped and raised to their predecessor, nothing outside the result."""
    E, M, N, K = 4, 50, 96, 64
    w = ternary(1, E, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    x = codes(2, M, K)
    for raw in ([-7, 10, 5, 30, 999], [0, 50, 50, 50, 50], [60, 70, 80, 90, 100], [20, 10, 0, -1, 40], [0, 0, 0, 0, 0]):
        seen, fixed = 0, []
        for v in raw:
            seen = max(seen, min(max(v, 0), M))
            fixed.append(seen)
        guard = torch.full((M + 8, N), 5.0, device="cuda")
        off = torch.tensor(raw, dtype=torch.int64, device="cuda")
        y = ops.ternary_gemm_grouped(x.cuda(), wt, N, off, out_dtype=torch.float32, out=guard[4:4 + M])
        assert (guard[:4] == 5).all() and (guard[4 + M:] == 5).all()
        for e in range(E):
            rows = slice(fixed[e], fixed[e + 1])
            assert torch.equal(y[rows].cpu().double(), x[rows].double() @ w[e].double().t())
        assert (y[:fixed[0]] == 5).all() and (y[fixed[-1]:] == 5).all()
    ops.check_gemm_status()


def test_grouped_many_groups(ops):
    E, N, K = ops.GROUPS_MAX, 40, 48
    counts = [(i * 7) % 4 for i in range(E)]
    x, w = codes(1, sum(counts), K), codes(2, E, N, K)
    off = boundaries(counts)
    y = ops.gemm_i8_grouped(x.cuda(), w.cuda(), off.cuda(), out_dtype=torch.float32).cpu().double()
    for e in range(E):
        rows = slice(int(off[e]), int(off[e + 1]))
        assert torch.equal(y[rows], x[rows].double() @ w[e].double().t())


# ---------------------------------------------------------------------------------------------------------- streams, graphs

def test_calls_on_another_stream_and_captured(ops):
    N, K, E = 300, 520, 3
    w = ternary(1, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    we = ternary(2, E, N, K)
    wts = prepacked(ops, we, ops.FMT_I8)
    x = torch.zeros(40, K, device="cuda", dtype=torch.bfloat16)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")

    def layer():
        y = ops.ternary_gemm_a8(x[:1], wt, N, out_dtype=torch.float32)
        q, s = ops.quantize_rows(x)
        z = ops.ternary_gemm_a8(q, wt, N, s, out_dtype=torch.float32)
        return y, z, ops.ternary_gemm_grouped(q, wts, N, off, s, out_dtype=torch.float32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, z, g = layer()
    torch.cuda.current_stream().wait_stream(side)
    for seed, bounds in ((1, [0, 10, 10, 40]), (2, [0, 40, 40, 40]), (3, [5, 6, 20, 31])):
        xs = torch.randn(40, K, generator=gen(seed)).to(torch.bfloat16)
        x.copy_(xs)
        off.copy_(torch.tensor(bounds))
        graph.replay()
        q, rs = quantized(xs)
        acc = q.double() @ w.double().t()
        check(y, acc[:1], rs[:1], torch.ones(N), None)
        check(z, acc, rs, torch.ones(N), None)
        for e in range(E):
            rows = slice(bounds[e], bounds[e + 1])
            if bounds[e] < bounds[e + 1]:
                check(g[rows], q[rows].double() @ we[e].double().t(), rs[rows], torch.ones(N), None)
        assert not g[:bounds[0]].any() and not g[bounds[-1]:].any()
    ops.check_gemm_status()


def test_same_call_twice_gives_the_same_bits(ops):
    x = torch.randn(300, 1030, generator=gen(1)).to(torch.bfloat16).cuda()
    wt = prepacked(ops, ternary(2, 700, 1030), ops.FMT_I8)
    for M in (1, 4, 60, 300):
        a = ops.ternary_gemm_a8(x[:M], wt, 700)
        b = ops.ternary_gemm_a8(x[:M], wt, 700)
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------- refusals

def test_refusals(ops):
    x = codes(1, 4, 64).cuda()
    w = ternary(2, 32, 64)
    wt = prepacked(ops, w, ops.FMT_I8)
    off = boundaries([2, 2]).cuda()
    wts = torch.stack([wt, wt])
    bad = [
        lambda: ops.quantize_rows(x),                                              # not floating point
        lambda: ops.quantize_rows(torch.zeros(2, 3)),                               # host tensor
        lambda: ops.quantize_rows(torch.zeros(3, device="cuda")),                   # not a matrix
        # width (packed rows are padded, so close widths cannot be told apart)
        lambda: ops.ternary_gemm_a8(codes(1, 4, 600).cuda(), wt, 32),
        lambda: ops.ternary_gemm_a8(x, prepacked(ops, w, ops.FMT_BF16), 32),        # layout of the other kind
        lambda: ops.ternary_gemm_a8(x, wt, 32, row_scale=torch.ones(5, device="cuda")),
        lambda: ops.ternary_gemm_a8(x, wt, 32, scale=torch.ones(31, device="cuda")),
        lambda: ops.ternary_gemm_a8(x, wt, 32, out=torch.empty(4, 32, device="cuda")),          # not the output dtype
        lambda: ops.ternary_gemm_a8(x.float(), wt, 32, row_scale=torch.ones(4, device="cuda")),
        lambda: ops.ternary_gemm_a8(x, wt, 32, out_dtype=torch.int32),
        lambda: ops.gemm_i8(x, codes(3, 32, 72).cuda()[:, 4:68]),                   # rows not aligned
        lambda: ops.gemm_i8(x, codes(3, 32, 48).cuda()),                            # width
        lambda: ops.gemm_i8(x, codes(3, 64, 32).cuda().t()),                        # column-major
        lambda: ops.ternary_gemm_grouped(x, wts, 32, off[:2]),                      # boundary count
        lambda: ops.ternary_gemm_grouped(x, wts, 32, off.cpu()),
        lambda: ops.ternary_gemm_grouped(x, wts, 32, off.float()),
        lambda: ops.ternary_gemm_grouped(x, wt, 32, off),                           # not stacked
        lambda: ops.ternary_gemm_grouped(x.to(torch.bfloat16), wts, 32, off),       # layout of the other kind
        lambda: ops.gemm_i8_grouped(x, codes(3, 2, 32, 80).cuda()[..., :64][:, :20], off),      # gaps inside the stack
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            call()
            pytest.fail(f"call {i} was not refused")
