"""Forms of the 8-bit and grouped products that lie between the others: few rows against a matrix too wide for one launch, rows with
NaN and infinities beside other experts' rows, one expert over a part of the rows.

Tolerances as for every product of this kind (u = 2^-24): 4 u |acc rs sc| + 2 u |y| for 8 bits, where the sums are exact; for
bf16 rows of small integers the sums are exact in fp32 and results are compared bit for bit."""
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


def prepacked(ops, w, fmt):
    return ops.prepack(ops.compactify_ternary(w), w.shape[0], fmt)


@pytest.mark.parametrize("M", [1, 2, 5, 8])
@pytest.mark.parametrize("N,K", [(11840, 520), (11841, 520), (14336, 300), (28672, 1030), (700, 33000), (11008, 20000)])
def test_few_rows_of_wide_matrices(ops, M, N, K):
    w = ternary(N, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)
    x = torch.randn(M, K, generator=gen(M), device="cuda")
    sc, bi = torch.rand(N, generator=gen(1), device="cuda") + 0.5, torch.randn(N, generator=gen(2), device="cuda")
    q, s = ops.quantize_rows(x)
    xd = x.double()
    assert torch.equal(q, (127.0 * xd / xd.abs().amax(1, keepdim=True)).round().to(torch.int8))
    acc = torch.stack([(w.float() @ row.float()) for row in q]).double()          # |sums| < 2^24: exact
    prod = acc * s.double()[:, None] * sc.double()
    ref = prod + bi.double()
    a = ops.ternary_gemm_a8(x, wt, N, scale=sc, bias=bi, out_dtype=torch.float32)
    b = ops.ternary_gemm_a8(q, wt, N, s, sc, bi, out_dtype=torch.float32)
    assert torch.equal(a, b)
    assert float(((a.double() - ref).abs() - 2.0 ** -24 * (4 * prod.abs() + 2 * ref.abs())).max()) <= 0


@pytest.mark.parametrize("counts", [[3, 1, 0, 4], [40, 1, 17, 90], [200, 2, 130, 300]])
def test_non_finite_rows_beside_other_experts(ops, counts):
    """NaN and infinities in a group's rows, and in rows of no group, reach that row's results only."""
    N, K, E = 200, 328, len(counts)
    lead, T = 2, sum(counts)
    M = lead + T + 2
    at = [lead]
    for c in counts:
        at.append(at[-1] + c)
    x = torch.randint(-8, 9, (M, K), generator=gen(T), dtype=torch.int8, device="cuda").to(torch.bfloat16)
    w = ternary(T + 1, E, N, K)
    w[:, :, 7] = 1                                                                # every channel sees the column
    wts = torch.stack([prepacked(ops, t, ops.FMT_BF16) for t in w.unbind(0)])
    want = torch.zeros(M, N, device="cuda")
    for e in range(E):
        want[at[e]:at[e + 1]] = x[at[e]:at[e + 1]].float() @ w[e].float().t()
    bad = {0: float("nan"), at[1] - 1: float("nan"), at[1]: float("inf"), at[-1] - 1: float("-inf"), at[-1]: float("inf")}
    for row, value in bad.items():
        x[row, 7] = value
    y = ops.ternary_gemm_grouped(x, wts, N, torch.tensor(at, device="cuda"), out_dtype=torch.float32)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[[at[1] - 1, at[1], at[-1] - 1]] = False
    assert torch.equal(y[keep], want[keep])
    assert not torch.isfinite(y[~keep]).any()


@pytest.mark.parametrize("M", [5, 100, 300, 1000])
def test_one_expert_over_a_part_of_the_rows(ops, M):
    N, K = 300, 456
    x = torch.randint(-127, 128, (M, K), generator=gen(M), dtype=torch.int8, device="cuda")
    w = ternary(M + 1, N, K)
    wt = prepacked(ops, w, ops.FMT_I8)[None]
    full = x.float() @ w.float().t()
    for lo, hi in ((0, M), (0, M // 2), (1, M - 1), (M // 3, M // 2), (M - 1, M), (M, M)):
        y = ops.ternary_gemm_grouped(x, wt, N, torch.tensor([lo, hi], device="cuda"), out_dtype=torch.float32)
        z = ops.gemm_i8_grouped(x, torch.nn.functional.pad(w, (0, -K % 16))[None, :, :K], torch.tensor([lo, hi], device="cuda"),
                                out_dtype=torch.float32)
        want = torch.zeros_like(full)
        want[lo:hi] = full[lo:hi]
        assert torch.equal(y, want) and torch.equal(z, want), (lo, hi)
