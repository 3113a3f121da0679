"""Tiles of 65 .. 128 rows with packed weights, where two pairs of decode warps share the ring of packed words: short rows, many
units per CTA, weights that come from memory and from L2 by turns, so that their copies land out of order.  All numbers are
small integers, so every sum is exact in fp32 and results are compared bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from tmq_b200 import ops
    yield ops
    ops.check_gemm_status()


@pytest.fixture(scope="module")
def flush():
    return torch.empty(1 << 28, dtype=torch.uint8, device="cuda")          # larger than L2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ternary(seed, *shape):
    return torch.randint(-1, 2, shape, generator=gen(seed), dtype=torch.int8, device="cuda")


def prepacked(ops, w, fmt):
    return ops.prepack(ops.compactify_ternary(w), w.shape[0], fmt)


@pytest.mark.parametrize("M,N,K", [(3131, 10119, 64), (2981, 7175, 128), (4096, 4096, 200), (4096, 4096, 256), (2128, 3272, 384),
                                   (1649, 7102, 512), (2680, 3574, 1000), (560, 7997, 2048)])
def test_products(ops, flush, M, N, K):
    x = torch.randint(-127, 128, (M, K), generator=gen(K), dtype=torch.int8, device="cuda")
    w = [ternary(K + i, N, K) for i in range(3)]
    wt = [prepacked(ops, t, ops.FMT_I8) for t in w]
    want = [x.float() @ t.float().t() for t in w]                          # |sums| < 2^24
    for turn in range(4):
        if turn % 2:
            flush.zero_()
        for i in range(3):
            assert torch.equal(ops.ternary_gemm_a8(x, wt[i], N, out_dtype=torch.float32), want[i]), (turn, i)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("E,M,N,K", [(16, 2901, 8606, 64), (16, 4218, 4064, 128), (16, 5786, 2806, 200), (16, 3307, 4968, 256),
                                     (16, 2555, 5061, 512), (40, 5411, 1614, 1000), (40, 4047, 1672, 1500)])
def test_grouped_products(ops, flush, E, M, N, K, bf16):
    top = 8 if bf16 else 127                                               # integers that bf16 holds
    x = torch.randint(-top, top + 1, (M, K), generator=gen(K), dtype=torch.int8, device="cuda")
    x = x.to(torch.bfloat16) if bf16 else x
    w = ternary(K + 1, E, N, K)
    wts = torch.stack([prepacked(ops, t, ops.FMT_BF16 if bf16 else ops.FMT_I8) for t in w.unbind(0)])
    cut = torch.randint(0, M + 1, (E - 1,), generator=gen(M), device="cuda").sort().values
    off = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), M)])
    at = off.tolist()
    want = torch.cat([x[a:b].float() @ t.float().t() for a, b, t in zip(at, at[1:], w.unbind(0))])
    for turn in range(4):
        if turn % 2:
            flush.zero_()
        assert torch.equal(ops.ternary_gemm_grouped(x, wts, N, off, out_dtype=torch.float32), want), turn
