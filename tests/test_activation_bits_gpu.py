"""8-bit activations through the API: tmq.set_activation_bits on packed Linear layers, tmq.PackedExperts, and a small
feed-forward block of experts that uses quantisation, grouped and plain products together.

Reference: the definition in 64 bits.  A row's codes are exact, so the only errors are the roundings of the scaling (a few
2^-24) and of the result (half a step of its type); an intermediate result that is rounded and quantised again is rounded
in the reference as well, and where a value lies next to a rounding border of the codes the reference takes the codes of the
kernel's own input."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tmq():
    import tmq_b200
    return tmq_b200


def packed_linear(tmq, n_in, n_out, seed, bias=True, post_scale=False):
    torch.manual_seed(seed)
    ctrl = tmq.QuantizationControl(post_scale=post_scale)
    lin = tmq.Linear(n_in, n_out, bias=bias, ctrl=ctrl, quant_mode=tmq.QuantMode.TERNARY, post_scale=post_scale)
    w = torch.randint(-1, 2, (n_out, n_in)).float()
    with torch.no_grad():
        lin.weight.copy_(w)
        if bias:
            lin.bias.normal_()
    ctrl.register_node("0", lin)
    holder = nn.Sequential(lin).cuda().eval()
    tmq.compressed_state_dict(holder)
    assert lin.compact
    return lin, w


def row_codes(x):
    """(codes, scale) in 64 bits of the exact definition; scale is the fp32 number"""
    xd = x.double()
    amax = xd.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, 127.0 * xd / amax.clamp_min(1e-300), torch.zeros_like(xd)).round()
    return q, (amax.float() / torch.tensor(127.0)).double()


def want(x, w, scale, bias):
    q, s = row_codes(x)
    y = (q @ w.double().t()) * s * scale
    return y if bias is None else y + bias.double()


def close(y, ref, prod_bound):
    h = torch.finfo(y.dtype).eps / 2
    tol = 4 * 2.0 ** -24 * prod_bound + (h + 2.0 ** -23) * ref.abs() + 2.0 ** -24
    over = (y.double().cpu() - ref).abs() - tol
    assert float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("post_scale", [False, True])
def test_linear_with_8_bit_activations(tmq, dtype, post_scale):
    lin, w = packed_linear(tmq, 203, 77, 3, post_scale=post_scale)
    holder = nn.Sequential(lin)
    before = lin(torch.randn(5, 203, device="cuda"))
    assert before.dtype == torch.float32
    tmq.set_activation_bits(holder, 8)
    for shape in [(203,), (1, 203), (4, 203), (2, 3, 203), (40, 203), (150, 203)]:
        x = torch.randn(*shape).to(dtype)
        y = lin(x.cuda())
        assert y.dtype == dtype and y.shape == shape[:-1] + (77,)
        x2 = x.reshape(-1, 203)
        ref = want(x2, w, lin.post_scale_imm, lin.bias.detach().cpu())
        q, s = row_codes(x2)
        close(y.reshape(-1, 77), ref, (q.abs() @ w.abs().double().t()) * s * abs(lin.post_scale_imm))
    with pytest.raises(RuntimeError):
        lin(torch.ones(2, 204, device="cuda", dtype=dtype))
    raw = lin(torch.ones(2, 203, dtype=torch.int8, device="cuda"))          # codes keep their raw sums
    assert raw.dtype == torch.int32
    tmq.set_activation_bits(holder, None)
    x = torch.randn(3, 203, device="cuda")
    assert torch.equal(lin(x), lin(x)) and lin.activation_bits is None
    with pytest.raises(ValueError):
        tmq.set_activation_bits(holder, 4)


@pytest.mark.parametrize("bits", [None, 8])
def test_packed_experts(tmq, bits):
    n_in, n_out = 200, 96
    pairs = [packed_linear(tmq, n_in, n_out, 10 + e, bias=e % 2 == 0, post_scale=e == 1) for e in range(4)]
    experts = tmq.PackedExperts([p[0] for p in pairs], activation_bits=bits)
    counts = [3, 0, 70, 5]
    off = torch.tensor([0, 3, 3, 73, 78], device="cuda")
    x = torch.randn(78, n_in).to(torch.bfloat16)
    y = experts(x.cuda(), off)
    assert y.dtype == torch.bfloat16 and y.shape == (78, n_out)
    row = 0
    for (lin, w), c in zip(pairs, counts):
        if c:
            xe, sc = x[row:row + c], float(lin.post_scale_imm)
            bias = None if lin.bias is None else lin.bias.detach().cpu()
            if bits == 8:
                q, s = row_codes(xe)
                close(y[row:row + c], want(xe, w, sc, bias), (q.abs() @ w.abs().double().t()) * s * sc)
            else:
                # fp32 accumulation on the tensor cores: 2^-22 of sum |x w| for each of the K / 16 steps
                ref = (xe.double() @ w.double().t()) * sc + (0 if bias is None else bias.double())
                close(y[row:row + c], ref, (n_in / 16 + 1) * (xe.double().abs() @ w.abs().double().t()) * sc)
        row += c


def test_packed_experts_refusals(tmq):
    a, _ = packed_linear(tmq, 64, 32, 1)
    b, _ = packed_linear(tmq, 64, 48, 2)
    fresh = tmq.Linear(64, 32, ctrl=tmq.QuantizationControl(), quant_mode=tmq.QuantMode.TERNARY).cuda()
    for layers, kw in (([a, b], {}), ([a, fresh], {}), ([], {}), ([a], {"activation_bits": 4})):
        with pytest.raises((RuntimeError, ValueError)):
            tmq.PackedExperts(layers, **kw)
    ex = tmq.PackedExperts([a, a])
    with pytest.raises(RuntimeError):
        ex(torch.zeros(4, 60, device="cuda", dtype=torch.bfloat16), torch.tensor([0, 2, 4], device="cuda"))
    with pytest.raises(RuntimeError):
        ex(torch.zeros(4, 64, device="cuda"), torch.tensor([0, 2, 4], device="cuda"))      # fp32 rows need activation_bits


@pytest.mark.parametrize("tokens", [1, 7, 130])
def test_expert_block_together(tmq, tokens):
    """Router choice -> rows sorted by expert -> 8-bit grouped up projection -> ReLU -> 8-bit grouped down projection ->
    rows back in token order -> an 8-bit head with 8-bit weights."""
    from tmq_b200 import ops
    d, hidden, E, top, vocab = 128, 264, 6, 2, 100
    ups = [packed_linear(tmq, d, hidden, 20 + e) for e in range(E)]
    downs = [packed_linear(tmq, hidden, d, 40 + e) for e in range(E)]
    up = tmq.PackedExperts([p[0] for p in ups], activation_bits=8)
    down = tmq.PackedExperts([p[0] for p in downs], activation_bits=8)
    gen = torch.Generator().manual_seed(tokens)
    head = torch.randn(vocab, d, generator=gen)
    head_q, head_s = ops.quantize_rows(head.cuda())
    x = torch.randn(tokens, d, generator=gen)
    choice = torch.stack([torch.randperm(E, generator=gen)[:top] for _ in range(tokens)])
    flat = choice.flatten()
    order = torch.argsort(flat, stable=True)
    off = torch.zeros(E + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.bincount(flat, minlength=E), 0)
    rows = x[order // top].cuda()
    h = torch.relu(up(rows, off.cuda()))
    y = down(h, off.cuda())
    out = torch.zeros(tokens, d, device="cuda").index_add_(0, (order // top).cuda(), y)
    logits = ops.gemm_i8(out, head_q, scale=head_s, out_dtype=torch.float32)

    for e in range(E):
        r = slice(int(off[e]), int(off[e + 1]))
        if r.start == r.stop:
            continue
        for got, src, (lin, w) in ((h, rows, ups[e]), (y, h, downs[e])):
            q, s = row_codes(src[r].cpu())
            ref = want(src[r].cpu(), w, 1.0, lin.bias.detach().cpu())
            close(got[r], torch.relu(ref) if got is h else ref, (q.abs() @ w.abs().double().t()) * s)
    q, s = row_codes(out.cpu())
    hq, hs = row_codes(head)
    acc = q @ hq.t()
    close(logits, acc * s * hs.t(), acc.abs() * s * hs.t())
    ops.check_gemm_status()
