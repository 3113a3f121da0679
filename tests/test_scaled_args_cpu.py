"""Host-side refusals of the 8-bit and grouped products: status codes before anything is launched (no GPU)."""
import ctypes

P = ctypes.c_void_p
A, B, C, S = P(4096), P(8192), P(12288), P(16384)        # aligned, never dereferenced


def lib():
    from tmq_b200 import _lib
    return _lib.lib()


def test_quantize_rows_arguments():
    f = lib().tmq_quantize_rows
    assert f(A, 1, B, C, 0, 16, 16, 16, 16, None) == 0                     # no rows
    assert f(None, 1, B, C, 2, 16, 16, 16, 16, None) == -1
    assert f(A, 3, B, C, 2, 16, 16, 16, 16, None) == -1                    # type
    assert f(A, 1, B, C, 2, 0, 16, 16, 16, None) == -1
    assert f(A, 1, B, C, 2, 16, 15, 16, 16, None) == -1                    # rows overlap
    assert f(A, 1, B, C, 2, 16, 16, 15, 16, None) == -1                    # columns beyond the row stride
    assert f(A, 1, B, C, 2, 16, 16, 16, 15, None) == -1                    # fewer columns than codes
    assert f(A, 1, B, C, -1, 16, 16, 16, 16, None) == -1
    assert f(P(4097), 1, B, C, 2, 16, 16, 16, 16, None) == -2
    assert f(A, 0, B, P(12289), 2, 16, 16, 16, 16, None) == -2


def a8(X=A, x_type=-1, ldx=64, rs=None, W=B, sc=None, bi=None, Y=C, y_type=1, M=32, N=40, K=64, ldy=40, ws=None, nws=0, st=S):
    return lib().tmq_ternary_gemm_a8(X, x_type, ldx, rs, W, sc, bi, Y, y_type, M, N, K, ldy, ws, nws, st, None)


def i8(X=A, x_type=-1, ldx=64, rs=None, W=B, ldw=64, sc=None, bi=None, Y=C, y_type=1, M=32, N=40, K=64, ldy=40, ws=None, nws=0,
       st=S):
    return lib().tmq_gemm_i8(X, x_type, ldx, rs, W, ldw, sc, bi, Y, y_type, M, N, K, ldy, ws, nws, st, None)


def test_product_arguments():
    for f in (a8, i8):
        assert f(M=0) == 0
        for bad in (dict(X=None), dict(W=None), dict(Y=None), dict(st=None), dict(M=-1), dict(N=0), dict(K=0), dict(ldx=63),
                    dict(ldy=39), dict(y_type=3), dict(x_type=-2), dict(x_type=3)):
            assert f(**bad) == -1, bad
        for bad in (dict(X=P(4100)), dict(W=P(8196)), dict(st=P(16386)), dict(Y=P(12289)), dict(rs=P(2)), dict(sc=P(2)),
                    dict(bi=P(2))):
            assert f(**bad) == -2, bad
        assert f(K=131072, ldx=131072) == -6 if f is a8 else f(K=131072, ldx=131072, ldw=131072) == -6    # int32 sums
        assert f(ldx=72) == -6                                             # rows not at multiples of 16 bytes
        # floating point: scratch, and no row scale
        assert f(x_type=1) == -5 and f(x_type=1, ws=P(65536), nws=32 * 64) == -5
        assert f(x_type=1, ws=P(65537), nws=1 << 20) == -2
        assert f(x_type=1, rs=P(4096), ws=P(65536), nws=1 << 20) == -1
        assert f(x_type=1, X=P(4097), ws=P(65536), nws=1 << 20) == -2
    assert i8(ldw=63) == -1 and i8(ldw=72) == -6
    assert a8(M=4, x_type=1, rs=P(4096)) == -1 and a8(M=4, X=P(4100)) == -2     # the one-launch form
    assert a8(M=4, x_type=1, N=12000, ldy=12000) == -5                     # too wide for it: scratch
    assert a8(M=8, x_type=1, K=2064, ldx=2064) == -5                       # too many elements for it


def test_scratch_size():
    n = lib().tmq_a8_workspace_bytes
    assert n(-1, 4, 100) == 0 and n(3, 4, 100) == 0 and n(1, 0, 100) == 0
    assert n(1, 4, 100) == 4 * 112 + 16


def test_grouped_arguments():
    L = lib()

    def grouped(form, off=P(20480), ob=4, E=3, M=32, N=40, K=64, ldx=64, ldw=64, ldy=40, y_type=1, X=A, st=S):
        tail = (off, ob, E, C, y_type, M, N, K, ldy, 0, st, None)
        if form == "bf16":
            return L.tmq_ternary_gemm_grouped_bf16(X, ldx, B, None, None, *tail)
        if form == "a8":
            return L.tmq_ternary_gemm_grouped_a8(X, ldx, None, B, None, None, *tail)
        return L.tmq_gemm_grouped_i8(X, ldx, None, B, ldw, None, None, *tail)

    for form in ("bf16", "a8", "i8"):
        assert grouped(form, M=0) == 0
        for bad in (dict(off=None), dict(ob=2), dict(E=0), dict(N=0), dict(K=-1), dict(ldx=60), dict(ldy=3), dict(y_type=-1),
                    dict(X=None), dict(st=None)):
            assert grouped(form, **bad) == -1, (form, bad)
        for bad in (dict(off=P(20482)), dict(off=P(20484), ob=8), dict(X=P(4104))):
            assert grouped(form, **bad) == -2, (form, bad)
        assert grouped(form, E=513) == -6                                  # TMQ_GROUPS_MAX
        assert grouped(form, M=2 ** 31) == -6
        assert grouped(form, N=2 ** 30, ldy=2 ** 30) == -6                 # weight rows beyond 2^31
    assert grouped("bf16", ldx=68) == -6 and grouped("i8", ldw=72) == -6
