"""Argument checks of the group norm, dropout, quantiser and 8-bit product entry
points: every refusal happens before any device work, so no GPU is needed."""
import ctypes as C

import pytest

from support import nb

P = C.c_void_p(4096)  # never dereferenced: every call below fails its checks
ODD = C.c_void_p(4097)
BAD, UNSUP = nb.NPL_ERR_INVALID_ARG, nb.NPL_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    return nb.load()


def norm(lib, n=2, hw=5, c=6, groups=3, dtype=0, x=P, ldx=6, eps=1e-5, act=0, y=P, ldy=6, work=P,
         size=1 << 40):
    return lib.nplk_group_norm_act(None, n, hw, c, groups, dtype, x, ldx, None, None, eps, act,
                                   0.0, y, ldy, None, None, work, size)


def grad(lib, n=2, hw=5, c=6, groups=3, dtype=0, dy=P, lddy=6, x=P, ldx=6, mean=P, rstd=P, act=0,
         dx=P, lddx=6, work=P, size=1 << 40):
    return lib.nplk_group_norm_act_backward(None, n, hw, c, groups, dtype, dy, lddy, x, ldx, mean,
                                            rstd, None, None, act, 0.0, dx, lddx, None, None,
                                            work, size)


SIZES = [dict(n=0), dict(hw=0), dict(c=0, groups=1), dict(groups=0), dict(groups=4), dict(n=-1),
         dict(dtype=3), dict(dtype=-1), dict(act=11), dict(act=-1), dict(work=None),
         dict(size=16), dict(work=C.c_void_p(4096 + 128))]


@pytest.mark.parametrize("change", SIZES + [
    dict(x=None), dict(y=None), dict(ldx=5), dict(ldy=5), dict(x=ODD), dict(y=ODD),
    dict(dtype=1, x=ODD), dict(ldx=8, x=P, y=P)])
def test_group_norm_refuses(lib, change):
    assert norm(lib, **change) == BAD


@pytest.mark.parametrize("change", SIZES + [
    dict(x=None), dict(dy=None), dict(dx=None), dict(mean=None), dict(rstd=None), dict(ldx=5),
    dict(lddy=5), dict(lddx=5), dict(x=ODD), dict(dy=ODD), dict(dx=ODD),
    dict(lddy=8, x=C.c_void_p(8192)), dict(ldx=8, dy=C.c_void_p(8192))])
def test_group_norm_gradient_refuses(lib, change):
    assert grad(lib, **change) == BAD


def test_group_norm_too_large(lib):
    wide = dict(c=8193 * 2, groups=2, ldx=8193 * 2)
    assert norm(lib, **wide, ldy=8193 * 2) == UNSUP
    assert grad(lib, **wide, lddy=8193 * 2, lddx=8193 * 2) == UNSUP
    assert norm(lib, hw=1 << 31) == UNSUP and norm(lib, n=1 << 31) == UNSUP
    assert norm(lib, n=1 << 30, c=64, groups=32, ldx=64, ldy=64) == UNSUP
    assert lib.nplk_group_norm_workspace_size(2, 5, 6, 4) == 0
    assert lib.nplk_group_norm_workspace_size(1 << 31, 5, 6, 3) == 0
    assert lib.nplk_group_norm_workspace_size(2, 5, 6, 3) > 0


def test_dropout_refuses(lib):
    def call(n=8, dtype=0, x=P, y=P, p=0.5, at=None):
        return lib.nplk_dropout(None, n, dtype, x, y, p, 1, 0, at)

    for change in (dict(n=0), dict(n=-3), dict(dtype=3), dict(x=None), dict(y=None), dict(p=-0.1),
                   dict(p=1.5), dict(p=float("nan")), dict(x=ODD), dict(y=ODD),
                   dict(at=C.c_void_p(4100))):
        assert call(**change) == BAD, change


@pytest.mark.parametrize("name", ["nplk_quantize_rows", "nplk_quantize_cols"])
def test_quantize_refuses(lib, name):
    def call(rows=4, cols=4, dtype=0, x=P, ldx=4, q=P, ldq=16, scale=P):
        return getattr(lib, name)(None, rows, cols, dtype, x, ldx, q, ldq, scale)

    for change in (dict(rows=0), dict(cols=0), dict(dtype=4), dict(x=None), dict(q=None),
                   dict(scale=None), dict(ldx=3), dict(ldq=3), dict(x=ODD), dict(rows=-1)):
        assert call(**change) == BAD, change
    big = 1 << 31
    assert call(rows=big, ldq=big) == UNSUP
    assert call(cols=big, ldx=big, ldq=big) == UNSUP


def test_gemm_i8_refuses(lib):
    def call(m=4, n=4, k=16, a=P, lda=16, sa=P, b=P, ldb=16, sb=P, act=0, dtype=0, c=P, ldc=4):
        return lib.nplk_gemm_i8(None, m, n, k, a, lda, sa, b, ldb, sb, None, act, 0.0, dtype, c,
                                ldc, None)

    for change in (dict(m=0), dict(n=0), dict(k=0), dict(m=-1), dict(a=None), dict(b=None),
                   dict(sa=None), dict(sb=None), dict(c=None), dict(lda=15), dict(ldb=15),
                   dict(ldc=3), dict(act=11), dict(act=-1), dict(dtype=3), dict(c=ODD),
                   dict(dtype=2, c=ODD)):
        assert call(**change) == BAD, change
    assert call(k=131072, lda=131072, ldb=131072) == UNSUP
    assert call(m=(1 << 30) + 1) == UNSUP
    assert call(n=(1 << 30) + 1, ldc=1 << 31) == UNSUP


@pytest.mark.parametrize("which", range(6))
def test_misaligned_fp32_arguments_are_refused(lib, which):
    odd = [ODD if i == which else P for i in range(6)]
    work, size = P, 1 << 40
    if which < 4:
        assert lib.nplk_group_norm_act(None, 2, 5, 6, 3, 0, P, 6, odd[0], odd[1], 1e-5, 0, 0.0, P,
                                       6, odd[2], odd[3], work, size) == BAD
        assert lib.nplk_gemm_i8(None, 4, 4, 16, P, 16, odd[0], P, 16, odd[1], odd[2], 0, 0.0,
                                0, P, 4, odd[3]) == BAD
    assert lib.nplk_group_norm_act_backward(None, 2, 5, 6, 3, 0, P, 6, P, 6, odd[0], odd[1],
                                            odd[2], odd[3], 0, 0.0, P, 6, odd[4], odd[5], work,
                                            size) == BAD
    for call in (lib.nplk_quantize_rows, lib.nplk_quantize_cols):
        assert call(None, 4, 4, 0, P, 4, P, 16, ODD) == BAD
