"""Argument checks of the 4-bit and log-probability entry points: every refusal happens
before any device work, so no GPU is needed."""
import ctypes as C

import pytest

from support import nb

P = C.c_void_p(4096)  # never dereferenced: every call below fails its checks
ODD = C.c_void_p(4097)
BAD, UNSUP = nb.NPL_ERR_INVALID_ARG, nb.NPL_ERR_UNSUPPORTED
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return nb.load()


def quantize(lib, n=4, k=40, group=32, dtype=0, w=P, ldw=40, q=P, ldq=20, st=0, scale=P, lds=2,
             zero=P, ldz=2):
    return lib.nplk_quantize_w4(None, n, k, group, dtype, w, ldw, q, ldq, st, scale, lds, zero, ldz)


def product(lib, m=3, n=4, k=40, group=32, xt=0, x=P, ldx=40, q=P, ldq=20, st=0, scale=P, lds=2,
            zero=P, ldz=2, bias=P, act=0, ct=0, c=P, ldc=4, status=P):
    return lib.nplk_gemm_w4(None, m, n, k, group, xt, x, ldx, q, ldq, st, scale, lds, zero, ldz, bias,
                            act, 0.0, ct, c, ldc, status)


WEIGHTS = [dict(n=0), dict(n=-1), dict(k=0), dict(group=0), dict(group=-32), dict(q=None),
           dict(scale=None), dict(ldq=19), dict(lds=1), dict(ldz=1), dict(st=3), dict(st=-1),
           dict(scale=ODD), dict(st=1, scale=ODD), dict(scale=C.c_void_p(4098))]


@pytest.mark.parametrize("change", WEIGHTS + [dict(w=None), dict(ldw=39), dict(dtype=3), dict(w=ODD),
                                              dict(dtype=1, w=ODD)])
def test_quantizer_refuses(lib, change):
    assert quantize(lib, **change) == BAD


@pytest.mark.parametrize("change", WEIGHTS + [
    dict(m=0), dict(m=-2), dict(x=None), dict(c=None), dict(ldx=39), dict(ldc=3), dict(xt=3),
    dict(ct=-1), dict(act=11), dict(act=-1), dict(x=ODD), dict(c=ODD), dict(ct=2, c=ODD),
    dict(bias=ODD), dict(status=ODD)])
def test_product_refuses(lib, change):
    assert product(lib, **change) == BAD


@pytest.mark.parametrize("group", [1, 16, 33, 48, 96, 256, 1 << 33])
def test_other_groups_are_unsupported(lib, group):
    wide = dict(lds=BIG, ldz=BIG)
    assert quantize(lib, group=group, **wide) == UNSUP
    assert product(lib, group=group, **wide) == UNSUP


def test_too_large(lib):
    over = (1 << 30) + 1
    assert quantize(lib, n=over) == UNSUP
    assert quantize(lib, k=over, ldw=BIG, ldq=BIG, lds=BIG, ldz=BIG) == UNSUP
    assert product(lib, m=over) == UNSUP and product(lib, n=over, ldc=BIG) == UNSUP
    assert product(lib, k=over, ldx=BIG, ldq=BIG, lds=BIG, ldz=BIG) == UNSUP


def forward(lib, rows=3, vocab=10, dtype=0, x=P, ld=10, scale=1.0, targets=P, lp=P, ent=P, stats=P,
            top=2, ids=P, tlp=P):
    return lib.nplk_token_logprobs(None, rows, vocab, dtype, x, ld, scale, targets, lp, ent, stats, top,
                                   ids, tlp)


def backward(lib, rows=3, vocab=10, dtype=0, x=P, ld=10, scale=1.0, targets=P, stats=P, ent=P, g=P,
             h=P, dx=C.c_void_p(8192), ldd=10):
    return lib.nplk_token_logprobs_backward(None, rows, vocab, dtype, x, ld, scale, targets, stats, ent,
                                            g, h, dx, ldd)


ROWS = [dict(rows=0), dict(rows=-1), dict(vocab=0), dict(x=None), dict(ld=9), dict(dtype=3),
        dict(dtype=-1), dict(x=ODD), dict(dtype=2, x=ODD), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=float("nan")), dict(scale=float("inf")), dict(targets=C.c_void_p(4100)),
        dict(targets=None), dict(stats=ODD), dict(ent=ODD)]


@pytest.mark.parametrize("change", ROWS + [
    dict(top=-1), dict(ids=None), dict(tlp=None), dict(lp=ODD), dict(tlp=ODD),
    dict(ids=C.c_void_p(4100)), dict(lp=None, ent=None, stats=None, top=0)])
def test_forward_refuses(lib, change):
    assert forward(lib, **change) == BAD


@pytest.mark.parametrize("change", ROWS + [
    dict(stats=None), dict(dx=None), dict(ldd=9), dict(g=None, h=None), dict(ent=None),
    dict(g=ODD), dict(h=ODD), dict(dx=ODD), dict(dx=P, ldd=11)])
def test_backward_refuses(lib, change):
    assert backward(lib, **change) == BAD


def test_too_many_alternatives_or_tokens(lib):
    assert forward(lib, top=33) == UNSUP
    assert forward(lib, vocab=1 << 31, ld=1 << 31) == UNSUP
    assert backward(lib, vocab=1 << 31, ld=1 << 31, ldd=1 << 31) == UNSUP


@pytest.mark.parametrize("scale", [2.0 ** 126 * 1.001, 3.4e38])
def test_scales_whose_exponents_would_not_be_numbers(lib, scale):
    assert forward(lib, scale=scale) == BAD and backward(lib, scale=scale) == BAD
