"""Log probabilities at the limits of what the header allows, in every form of the kernel:
one warp, four and sixteen warps a row, a row over a cluster."""
import pytest
import torch

import support as S
from test_gpu_token_logprobs import (INF, NAN, TYPES, U, backward, check_backward, check_forward, f32,
                                     forward, gen, logits)

pytestmark = pytest.mark.gpu

FORMS = [(7, 9), (7, 1003), (600, 3001), (7, 12001), (7, 40001), (320, 20001)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_both_stats_of_a_row_with_a_nan_or_infinity(rows, vocab, dtype):
    lib = S.gpu_lib()
    x = logits(rows, vocab, dtype)
    clean = x.clone()
    x[1, 0] = NAN
    x[2, vocab - 1] = INF
    x[3] = NAN
    x[4, vocab // 2], x[4, 0] = INF, -INF
    x[5] = -INF
    x[5, 1] = NAN
    bad = slice(1, 6)
    t = torch.zeros(rows, device="cuda", dtype=torch.int64)
    lp, ent, st, ids, tlp = forward(lib, x, vocab, t, 3)
    assert st[bad].isnan().all() and lp[bad].isnan().all() and ent[bad].isnan().all()
    assert (ids[bad] == -1).all() and tlp[bad].isnan().all()
    want = forward(lib, clean, vocab, t, 3)
    for a, b in zip((lp, ent, st, ids, tlp), want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[6:], b[6:])
    # a row without a token has log probability 0, whatever it holds
    t[1:4] = torch.tensor([-100, vocab, -1], device="cuda")
    lp, ent, st, _, _ = forward(lib, x, vocab, t, 0)
    assert (lp[1:4] == 0).all() and lp[4:6].isnan().all() and st[bad].isnan().all()
    g = torch.ones(rows, device="cuda")
    dx = backward(lib, x, vocab, t, st, None, g, None)
    assert (dx[1:4] == 0).all() and dx[4:6].isnan().all()
    dx = backward(lib, x, vocab, t, st, ent, g, g)
    assert dx[bad].isnan().all() and torch.isfinite(dx[0]).all() and torch.isfinite(dx[6:]).all()


# 2.5e-37: the lowest finite number times such a scale is an exponent of some -100
SMALL = [1e-30, 2.5e-37, 3e-39, 1e-44]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", SMALL)
def test_masks_under_the_smallest_scales(rows, vocab, dtype, scale):
    # all of a row's logits that are left are alike: log n, wherever in the row they lie
    lib, x = S.gpu_lib(), logits(rows, vocab, dtype)
    x[0] = -INF
    x[1, ::2] = -INF
    x[2, 1::2] = -INF
    x[3, :-1] = -INF  # one left
    x[4, 1:] = -INF
    x[5, :vocab // 2] = -INF
    x[6] = x[6].abs().neg()  # none above 0
    x[6, -1] = -INF
    t = torch.full((rows,), vocab - 1, device="cuda")
    left = x != -INF
    n = left.sum(1).double()
    lp, ent, st, ids, tlp = forward(lib, x, vocab, t, 3, scale)
    assert lp[0] == -INF and ent[0] == 0 and (st[0] == -INF).all()
    assert (ids[0] == -1).all() and (tlp[0] == -INF).all()
    log_n = n[1:].log()
    # scale |d| is below 1e-28; the sum of n terms is off by (n / 512 + 64) 2^-24 at most, relative
    tol = (vocab / 512 + 66) * U * (1 + log_n)
    has = left[1:, -1]
    assert ((lp[1:].double() + log_n).abs() <= tol)[has].all() and (lp[1:][~has] == -INF).all()
    assert ((ent[1:].double() - log_n).abs() <= tol).all()
    assert ((st[1:, 1].double() - log_n).abs() <= tol).all()
    assert torch.equal(st[1:, 0].double(), x[1:].double().amax(1))
    g = torch.full((rows,), 2.0 ** 90, device="cuda")
    dx = backward(lib, x, vocab, t, st, ent, g, g, scale)
    assert torch.isfinite(dx).all()
    hit = torch.zeros_like(left)
    hit[:, -1] = True
    assert (dx[0] == 0).all() and (dx[~left & ~hit] == 0).all()
    check_backward(x[1:], vocab, t[1:], st[1:], ent[1:], g[1:], g[1:], scale, dx[1:])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1.0, 0.3] + SMALL)
def test_distances_beyond_fp32(rows, vocab, dtype, scale):
    # l - m down to -6e38, in every place of a row; scale (l - m) may be small all the same
    lib, x = S.gpu_lib(), logits(rows, vocab, dtype)
    far = torch.arange(vocab, device="cuda") % 3 == 1
    far[0] = far[-1] = True
    x[:, far] = -3e38
    x[:, vocab // 3] = 3e38
    t = torch.full((rows,), vocab - 1, device="cuda")
    t[::2] = vocab // 2
    got = forward(lib, x, vocab, t, 2, scale)
    check_forward(x, vocab, t, scale, got, 2)
    g = torch.ones(rows, device="cuda")
    dx = backward(lib, x, vocab, t, got[2], got[1], g, g, scale)
    check_backward(x, vocab, t, got[2], got[1], g, g, scale, dx)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1e30, 1e36, 2.0 ** 126])
def test_gradient_under_the_largest_scales(rows, vocab, dtype, scale):
    # p is 0 but for the largest logits: a gradient of 0 there, however large g and h times the
    # scale and the exponent
    lib = S.gpu_lib()
    x = torch.randint(-50, 50, (rows, vocab), device="cuda", generator=gen(6)).to(TYPES[dtype][0])
    x[:, 2] = 60.0
    x[::3, vocab - 1] = 60.0       # two of them
    x[1] = 1.0                     # all
    x[:, 4] = -INF
    x[5, 5:] = -INF
    t = torch.full((rows,), 2, device="cuda")
    t[::2] = 3
    g = torch.rand(rows, device="cuda", generator=gen(1)) * 6 - 3
    h = torch.rand(rows, device="cuda", generator=gen(2)) * 6 - 3
    _, ent, st, _, _ = forward(lib, x, vocab, t, 0, scale)
    for gg, hh in ((g, None), (None, h), (g, h)):
        dx = backward(lib, x, vocab, t, st, ent if hh is not None else None, gg, hh, scale)
        assert torch.isfinite(dx).all()
        check_backward(x, vocab, t, st, ent, gg, hh, scale, dx)
    # all of p on the token: nothing left to change, also where scale g leaves fp32
    sure = torch.arange(rows, device="cuda") % 6 == 5
    dx = backward(lib, x, vocab, t, st, None, torch.full_like(g, 1e4), None, scale)
    assert (dx[sure] == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1.0, 1 / 0.7, 2.0])
def test_the_gradient_of_a_masked_logit_is_zero(rows, vocab, dtype, scale):
    lib, x = S.gpu_lib(), logits(rows, vocab, dtype)
    x[0, ::2] = -INF
    x[1, 1::2] = -INF
    x[2, 3:] = -INF
    x[3, :-2] = -INF
    x[4, vocab // 3:vocab // 2] = -INF
    x[5, 1:] = -INF
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(5))
    t[0], t[1], t[5] = 0, 0, vocab - 1  # a masked token, one that is left, a masked one
    _, ent, st, _, _ = forward(lib, x, vocab, t, 0, scale)
    g = torch.randn(rows, device="cuda", generator=gen(1))
    h = torch.randn(rows, device="cuda", generator=gen(2))
    masked = x == -INF
    at = torch.arange(rows, device="cuda")
    masked[at, t] = False
    assert masked[:6].any(1).all()
    for gg, hh in ((g, None), (None, h), (g, h)):
        dx = backward(lib, x, vocab, t, st, ent if hh is not None else None, gg, hh, scale)
        assert (dx[masked] == 0).all()
        # the masked tokens' own: scale g, rounded in fp32 and to the type
        for r in (0, 5):
            want = f32(scale) * gg[r].double() if gg is not None else torch.zeros((), device="cuda")
            assert abs(dx[r, t[r]] - want) <= (U + torch.finfo(x.dtype).eps) * abs(want)
