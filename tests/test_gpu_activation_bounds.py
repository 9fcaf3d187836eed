"""GELU and swish of the residual-block operators in fp32, at arguments that are known
exactly, against the formulas in 64 bits.

With U = 2^-24: the exponential's argument rounds by 1.5 U of itself (swish) or 4 U
(GELU), the exponential by 4 U, its sum, reciprocal and product by 3.5 U together. Since
|z| s (1 - s) <= 0.23, z^2 s (1 - s) <= 0.45 and x 2u s (1 - s) <= 0.45 for the sigmoid s,
a value is off by at most U (3.4 + 3.5 |y|), with one reciprocal for two values 2 U |y|
more: below the documented 2^-21 (1 + |y|). Where the formula tends to 0 the value stays
within 4e-17 of it.

A slope s + z s (1 - s) u': s is off by s (1 - s) (4 U + 4 U |2u|) + 2.5 U, which (1 + |z u'|)
multiplies: the first part adds up to 20 U at most, the second ends at z = 17 (s is 1 in
fp32 from there on; GELU's 2u is 17 at z = 4.6, where u' is 3.1 and z u' 14): 2.5 (1 + 17) U
= 45 U; below the documented 2^-17 = 128 U."""
import pytest
import torch

import support as S

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def points():
    near = torch.linspace(-12, 12, 2401, dtype=torch.float64)
    wide = torch.linspace(-120, 120, 1603, dtype=torch.float64)
    far = torch.tensor([v * s for v in (150.0, 1e4, 1e12, 1e19, 1e30) for s in (1, -1)]).double()
    return torch.cat([near, wide, far, torch.zeros(2).double()]).float().cuda()  # 4016


def act64(z, act):
    z = z.double()
    if act == 6:
        return z * torch.sigmoid(z)
    u2 = 2 * 0.7978845608 * (z + 0.044715 * z ** 3)  # 0.5 z (1 + tanh u) = z sigmoid(2 u)
    return z * torch.sigmoid(u2)


def check_values(got, z, act):
    want = act64(z, act)
    err = (got.double() - want).abs()
    assert (err <= 2.0 ** -21 * (1 + want.abs())).all(), float((err / (1 + want.abs())).max() / U)
    gone = z < (-41.5 if act == 6 else -7.4)
    assert (err[gone.expand_as(err)] <= 4e-17).all()


@pytest.mark.parametrize("act", [5, 6])
@pytest.mark.parametrize("m,k,pitch", [(1, 64, 64), (12, 64, 64), (40, 512, 512), (40, 64, 64),
                                       (1021, 64, 64), (5, 64, 65)])
def test_product_epilogues(m, k, pitch, act):
    # sums of zero: the bias is the argument
    lib, z = S.gpu_lib(), points()
    n = z.numel()
    a, b = torch.zeros(m, pitch, device="cuda", dtype=torch.int8), torch.ones(
        n, pitch, device="cuda", dtype=torch.int8)
    one = torch.ones(max(m, n), device="cuda")
    c = torch.full((m, n), 99.0, device="cuda")
    assert lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, a.data_ptr(), pitch, one.data_ptr(),
                            b.data_ptr(), pitch, one.data_ptr(), z.data_ptr(), act, 0.0, 0,
                            c.data_ptr(), n, None) == 0
    check_values(c, z, act)


@pytest.mark.parametrize("act", [5, 6])
@pytest.mark.parametrize("hw", [1, 40, 9000])
@pytest.mark.parametrize("odd", [False, True])
def test_group_norm_of_zeros(hw, act, odd):
    # x = 0: beta is the argument; and one pixel's dbeta its slope
    lib, z = S.gpu_lib(), points()
    z = z[:-1] if odd else z
    c = z.numel()
    groups = c // 8 if not odd else c // 5
    assert c % groups == 0
    x = torch.zeros(1, hw, c, device="cuda")
    y, dx, dy = torch.full_like(x, 99.0), torch.empty_like(x), torch.zeros_like(x)
    dy[0, hw // 2] = 1.0
    gamma = torch.ones(c, device="cuda")
    mean, rstd = torch.empty(1, groups, device="cuda"), torch.empty(1, groups, device="cuda")
    dg, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    size = lib.nplk_group_norm_workspace_size(1, hw, c, groups)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)
    s = S.cuda_stream()
    assert lib.nplk_group_norm_act(s, 1, hw, c, groups, 0, x.data_ptr(), c, gamma.data_ptr(),
                                   z.data_ptr(), 1e-5, act, 0.0, y.data_ptr(), c,
                                   mean.data_ptr(), rstd.data_ptr(), work.data_ptr(), size) == 0
    check_values(y[0], z, act)
    assert lib.nplk_group_norm_act_backward(s, 1, hw, c, groups, 0, dy.data_ptr(), c,
                                            x.data_ptr(), c, mean.data_ptr(), rstd.data_ptr(),
                                            gamma.data_ptr(), z.data_ptr(), act, 0.0,
                                            dx.data_ptr(), c, dg.data_ptr(), db.data_ptr(),
                                            work.data_ptr(), size) == 0
    near = z.double().clamp(-200, 200).requires_grad_()  # 0 or 1 beyond, in 64 bits too
    slope, = torch.autograd.grad(act64(near, act).sum(), near)
    err = (db.double() - slope).abs()
    assert (err <= 2.0 ** -17).all(), float(err.max() / U)
