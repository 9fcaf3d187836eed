"""Group norm with an activation (channels last) and its gradient against a
plain implementation in 64 bits.

Tolerances count roundings of 2^-24 in the fp32 arithmetic and one half step of
the output's type. For a sum of M values spread over at least 256 threads the
longest chain of additions is taken as L = M / 256 + 16."""
import ctypes as C

import pytest
import torch

import support as S
from support import nb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"fp32": nb.NPLK_DTYPE_FP32, "fp16": nb.NPLK_DTYPE_FP16, "bf16": nb.NPLK_DTYPE_BF16}


def act64(z, act, alpha=0.1):
    if act == 1:
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == 2:
        return z.clamp(0, 6)
    if act == 3:
        return torch.tanh(z)
    if act == 4:
        return torch.sigmoid(z)
    if act == 5:
        return 0.5 * z * (1 + torch.tanh(0.7978845608 * (z + 0.044715 * z ** 3)))
    if act == 6:
        return z * torch.sigmoid(z)
    if act == 7:
        return torch.where(z > 0, z, alpha * z)
    if act == 8:
        return torch.where(z > 0, z, torch.expm1(z))
    if act == 9:
        return 1.05070098 * torch.where(z > 0, z, 1.67326324 * torch.expm1(z))
    if act == 10:
        return torch.log1p(torch.exp(z))
    return z


def norm64(x, groups, gamma, beta, eps):
    n, hw, c = x.shape
    v = x.double().view(n, hw, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    rstd = ((v - mean).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    return ((v - mean) * rstd).view(n, hw, c), mean.view(n, groups), rstd.view(n, groups)


def inputs(n, hw, c, dtype, seed=0, ld=None, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * hw + c)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    wide = torch.full((n, hw, ld or c), 77.0, device="cuda", dtype=TYPES[dtype])
    wide[..., :c] = (randn(n, hw, c) * (0.5 + randn(c).abs()) + randn(c) + shift).to(TYPES[dtype])
    dy = torch.full((n, hw, ld or c), 55.0, device="cuda", dtype=TYPES[dtype])
    dy[..., :c] = randn(n, hw, c).to(TYPES[dtype])
    return wide, dy, 1 + 0.2 * randn(c), 0.2 * randn(c)


def workspace(lib, n, hw, c, groups):
    size = lib.nplk_group_norm_workspace_size(n, hw, c, groups)
    assert size > 0
    return torch.empty(size, device="cuda", dtype=torch.uint8), size


def forward(lib, x, c, groups, gamma, beta, act=0, eps=1e-5, y=None, alpha=0.1, work=None,
            stats=True):
    n, hw, ld = x.shape
    y = torch.full_like(x, 99.0) if y is None else y
    mean = torch.full((n, groups), 9.0, device=x.device) if stats else None
    rstd = torch.full((n, groups), 9.0, device=x.device) if stats else None
    work, size = work or workspace(lib, n, hw, c, groups)
    code = {v: CODES[k] for k, v in TYPES.items()}[x.dtype]
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = lib.nplk_group_norm_act(S.cuda_stream(), n, hw, c, groups, code, p(x), ld, p(gamma),
                                 p(beta), eps, act, alpha, p(y), y.shape[2], p(mean), p(rstd),
                                 p(work), size)
    assert rc == 0
    return y, mean, rstd


def backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=0, dx=None, alpha=0.1,
             want=(True, True), work=None):
    n, hw, ld = x.shape
    dx = torch.full_like(x, 99.0) if dx is None else dx
    dg = torch.full((c,), 9.0, device=x.device) if want[0] else None
    db = torch.full((c,), 9.0, device=x.device) if want[1] else None
    work, size = work or workspace(lib, n, hw, c, groups)
    code = {v: CODES[k] for k, v in TYPES.items()}[x.dtype]
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = lib.nplk_group_norm_act_backward(S.cuda_stream(), n, hw, c, groups, code, p(dy),
                                          dy.shape[2], p(x), ld, p(mean), p(rstd), p(gamma),
                                          p(beta), act, alpha, p(dx), dx.shape[2], p(dg), p(db),
                                          p(work), size)
    assert rc == 0
    return dx, dg, db


def per_channel(v, c):
    """[n, groups] to [n, 1, c]."""
    return v.repeat_interleave(c // v.shape[1], 1)[:, None, :]


def check_forward(x, c, groups, gamma, beta, act, eps, y, mean, rstd):
    xs = x[..., :c]
    n, hw, _ = xs.shape
    xh, m64, r64 = norm64(xs, groups, gamma, beta, eps)
    ga = torch.ones(c, device=x.device) if gamma is None else gamma
    be = torch.zeros(c, device=x.device) if beta is None else beta
    z = xh * ga.double() + be.double()
    ref = act64(z, act)
    L = hw * c // groups / 256 + 16
    top = xs.double().abs().view(n, hw, groups, -1).amax((1, 3))
    # the mean: L additions of values up to `top`
    assert ((mean.double() - m64).abs() <= L * U * top).all()
    # rstd: the variance's L additions of squares and a mean L * U * top off,
    # halved by the square root, and four roundings
    off = (L * U + (L * U * top * r64) ** 2 + 8 * U) * r64
    assert ((rstd.double() - r64).abs() <= off).all()
    # z: the mean's and rstd's errors, and its own roundings; act' <= 1.13 (1.8 for
    # SELU), and the activation's own error of a few steps of |z| + 1
    ez = ga.abs().double() * (per_channel(r64 * L * U * top, c) + xh.abs() * (L + 8) * U)
    ez = ez + 8 * U * (z.abs() + be.abs().double())
    tol = 1.8 * ez + 24 * U * (z.abs() + 1) + torch.finfo(x.dtype).eps / 2 * ref.abs()
    if x.dtype != torch.float32:
        tol = tol * (1 + torch.finfo(x.dtype).eps) + 2.0 ** -25  # and fp16's denormal step
    err = (y[..., :c].double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert y.shape[2] == c or (y[..., c:] == 99.0).all()


def grad64(xs, dys, groups, mean, rstd, gamma, beta, act):
    """dx, dgamma, dbeta by the formula, and what bounds their rounding errors."""
    n, hw, c = xs.shape
    m, r = per_channel(mean.double(), c), per_channel(rstd.double(), c)
    xh = (xs.double() - m) * r
    z = (xh * gamma.double() + beta.double()).requires_grad_()
    slope, = torch.autograd.grad(act64(z, act).sum(), z)
    dz = dys.double() * slope
    dh = dz * gamma.double()
    total = lambda v: per_channel(v.view(n, hw, groups, -1).mean((1, 3)), c)  # noqa: E731
    dx = r * (dh - total(dh) - xh * total(dh * xh))
    return dict(dx=dx, dg=(dz * xh).sum((0, 1)), db=dz.sum((0, 1)), r=r, xh=xh, z=z.detach(),
                total=total)


def check_backward(x, dy, c, groups, mean, rstd, gamma, beta, act, dx, dg, db):
    xs, dys = x[..., :c], dy[..., :c]
    n, hw, _ = xs.shape
    f = grad64(xs, dys, groups, mean, rstd, gamma, beta, act)
    if act in (1, 2, 7):  # a value on the bend would make the slope a matter of rounding
        assert f["z"].abs().min() > 2e-6 and (f["z"] - 6).abs().min() > 2e-6
    L, ga = hw * c // groups / 256 + 16, gamma.abs().double()
    # dz: slopes are at most 1.8 and change by at most 1.8 * the error of z, whose
    # parts (x - mean, * rstd, * gamma, + beta) round four times; the slope's own
    # formula rounds a few steps of 1 + |z|
    ez = 8 * U * (f["z"].abs() + f["xh"].abs() * ga + beta.abs().double()
                  + per_channel(mean.double().abs() * rstd, c) * ga)
    edz = dys.double().abs() * (1.8 * ez + 24 * U * (1 + f["z"].abs()))
    size = 1.8 * dys.double().abs()
    exh = 4 * U * (f["xh"].abs() + per_channel(mean.double().abs() * rstd, c))
    e_b = edz * f["xh"].abs() + size * exh
    tol_dx = f["r"] * (ga * edz + 8 * U * ga * size
                       + f["total"](ga * (edz + (L + 8) * U * size))
                       + f["xh"].abs() * f["total"](ga * (e_b + (L + 8) * U * size * f["xh"].abs()))
                       + exh * f["total"](ga * size * f["xh"].abs()))
    tol_dx = tol_dx + torch.finfo(x.dtype).eps / 2 * (f["dx"].abs() + tol_dx)
    if x.dtype == torch.float16:
        tol_dx = tol_dx + 2.0 ** -25
    err = (dx[..., :c].double() - f["dx"]).abs()
    assert (err <= tol_dx).all(), float((err / tol_dx).max())
    Lc = n * hw / 8 + 64  # a channel's sum: its longest chain of additions
    if dg is not None:
        tol = (e_b + Lc * U * size * f["xh"].abs()).sum((0, 1))
        assert ((dg.double() - f["dg"]).abs() <= tol).all()
    if db is not None:
        tol = (edz + Lc * U * size).sum((0, 1))
        assert ((db.double() - f["db"]).abs() <= tol).all()
    assert dx.shape[2] == c or (dx[..., c:] == 99.0).all()


# n, hw, c, groups: one value a group, one pixel, odd channels, groups that end
# inside a 16-byte piece, one group, as many groups as channels, wide groups,
# long planes, many images, groups wider than a block
SHAPES = [(1, 1, 1, 1), (1, 1, 32, 32), (2, 1, 64, 4), (3, 7, 510, 30), (2, 64, 320, 32),
          (1, 64, 1280, 32), (2, 33, 30, 30), (1, 1000, 8, 1), (2, 257, 24, 2), (5, 100, 36, 3),
          (1, 4099, 320, 32), (1, 20000, 128, 32), (300, 3, 16, 2), (1, 5, 8192, 1),
          (1, 9, 4098, 2), (2, 1500, 2560, 32), (1, 70000, 130, 10), (1, 40000, 512, 1),
          (3, 16400, 256, 32)]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,hw,c,groups", SHAPES)
def test_forward_shapes(n, hw, c, groups, dtype):
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(n, hw, c, dtype)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    check_forward(x, c, groups, gamma, beta, 6, 1e-5, y, mean, rstd)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,hw,c,groups", [s for s in SHAPES if s[1] * s[2] // s[3] >= 4])
def test_backward_shapes(n, hw, c, groups, dtype):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(n, hw, c, dtype)
    _, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    dx, dg, db = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6)
    check_backward(x, dy, c, groups, mean, rstd, gamma, beta, 6, dx, dg, db)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", range(11))
def test_every_activation(act, dtype):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(2, 50, 48, dtype, seed=3)
    y, mean, rstd = forward(lib, x, 48, 6, gamma, beta, act=act)
    check_forward(x, 48, 6, gamma, beta, act, 1e-5, y, mean, rstd)
    dx, dg, db = backward(lib, dy, x, 48, 6, mean, rstd, gamma, beta, act=act)
    check_backward(x, dy, 48, 6, mean, rstd, gamma, beta, act, dx, dg, db)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", [5, 6])
def test_gelu_and_swish_far_from_zero(act, dtype):
    # the value and the slope tend to 0 and 0 on the left, to z and 1 on the right
    lib = S.gpu_lib()
    far = [7.0, 30.0, 45.0, 100.0, 1e4, 1e12, 1e19, 1e30]
    beta = torch.tensor(far + [-v for v in far], device="cuda")
    x, _, _, _ = inputs(2, 300, 16, dtype)
    gamma = torch.ones(16, device="cuda")
    y, mean, rstd = forward(lib, x, 16, 4, gamma, beta, act)
    xh, _, _ = norm64(x, 4, gamma, beta, 1e-5)
    z = xh + beta.double()
    want = act64(z, act)
    # a few roundings of z, where it is above -30; below, nothing of it is left
    half = torch.finfo(TYPES[dtype]).eps / 2
    assert ((y.double() - want).abs() <= want.abs() * half + z.abs().clamp(max=1e32) *
            (z > -30) * 16 * U + 1e-11).all()
    dx, dg, db = backward(lib, torch.ones_like(x), x, 16, 4, mean, rstd, gamma, beta, act)
    assert torch.isfinite(dx).all() and torch.isfinite(dg).all()
    slope = (beta > 0).double()
    near = beta.abs() < 20  # slopes there are not yet 0 or 1
    assert ((db.double() / 600 - slope).abs()[~near] <= 1e-6).all()


@pytest.mark.parametrize("dtype,c,ld", [("fp32", 24, 40), ("bf16", 40, 41), ("fp16", 48, 64),
                                        ("bf16", 60, 62), ("fp16", 20, 24), ("fp32", 6, 7)])
@pytest.mark.parametrize("hw", [10, 9000])
def test_channel_slices_and_offsets(dtype, c, ld, hw):
    # x, y, dy and dx are channel slices of wider tensors, at odd pitches and
    # one element past an aligned address
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(2, hw, c, dtype, ld=ld)
    for skip in (0, 1):
        move = lambda t: torch.cat([t.new_zeros(skip), t.reshape(-1)])[skip:].view(t.shape)  # noqa: E731
        xs, dys, out = move(x), move(dy), move(torch.full_like(x, 99.0))
        y, mean, rstd = forward(lib, xs, c, 2, gamma, beta, act=5, y=out)
        check_forward(xs, c, 2, gamma, beta, 5, 1e-5, y, mean, rstd)
        out = move(torch.full_like(x, 99.0))
        dx, dg, db = backward(lib, dys, xs, c, 2, mean, rstd, gamma, beta, act=5, dx=out)
        check_backward(xs, dys, c, 2, mean, rstd, gamma, beta, 5, dx, dg, db)


@pytest.mark.parametrize("hw", [40, 30000])
def test_optional_arguments_and_in_place(hw):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(2, hw, 64, "bf16")
    one, zero = torch.ones_like(gamma), torch.zeros_like(beta)
    full = forward(lib, x, 64, 8, one, zero, act=6)
    bare, _, _ = forward(lib, x, 64, 8, None, None, act=6, stats=False)
    assert torch.equal(full[0], bare)
    y, mean, rstd = forward(lib, x, 64, 8, gamma, beta, act=6)
    dx, dg, db = backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6)
    again = backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6)
    assert all(torch.equal(a, b) for a, b in zip((dx, dg, db), again))  # a fixed order of sums
    d1, only_g, none = backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6,
                                want=(True, False))
    assert none is None and torch.equal(only_g, dg) and torch.equal(d1, dx)
    d2, none, only_b = backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6,
                                want=(False, True))
    assert none is None and torch.equal(only_b, db) and torch.equal(d2, dx)
    d3, _, _ = backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6, want=(False, False))
    assert torch.equal(d3, dx)
    in_dy, in_x = dy.clone(), x.clone()
    backward(lib, in_dy, x, 64, 8, mean, rstd, gamma, beta, act=6, dx=in_dy)
    assert torch.equal(in_dy, dx)
    backward(lib, dy, in_x, 64, 8, mean, rstd, gamma, beta, act=6, dx=in_x)
    assert torch.equal(in_x, dx)
    xi = x.clone()
    forward(lib, xi, 64, 8, gamma, beta, act=6, y=xi)
    assert torch.equal(xi, y)


@pytest.mark.parametrize("hw", [64, 50000])
def test_large_mean_and_outlier(hw):
    # means thousands of deviations from zero, and a first value far from the
    # rest: a one-pass sum of squares would lose the variance
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(2, hw, 32, "fp32", shift=4000.0)
    x[0, 0, :] = -3.0e4
    y, mean, rstd = forward(lib, x, 32, 4, gamma, beta)
    check_forward(x, 32, 4, gamma, beta, 0, 1e-5, y, mean, rstd)


@pytest.mark.parametrize("hw", [3, 200, 60000])
def test_non_finite_values_stay_in_their_group(hw):
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(2, hw, 32, "fp32")
    clean, _, _ = forward(lib, x, 32, 4, gamma, beta, act=6)
    x[0, hw // 2, 9] = float("nan")
    x[1, hw - 1, 31] = float("inf")
    y, mean, rstd = forward(lib, x, 32, 4, gamma, beta, act=6)
    bad = torch.zeros(2, hw, 32, dtype=torch.bool, device="cuda")
    bad[0, :, 8:16] = True
    bad[1, :, 24:] = True
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("act", [0, 1, 5, 6])
@pytest.mark.parametrize("dtype,c,groups", [("bf16", 36, 6), ("fp16", 35, 7), ("bf16", 320, 32),
                                            ("fp32", 33, 11)])
@pytest.mark.parametrize("hw", [3, 60000])
def test_non_finite_values_beside_groups_that_share_a_piece(hw, dtype, c, groups, act):
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(2, hw, c, dtype)
    clean, _, _ = forward(lib, x, c, groups, gamma, beta, act)
    cg = c // groups
    x[0, hw - 1, 2 * cg - 1], x[1, 0, 3 * cg] = float("nan"), float("-inf")
    y, _, _ = forward(lib, x, c, groups, gamma, beta, act)
    hit = torch.zeros(2, groups, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[1, 3] = True
    hit = per_channel(hit, c).expand_as(y)
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("act", [0, 1, 5, 6])
@pytest.mark.parametrize("hw", [3, 200, 60000])
def test_non_finite_gradients_stay_in_their_group(hw, act):
    lib = S.gpu_lib()
    for dtype, c, groups in (("fp32", 30, 10), ("bf16", 36, 6), ("bf16", 320, 32)):
        cg = c // groups
        x, dy, gamma, beta = inputs(2, hw, c, dtype)
        _, mean, rstd = forward(lib, x, c, groups, gamma, beta, act)
        clean = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act)
        dy[0, hw // 2, cg + 1], dy[1, 0, 4 * cg] = float("nan"), float("inf")
        x[1, hw - 1, 3 * cg - 1] = float("nan")
        dx, dg, db = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act)
        hit = torch.zeros(2, groups, dtype=torch.bool, device="cuda")
        hit[0, 1] = hit[1, 4] = hit[1, 2] = True
        reached = per_channel(hit, c).expand_as(dx)
        # ReLU's zero slope makes the infinity a NaN or keeps it: not finite either way
        assert torch.equal(dx[~reached], clean[0][~reached])
        where = (cg + 1, 3 * cg - 1, 4 * cg)
        other = torch.ones(c, dtype=torch.bool, device="cuda")
        other[list(where)] = False
        assert torch.equal(dg[other], clean[1][other]) and torch.equal(db[other], clean[2][other])
        assert torch.isnan(dx[0, :, cg:2 * cg]).all() and torch.isnan(db[cg + 1])
        if act:  # z is NaN there, and its slope with it, but ReLU's, which is 0
            assert torch.isnan(dg[3 * cg - 1])
        if hw > 3:
            assert not torch.isfinite(db[4 * cg])


def test_constant_groups_give_beta():
    lib = S.gpu_lib()
    x = torch.full((2, 77, 12), 3.25, device="cuda")
    beta = torch.arange(12.0, device="cuda")
    y, mean, rstd = forward(lib, x, 12, 3, None, beta)
    assert torch.equal(y, beta.expand_as(y)) and (mean == 3.25).all()


@pytest.mark.parametrize("hw", [30, 20000])
def test_gradient_against_differences(hw):
    # (f(x + h d) - f(x - h d)) / 2h of the forward kernel, f = sum dy * y. The
    # definition's own difference in 64 bits has the same remainder, and its
    # distance from the gradient shows that remainder (h^2 times a constant).
    lib = S.gpu_lib()
    c, groups, h = 24, 4, 2.0 ** -6
    x, dy, gamma, beta = inputs(1, hw, c, "fp32", seed=11)
    d = torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=5)
    dx, _, _ = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=5)

    def exact(v):
        xh, _, _ = norm64(v, groups, gamma, beta, 1e-5)
        return (dy.double() * act64(xh * gamma.double() + beta.double(), 5)).sum()

    kernel = [(dy.double() * forward(lib, v, c, groups, gamma, beta, act=5)[0].double()).sum()
              for v in (x + h * d, x - h * d)]
    whole = [exact(v) for v in (x + h * d, x - h * d)]
    by_kernel, by_exact = [(p[0] - p[1]) / (2 * h) for p in (kernel, whole)]
    # each y is within 64 U of 4 (|y| <= 4, act' <= 1.13); errors of both signs
    # add like a random walk, taken eight deep
    noise = 8 * 64 * U * 4 * dy.double().norm() / h
    assert (by_kernel - by_exact).abs() <= noise
    slope = (dx.double() * d.double()).sum()
    half = [exact(v) for v in (x.double() + h / 2 * d, x.double() - h / 2 * d)]
    finer = (half[0] - half[1]) / h
    # halving h takes away 3/4 of the remainder: the finer one's is a third of the change
    remainder = (finer - by_exact).abs()
    assert (finer - slope).abs() <= remainder + 1e-4 * slope.abs() + 64 * U * hw ** 0.5 * 8


def test_other_stream_and_two_calls_at_once():
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(2, 9000, 64, "bf16")
    want, _, _ = forward(lib, x, 64, 8, gamma, beta, act=6)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(forward(lib, x, 64, 8, gamma, beta, act=6)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("hw", [60, 30000])
def test_captured_and_replayed(hw):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(2, hw, 64, "bf16")
    work = workspace(lib, 2, hw, 64, 8)
    y, dx = torch.empty_like(x), torch.empty_like(x)

    def step():
        _, mean, rstd = forward(lib, x, 64, 8, gamma, beta, act=6, y=y, work=work)
        return backward(lib, dy, x, 64, 8, mean, rstd, gamma, beta, act=6, dx=dx, work=work)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, dg, db = step()
    x.copy_(inputs(2, hw, 64, "bf16", seed=9)[0])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y, dx, dg, db)]
    _, dg2, db2 = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (y, dx, dg2, db2)))
