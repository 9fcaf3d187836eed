"""The sums of group norm where a careless one loses them: means thousands of
deviations from zero on planes of every form, outliers, and long sums of the gradient,
against 64 bits.

Bounds. A mean is formed by batches of up to four values, joined along a thread's
batches, then over a pack's channels, row lanes, warps, CTAs and chunks. Joining a batch
to the running mean of J batches rounds that mean once and weighs down what was rounded
before, so J / 2 such roundings stay; J is at most 12 at the sizes below (112 KB of rows
for 256 threads, or 226 rows on 7 lanes). The difference that is joined, of 2 `top` at
most, rounds three times with its weight, and the weights of all joins add up to one: 6
more for a chain. In roundings of `top`, with U = 2^-24:
  batch 4; chain of batches 6 + 6; pack (7 additions, a reciprocal of 2, a product) 10;
  a lane's entries 4 + 6; a warp (product, 5 additions, reciprocal, product) 9; warps of
  a group 9; cluster 7; chunks 2 + 6, twice 9: 93, taken as K = 96.
So |mean - mean64| <= K U top =: D.

M2 adds up squares of differences, at each of these seven steps, of means that are D at
most from their values' own, by the last step; with what had been rounded by each step (4,
16, 26, 36, 54, 61, 87) the root of the sum of the squares of twice these is 257 roundings,
below 3 K. By the triangle inequality of the root mean square the deviation s is then
within 3 D of the true one, besides K relative roundings of sums and weights:
|s - s64| <= 3 D + K U s. A sum of squares about zero would lose U top^2 of the variance
instead."""
import pytest
import torch

import support as S
from test_gpu_group_norm import U, backward, forward, grad64, inputs, norm64, per_channel

pytestmark = pytest.mark.gpu

K, EPS = 96, 1e-5


def bounds(x, groups):
    n, hw, c = x.shape
    _, mean, rstd = norm64(x, groups, None, None, EPS)
    top = x.double().abs().view(n, hw, groups, -1).amax((1, 3))
    off = K * U * top
    # rstd = 1 / sqrt(s^2 + eps): s off by a share a of 1 / rstd moves it by a / (1 - a) at
    # most, and it rounds four times itself
    a = (3 * off + K * U / rstd) * rstd
    assert (a < 0.5).all()
    return mean, rstd, off, a * (1 + 2 * a) + 4 * U


def check(x, groups, gamma, beta, y, mean, rstd):
    c = x.shape[2]
    m64, r64, off, rel = bounds(x, groups)
    assert ((mean.double() - m64).abs() <= off).all()
    assert ((rstd.double() / r64 - 1).abs() <= rel).all()
    xh = (x.double() - per_channel(m64, c)) * per_channel(r64, c)
    want = xh * gamma.double() + beta.double()
    # y moves with the mean and rstd; x - mean, the scale, its product and the sum round
    ga, r1 = gamma.double().abs(), per_channel(rel, c)
    tol = ga * (per_channel(r64 * off, c) * (1 + r1) + xh.abs() * r1)
    tol = tol + 5 * U * (xh.abs() * ga + want.abs())
    if x.dtype != torch.float32:  # its own rounding, and fp16's denormal step
        tol = tol + torch.finfo(x.dtype).eps / 2 * (want.abs() + tol) + 2.0 ** -25
    assert ((y.double() - want).abs() <= tol).all()
    return m64, r64, off, rel


def one_pass_rstd(x, groups):
    """The variance as the mean of squares minus the squared mean, in 32 bits."""
    n, hw, c = x.shape
    v = x.float().view(n, hw, groups, -1)
    var = v.square().mean((1, 3)) - v.mean((1, 3)).square()
    return 1 / (var.clamp(min=0) + EPS).sqrt()


# kept in one CTA and in clusters, in passes; packs within a group, across groups, of one
# value, several groups a pack
SHAPES = [(2, 64, 32, 4), (2, 300, 30, 5), (1, 2000, 33, 3), (2, 3000, 24, 12), (2, 4096, 320, 32),
          (2, 50000, 32, 4), (2, 50000, 33, 3), (2, 50000, 30, 5), (2, 50000, 24, 12)]


@pytest.mark.parametrize("n,hw,c,groups", SHAPES)
def test_mean_thousands_of_deviations_from_zero(n, hw, c, groups):
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(n, hw, c, "fp32", shift=4000.0)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta)
    _, r64, off, rel = check(x, groups, gamma, beta, y, mean, rstd)
    # the bounds tell something: a small part of a deviation, and not a lost variance
    assert (off * r64).max() < 0.1 and rel.max() < 0.3
    if hw >= 3000:
        assert ((one_pass_rstd(x, groups).double() / r64 - 1).abs() > rel).any()


@pytest.mark.parametrize("n,hw,c,groups", SHAPES)
def test_outliers_beside_small_values(n, hw, c, groups):
    # a group's first or last values far from the rest, which are around zero
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(n, hw, c, "fp32")
    cg = c // groups
    x[0, 0, :cg] = -3.0e4
    x[n - 1, hw - 1, -1] = 2.0e5
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta)
    check(x, groups, gamma, beta, y, mean, rstd)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,hw,c,groups", SHAPES)
def test_large_means_in_16_bits(n, hw, c, groups, dtype):
    # as far from zero as the types' own steps leave a variance
    lib = S.gpu_lib()
    x, _, gamma, beta = inputs(n, hw, c, dtype, shift=1000.0 if dtype == "fp16" else 100.0)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta)
    _, r64, off, rel = check(x, groups, gamma, beta, y, mean, rstd)
    assert (off * r64).max() < 0.1


# The gradient's sums, without an activation (dz = dy exactly). A channel's sum is a
# thread's rows (at most 112: 56 KB of 2-byte values for 256 threads; or 338 rows on 7
# lanes, 237 on 3), 8 halvings, 8 CTAs, then an eighth of the runs of rows (at most 296 an
# image) and 8 warps: below KG = 144 + 37 n additions of its terms. A group's adds 16 more
# over its channels.
GRADIENT_SHAPES = SHAPES + [(1, 70000, 130, 10)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,hw,c,groups", GRADIENT_SHAPES)
def test_sums_of_the_gradient(n, hw, c, groups, dtype):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(n, hw, c, dtype)
    _, mean, rstd = forward(lib, x, c, groups, gamma, beta)
    dx, dg, db = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta)
    f = grad64(x, dy, groups, mean, rstd, gamma, beta, 0)
    KG, total = 144 + 37 * n, f["total"]
    size, xh, ga = dy.double().abs(), f["xh"].abs(), gamma.double().abs()
    # x - mean and its product with rstd round
    exh = 2 * U * (xh + per_channel(mean.double().abs() * rstd, c))
    assert ((db.double() - f["db"]).abs() <= KG * U * size.sum((0, 1))).all()
    assert ((dg.double() - f["dg"]).abs() <= (size * (exh + (KG + 1) * U * xh)).sum((0, 1))).all()
    # A / M and B / M, then rstd * (gamma dz - A / M - xh B / M): a few roundings each
    dh = f["dx"] / f["r"]  # gamma dz - A / M - xh B / M
    sum_a = (KG + 20) * U * total(ga * size)
    sum_b = total(ga * size * (exh + (KG + 20) * U * xh))
    both = total(ga * size * xh)
    tol = f["r"] * (8 * U * (ga * size + dh.abs()) + sum_a + xh * sum_b + exh * both
                    + 8 * U * (total(ga * size) + xh * both))
    tol = tol + torch.finfo(x.dtype).eps / 2 * (f["dx"].abs() + tol)
    assert ((dx.double() - f["dx"]).abs() <= tol).all()
