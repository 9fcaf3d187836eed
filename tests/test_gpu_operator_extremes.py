"""Residual-block operators at the largest counts of rows, columns and images that they
take, where a product of two sizes passes 2^31, against the definition on parts and, for
the statistics, on all of the values."""
import pytest
import torch

import support as S
from support import nb
from test_gpu_gemm_i8 import check_product, check_quantized
from test_gpu_group_norm import backward, check_backward, check_forward, forward, inputs

pytestmark = pytest.mark.gpu

FP16, U = nb.NPLK_DTYPE_FP16, 2.0 ** -24
MOST = (1 << 31) - 1


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn16(*shape):
    out = torch.empty(*shape, device="cuda", dtype=torch.float16)
    return out.normal_(generator=gen(len(shape)))


def test_group_norm_of_many_rows():
    # 3 images of 2^30 - 7 pixels and one channel: rows past 2^31
    lib, n, hw = S.gpu_lib(), 3, (1 << 30) - 7
    x = randn16(n, hw, 1)
    for i in range(n):
        x[i] += i
    size = lib.nplk_group_norm_workspace_size(n, hw, 1, 1)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)
    y = torch.empty_like(x)
    mean, rstd = torch.empty(n, 1, device="cuda"), torch.empty(n, 1, device="cuda")
    s = S.cuda_stream()
    assert lib.nplk_group_norm_act(s, n, hw, 1, 1, FP16, x.data_ptr(), 1, None, None, 1e-5, 0, 0.0,
                                   y.data_ptr(), 1, mean.data_ptr(), rstd.data_ptr(),
                                   work.data_ptr(), size) == 0
    parts = [slice(0, 5000), slice(hw // 2, hw // 2 + 5000), slice(hw - 5000, hw)]
    dy = randn16(n, hw, 1)
    sums = []
    for i in range(n):
        whole = x[i].double()
        m, v = whole.mean(), whole.var(correction=0)
        # a thread joins 2400 batches of four (half of their roundings stay) and a few
        # dozen more joins follow, of values up to 10
        assert abs(mean[i, 0].item() - m.item()) <= 1300 * U * 10
        assert abs(rstd[i, 0].item() / (v.item() + 1e-5) ** -0.5 - 1) <= 3 * 1300 * U * 10 + 1300 * U
        m, r = mean[i, 0].double(), rstd[i, 0].double()
        for p in parts:
            want = (x[i, p].double() - m) * r
            assert ((y[i, p].double() - want).abs() <= 8 * U * (want.abs() + 1)
                    + 2.0 ** -11 * want.abs() + 2.0 ** -25).all()
        # the gradient's sums, in 64 bits
        whole = (whole - m) * r
        d = dy[i].double()
        sums.append((d.sum(), (d * whole).sum(), d.abs().sum(), (d * whole).abs().sum()))
        del whole, d
    dg, db = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    dx = y  # the result's place is free
    assert lib.nplk_group_norm_act_backward(s, n, hw, 1, 1, FP16, dy.data_ptr(), 1, x.data_ptr(), 1,
                                            mean.data_ptr(), rstd.data_ptr(), None, None, 0, 0.0,
                                            dx.data_ptr(), 1, dg.data_ptr(), db.data_ptr(),
                                            work.data_ptr(), size) == 0
    # a thread's 14200 rows (hw / (296 runs * 256 lanes)) and fewer than 300 more
    K = 14500 * U
    assert abs(db.item() - sum(t[0] for t in sums).item()) <= K * sum(t[2] for t in sums).item()
    assert abs(dg.item() - sum(t[1] for t in sums).item()) <= (K + 4 * U) * 1.01 * sum(
        t[3] for t in sums).item()
    for i in range(n):
        a, b, a_abs, b_abs = (t.item() / hw for t in sums[i])
        m, r = mean[i, 0].double(), rstd[i, 0].double()
        for p in parts:
            xh = (x[i, p].double() - m) * r
            want = r * (dy[i, p].double() - a - xh * b)
            tol = r * (K * (a_abs + xh.abs() * b_abs) + 16 * U * (dy[i, p].double().abs()
                                                                  + xh.abs() + 1))
            assert ((dx[i, p].double() - want).abs() <= tol + 2.0 ** -11 * (want.abs() + tol)
                    + 2.0 ** -25).all()
    assert lib.nplk_read_status(s) == 0


def test_group_norm_of_many_images():
    # 2^29 + 5 images of 4 pixels and two channels
    lib, n, hw, c = S.gpu_lib(), (1 << 29) + 5, 4, 2
    x = randn16(n, hw, c)
    size = lib.nplk_group_norm_workspace_size(n, hw, c, 1)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)
    y, s = torch.empty_like(x), S.cuda_stream()
    mean, rstd = torch.empty(n, 1, device="cuda"), torch.empty(n, 1, device="cuda")
    assert lib.nplk_group_norm_act(s, n, hw, c, 1, FP16, x.data_ptr(), c, None, None, 1e-5, 1, 0.0,
                                   y.data_ptr(), c, mean.data_ptr(), rstd.data_ptr(),
                                   work.data_ptr(), size) == 0
    for start in (0, n // 2, n - 4000):
        p = slice(start, start + 4000)
        v = x[p].double().view(-1, hw * c)
        m = v.mean(1, keepdim=True)
        r = (v.var(1, correction=0, keepdim=True) + 1e-5).rsqrt()
        assert ((mean[p].double() - m).abs() <= 32 * U * v.abs().amax(1, keepdim=True)).all()
        # a mean 32 U top off moves the deviation by no more (times 3, and 32 roundings)
        rel = (3 * 32 * U * v.abs().amax(1, keepdim=True) * r + 32 * U)
        assert ((rstd[p].double() / r - 1).abs() <= rel * (1 + 2 * rel)).all()
        want = ((v - m) * r).clamp(min=0)
        tol = 2 * rel * (want + 1) + 8 * U * (want + 1)
        assert ((y[p].double().view(-1, hw * c) - want).abs() <= tol + 2.0 ** -11 * (want + tol)
                + 2.0 ** -25).all()
    assert lib.nplk_read_status(s) == 0


@pytest.mark.parametrize("axis,rows,cols", [("rows", MOST, 1), ("rows", 1, (1 << 28) + 3),
                                            ("cols", MOST, 1), ("cols", 1, MOST)])
def test_quantisers_of_many_lines_and_long_ones(axis, rows, cols):
    lib, s = S.gpu_lib(), S.cuda_stream()
    x = randn16(rows * cols)
    lines, length = (rows, cols) if axis == "rows" else (cols, rows)
    q = torch.empty(rows * cols, device="cuda", dtype=torch.int8)
    scale = torch.empty(lines, device="cuda")
    assert getattr(lib, f"nplk_quantize_{axis}")(s, rows, cols, FP16, x.data_ptr(), cols,
                                                 q.data_ptr(), length, scale.data_ptr()) == 0
    if length == 1:  # each value is its line's largest
        for start in (0, rows * cols // 2, rows * cols - 5000):
            p = slice(start, start + 5000)
            check_quantized(x[p].view(-1, 1), "rows", q[p].view(-1, 1), scale[p])
    else:
        top = x.abs().amax().float()
        assert torch.equal(scale[0], top / torch.full_like(top, 127.0))
        for start in range(0, length, 1 << 28):
            p = slice(start, min(length, start + (1 << 28)))
            assert torch.equal(q[p], torch.round(x[p].float() / scale[0]).to(torch.int8))


@pytest.mark.parametrize("m,n", [(1 << 30, 1), ((1 << 28) + 3, 3), (1, 1 << 30),
                                 (20, (1 << 28) + 5)])
def test_product_of_many_tokens_or_channels(m, n):
    lib, k = S.gpu_lib(), 16

    def operand(rows):
        return torch.randint(-128, 128, (rows, k), device="cuda", generator=gen(rows % 97),
                             dtype=torch.int8)

    a, b = operand(m), operand(n)
    sa, sb, bias = (torch.rand(r, device="cuda", generator=gen(r % 89)) for r in (m, n, n))
    c = torch.empty(m, n, device="cuda", dtype=torch.float16)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    # scales that keep the results in fp16's range
    sa *= 2.0 ** -9
    assert lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, a.data_ptr(), k, sa.data_ptr(), b.data_ptr(),
                            k, sb.data_ptr(), bias.data_ptr(), 0, 0.0, FP16, c.data_ptr(), n,
                            status.data_ptr()) == 0
    assert status.item() == 0
    big = max(m, n)
    for start in (0, big // 2, big - 3000):
        p = slice(start, start + 3000)
        if m > n:
            check_product(c[p], a[p], b, sa[p], sb, bias, "fp16")
        else:
            check_product(c[:, p], a, b[p], sa, sb[p], bias[p], "fp16")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("groups,hw", [(1 << 24, 5), (1 << 20, 3), (2048, 2), (1 << 21, 40)])
def test_group_norm_of_the_most_channels(groups, hw, dtype):
    lib, c = S.gpu_lib(), 1 << 24
    x, dy, gamma, beta = inputs(1, hw, c, dtype)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    check_forward(x, c, groups, gamma, beta, 6, 1e-5, y, mean, rstd)
    dx, dg, db = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6)
    check_backward(x, dy, c, groups, mean, rstd, gamma, beta, 6, dx, dg, db)
    assert lib.nplk_read_status(S.cuda_stream()) == 0


def test_group_norm_of_the_most_groups_and_one_pixel():
    # a group a value: x - mean is 0, y is beta, every gradient of x 0
    lib, n, c = S.gpu_lib(), 127, 1 << 24
    x, dy, gamma, beta = inputs(1, n, c, "bf16")
    x, dy = x.view(n, 1, c), dy.view(n, 1, c)
    y, mean, rstd = forward(lib, x, c, c, gamma, beta)
    assert torch.equal(y, beta.bfloat16().expand_as(y)) and torch.equal(mean, x[:, 0].float())
    dx, dg, db = backward(lib, dy, x, c, c, mean, rstd, gamma, beta)
    assert (dg == 0).all()
    # rstd (gamma dy - gamma dy): two roundings of rstd gamma dy
    assert (dx.float().abs() <= 4 * U * rstd[:, None] * (gamma * dy.float()).abs()).all()
