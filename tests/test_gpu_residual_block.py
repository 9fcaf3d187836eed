"""The operators of a trained and served residual block run together, as
npl_b200.workloads composes them, against the same steps in 64 bits."""
import pytest
import torch

import support as S
from npl_b200 import workloads as W
from philox import dropout_bits
from support import nb
from test_gpu_group_norm import TYPES, act64, norm64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def block(n, hw, c, groups, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + hw + c)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (randn(n, hw, c) * 1.5 + 0.3 * randn(c)).to(TYPES[dtype])
    ws = S.gpu_lib().nplk_group_norm_workspace_size(n, hw, c, groups)
    return x, 1 + 0.2 * randn(c), 0.2 * randn(c), torch.empty(ws, device="cuda",
                                                              dtype=torch.uint8), ws, randn


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n,hw,c,groups,d,dtype", [
    (1, 1, 64, 8, 96, "bf16"), (2, 64, 320, 32, 320, "bf16"), (1, 257, 48, 6, 33, "fp32"),
    (3, 961, 510, 30, 130, "fp16"), (1, 4096, 640, 32, 1280, "bf16")])
def test_served_projection(n, hw, c, groups, d, dtype, captured):
    lib = S.gpu_lib()
    x, gamma, beta, work, ws, randn = block(n, hw, c, groups, dtype)
    weights, bias = randn(c, d) / c ** 0.5, 0.1 * randn(d)
    ldq = (c + 15) // 16 * 16
    w = torch.zeros(d, ldq, device="cuda", dtype=torch.int8)
    w_scale = torch.empty(d, device="cuda")
    assert lib.nplk_quantize_cols(S.cuda_stream(), c, d, 0, weights.data_ptr(), d, w.data_ptr(),
                                  ldq, w_scale.data_ptr()) == 0
    y, out = torch.empty_like(x), torch.empty(n, hw, d, device="cuda", dtype=x.dtype)
    q = torch.empty(n * hw, ldq, device="cuda", dtype=torch.int8)
    q_scale = torch.empty(n * hw, device="cuda")

    def run():
        assert W.norm_act_project_i8(lib, S.cuda_stream(), x, groups, gamma, beta, 6, y, q,
                                     q_scale, w, w_scale, bias, out, work, ws) == 0

    run()
    torch.cuda.synchronize()
    if captured:
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for t in (y, q, out):
            t.zero_()
        q_scale.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    xh, _, _ = norm64(x, groups, gamma, beta, 1e-5)
    a = act64(xh * gamma.double() + beta.double(), 6).view(n * hw, c)
    # each step against the one before it: y as in the norm's own tests; the
    # quantiser exactly; the product within its roundings
    eps = torch.finfo(x.dtype).eps
    assert ((y.view(n * hw, c).double() - a).abs() <= eps / 2 * a.abs() + 2e-5 * (1 + a.abs())).all()
    v = y.view(n * hw, c).float()
    top = v.abs().amax(1)
    scale = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)
    assert torch.equal(q_scale, scale)
    assert torch.equal(q[:, :c], torch.round(v / scale[:, None]).to(torch.int8))
    exact = (q[:, :c].double() * scale.double()[:, None]) @ (
        w[:, :c].double() * w_scale.double()[:, None]).t() + bias.double()
    half = eps / 2 if dtype != "fp32" else 0.0
    got = out.view(n * hw, d).double()
    tol = half * exact.abs() + 8 * U * (exact.abs() + bias.double().abs() + 1)
    assert ((got - exact).abs() <= tol + (2.0 ** -25 if dtype == "fp16" else 0)).all()
    # and the whole against the block without quantisation: half a step of each
    # operand per product
    whole = a @ weights.double() + bias.double()
    steps = (scale.double()[:, None] / 2) @ weights.double().abs().sum(0)[None]
    steps = steps + a.abs().sum(1, keepdim=True) * w_scale.double()[None] / 2
    steps = steps + c * scale.double()[:, None] * w_scale.double()[None] / 4
    close = (eps / 2 * a.abs() + 2e-5 * (1 + a.abs())) @ weights.double().abs()
    assert ((got - whole).abs() <= 1.001 * (steps + close + tol) + (2.0 ** -25)).all()


@pytest.mark.parametrize("n,hw,c,groups,dtype", [(2, 64, 320, 32, "bf16"), (1, 961, 34, 2, "fp32"),
                                                 (2, 20000, 64, 8, "fp16")])
def test_trained_block_and_its_gradient(n, hw, c, groups, dtype):
    lib = S.gpu_lib()
    x, gamma, beta, work, ws, randn = block(n, hw, c, groups, dtype, seed=5)
    p, seed, offset = 0.25, 1234567890123, 37
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(2, n, groups, device="cuda")
    dgamma, dbeta = torch.empty(2, c, device="cuda")
    dy = randn(n, hw, c).to(x.dtype)
    st = S.cuda_stream()
    assert W.norm_act_dropout(lib, st, x, groups, gamma, beta, 6, p, seed, offset, y, mean, rstd,
                              work, ws) == 0
    assert W.norm_act_dropout_backward(lib, st, dy, x, groups, mean, rstd, gamma, beta, 6, p, seed,
                                       offset, dx, dgamma, dbeta, work, ws) == 0
    t = int(p * 65536)
    keep = torch.from_numpy(dropout_bits(x.numel(), seed, offset) >= t).cuda().view(x.shape)
    mask = keep.double() * 65536 / (65536 - t)
    x64, g64, b64 = (v.double().requires_grad_() for v in (x, gamma, beta))
    v = x64.view(n, hw, groups, c // groups)
    m = v.mean((1, 3), keepdim=True)
    r = ((v - m).square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    z = ((v - m) * r).view(n, hw, c) * g64 + b64
    out = z * torch.sigmoid(z) * mask
    want = torch.autograd.grad((out * dy.double()).sum(), (x64, g64, b64))
    # the norm's result and the masked gradient are rounded to the type on the way
    # (half a step each), the results once more; fp32 arithmetic below 2e-5
    eps = torch.finfo(x.dtype).eps if dtype != "fp32" else 0.0
    assert ((y == 0) | keep).all()
    assert ((y.double() - out).abs() <= eps * out.abs() * 1.01 + 3e-5 * (1 + out.abs())).all()
    # a rounding of dy moves dx by at most itself times rstd gamma slope, and the
    # group's means of such
    size = r.expand_as(v).reshape(n, hw, c) * g64.abs() * 1.13 * mask.max() * dy.double().abs()
    mean_of = lambda q: q.view(n, hw, groups, -1).mean((1, 3), keepdim=True).expand_as(v).reshape(n, hw, c)  # noqa: E731
    xh = ((v - m) * r).view(n, hw, c).abs()
    bound = (eps / 2 + 3e-5) * (size + mean_of(size) + xh * mean_of(size * xh))
    assert ((dx.double() - want[0]).abs() <= bound + eps / 2 * (want[0].abs() + bound) + 1e-6).all()
    each = 1.13 * mask.max() * dy.double().abs() * (eps / 2 + 3e-5)
    assert ((dgamma.double() - want[1]).abs() <= (each * xh).sum((0, 1))).all()
    assert ((dbeta.double() - want[2]).abs() <= each.sum((0, 1))).all()
