"""Residual-block operators on tensors whose elements lie past 2^32: few channels
of very wide rows, against the same call on packed rows (the same kernels, so the
same bits)."""
import pytest
import torch

import support as S
from support import nb

pytestmark = pytest.mark.gpu

PITCH = 32784  # elements; a multiple of 16
BF16 = nb.NPLK_DTYPE_BF16


def wide(rows, cols, dtype):
    """A [rows, cols] view of a [rows, PITCH] buffer (its other columns unset)."""
    return torch.empty(rows * PITCH, device="cuda", dtype=dtype).view(rows, PITCH)[:, :cols]


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


@pytest.mark.parametrize("n,hw", [(2, 70000), (500, 300)])
def test_group_norm_and_gradient(n, hw):
    lib, c, groups = S.gpu_lib(), 24, 3
    rows, stream = n * hw, S.cuda_stream()
    assert (rows - 1) * PITCH > 1 << 32
    packed = torch.randn(rows, c, device="cuda", generator=gen(hw)).bfloat16()
    dy = torch.randn(rows, c, device="cuda", generator=gen(n)).bfloat16()
    gamma, beta = torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
    size = lib.nplk_group_norm_workspace_size(n, hw, c, groups)
    work = torch.empty(size, device="cuda", dtype=torch.uint8)

    def run(x, d):
        y, ld = torch.empty_like(packed), x.stride(0)
        mean, rstd = (torch.empty(n, groups, device="cuda") for _ in range(2))
        dg, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        assert lib.nplk_group_norm_act(stream, n, hw, c, groups, BF16, x.data_ptr(), ld,
                                       gamma.data_ptr(), beta.data_ptr(), 1e-5, 6, 0.0,
                                       y.data_ptr(), c, mean.data_ptr(), rstd.data_ptr(),
                                       work.data_ptr(), size) == 0
        # the gradient in place of x's copy in the wide rows
        assert lib.nplk_group_norm_act_backward(stream, n, hw, c, groups, BF16, d.data_ptr(), c,
                                                x.data_ptr(), ld, mean.data_ptr(),
                                                rstd.data_ptr(), gamma.data_ptr(),
                                                beta.data_ptr(), 6, 0.0, x.data_ptr(), ld,
                                                dg.data_ptr(), db.data_ptr(), work.data_ptr(),
                                                size) == 0
        return y, mean, rstd, x, dg, db

    x = wide(rows, c, torch.bfloat16)
    x.copy_(packed)
    got = run(x, dy)
    want = run(packed.clone(), dy)
    assert torch.isfinite(want[0]).all() and torch.isfinite(want[3]).all()
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    assert lib.nplk_read_status(stream) == 0


@pytest.mark.parametrize("axis", ["rows", "cols"])
def test_quantisers(axis):
    lib, rows, cols = S.gpu_lib(), 140000, 40
    packed = torch.randn(rows, cols, device="cuda", generator=gen(3)).bfloat16()
    x = wide(rows, cols, torch.bfloat16)
    x.copy_(packed)
    lines, length = (rows, cols) if axis == "rows" else (cols, rows)
    ldq = PITCH if axis == "rows" else 1 << 27
    assert (lines - 1) * ldq > 1 << 32

    def run(src, q):
        scale = torch.empty(lines, device="cuda")
        assert getattr(lib, f"nplk_quantize_{axis}")(S.cuda_stream(), rows, cols, BF16,
                                                     src.data_ptr(), src.stride(0), q.data_ptr(),
                                                     q.stride(0), scale.data_ptr()) == 0
        return q[:, :length], scale

    far = torch.empty(lines * ldq, device="cuda", dtype=torch.int8).view(lines, ldq)
    near = torch.empty(lines, (length + 15) // 16 * 16, device="cuda", dtype=torch.int8)
    for g, w in zip(run(x, far), run(packed, near)):
        assert torch.equal(g, w)


@pytest.mark.parametrize("m,n,k", [(140000, 48, 64), (7, 140000, 64), (40, 140000, 64)])
def test_product(m, n, k):
    lib = S.gpu_lib()
    a, b = (torch.randint(-127, 128, (r, k), device="cuda", generator=gen(r), dtype=torch.int8)
            for r in (m, n))
    sa, sb, bias = (torch.rand(r, device="cuda", generator=gen(r + 1)) for r in (m, n, n))
    big = max(m, n)
    assert (big - 1) * PITCH > 1 << 32

    def run(x, w, c):
        assert lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, x.data_ptr(), x.stride(0),
                                sa.data_ptr(), w.data_ptr(), w.stride(0), sb.data_ptr(),
                                bias.data_ptr(), 1, 0.0, BF16, c.data_ptr(), c.stride(0),
                                None) == 0
        return c

    far = wide(big, k, torch.int8)
    far.copy_(a if m > n else b)
    c = wide(m, n, torch.bfloat16) if m > n else torch.empty(m, n, device="cuda",
                                                             dtype=torch.bfloat16)
    got = run(far, b, c) if m > n else run(a, far, c)
    want = run(a, b, torch.empty(m, n, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(got, want)
    assert lib.nplk_read_status(S.cuda_stream()) == 0
