"""Calls of the residual-block operators that their documentation allows beside the plain
one: in place at every form, results inside larger buffers, several streams and graphs at
once, a stream that is not the current one."""
import pytest
import torch

import support as S
from support import nb
from test_gpu_gemm_i8 import operands, product, quantize
from test_gpu_group_norm import TYPES, backward, forward, inputs, workspace

pytestmark = pytest.mark.gpu

# kept in one CTA, in clusters (rows by TMA where packs are of 16 bytes, runs of rows that
# do not fill their boxes), in passes by one and by several batches of images
FORMS = [(3, 50, 64, 8), (2, 4001, 320, 32), (2, 1500, 640, 32), (2, 30000, 64, 8),
         (5, 40000, 128, 4), (2, 3001, 36, 6)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,hw,c,groups", FORMS)
def test_group_norm_in_place(n, hw, c, groups, dtype):
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(n, hw, c, dtype)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    want = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6)
    for _ in range(3):
        same = x.clone()
        got = forward(lib, same, c, groups, gamma, beta, act=6, y=same)
        assert torch.equal(same, y) and torch.equal(got[1], mean) and torch.equal(got[2], rstd)
        over_dy, over_x = dy.clone(), x.clone()
        a = backward(lib, over_dy, x, c, groups, mean, rstd, gamma, beta, act=6, dx=over_dy)
        b = backward(lib, dy, over_x, c, groups, mean, rstd, gamma, beta, act=6, dx=over_x)
        for g, h, w in zip(a, b, want):
            assert torch.equal(g, w) and torch.equal(h, w)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,hw,c,groups", FORMS)
def test_group_norm_leaves_the_rows_around_its_images(n, hw, c, groups, dtype):
    # n images of a batch of n + 2, pitches wider than the channels
    lib, ld = S.gpu_lib(), c + 16
    x, dy, gamma, beta = inputs(n + 2, hw, c, dtype, ld=ld)
    x[0], x[-1], dy[0], dy[-1] = (float("nan"),) * 4
    y, dx = torch.full_like(x, 99.0), torch.full_like(x, 99.0)
    _, mean, rstd = forward(lib, x[1:-1], c, groups, gamma, beta, act=5, y=y[1:-1])
    backward(lib, dy[1:-1], x[1:-1], c, groups, mean, rstd, gamma, beta, act=5, dx=dx[1:-1])
    for t in (y, dx):
        assert (t[0] == 99.0).all() and (t[-1] == 99.0).all() and (t[1:-1, :, c:] == 99.0).all()
        assert torch.isfinite(t).all()


@pytest.mark.parametrize("n,hw,c,groups", FORMS)
def test_gradients_on_several_streams_and_replayed_graphs(n, hw, c, groups):
    # the same tensors read by all, a workspace and results each
    lib = S.gpu_lib()
    x, dy, gamma, beta = inputs(n, hw, c, "bf16")
    _, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    want = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    works = [workspace(lib, n, hw, c, groups) for _ in streams]
    graphs, got = [], []
    for st, work in zip(streams, works):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got.append(backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6, work=work))
        graphs.append(graph)
    for _ in range(5):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(g, w) for g, w in zip(out, want))
    assert lib.nplk_read_status(S.cuda_stream()) == 0


def test_products_of_all_kernels_at_once():
    # CTA pairs with fp32 and 16-bit results, clusters that share K, single tiles, rows and
    # the library's fp32 product, each on a stream of its own
    lib = S.gpu_lib()
    cases = [(2048, 2048, 512, "fp32"), (2048, 2048, 512, "bf16"), (20, 1000, 1024, "fp32"),
             (31, 300, 512, "fp16"), (127, 4096, 4096, "bf16"), (700, 4096, 128, "fp32"),
             (1, 4096, 4096, "bf16")]
    ops = [operands(m, n, k) for m, n, k, _ in cases]
    want = [product(lib, *o, dtype=case[3], act=6) for o, case in zip(ops, cases)]
    a, b = torch.randn(512, 512, device="cuda"), torch.randn(512, 512, device="cuda")

    def fp32_product(stream):
        c = torch.empty(512, 512, device="cuda")
        assert lib.nplk_gemm(stream, 512, 512, 512, 1.0, a.data_ptr(), 512, b.data_ptr(), 512,
                             0.0, c.data_ptr(), 512, None, 0, 0.0, 0, None, 0, None) == 0
        return c

    streams = [torch.cuda.Stream() for _ in range(len(cases) + 1)]
    whole = fp32_product(S.cuda_stream())
    torch.cuda.synchronize()
    got, others = [[] for _ in cases], []
    outs = [[torch.empty_like(w) for _ in range(10)] for w in want]
    for i in range(10):
        for j, (o, case) in enumerate(zip(ops, cases)):
            m, n, k, dtype = case
            x, w, sa, sb, bias = o
            c = outs[j][i]
            assert lib.nplk_gemm_i8(streams[j].cuda_stream, m, n, k, x.data_ptr(), x.stride(0),
                                    sa.data_ptr(), w.data_ptr(), w.stride(0), sb.data_ptr(),
                                    bias.data_ptr(), 6, 0.1,
                                    {"fp32": 0, "fp16": 1, "bf16": 2}[dtype], c.data_ptr(), n,
                                    None) == 0
            got[j].append(c)
        with torch.cuda.stream(streams[-1]):
            others.append(fp32_product(streams[-1].cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(c, whole) for c in others)
    for out, w in zip(got, want):
        assert all(torch.equal(c, w) for c in out)
    assert lib.nplk_read_status(S.cuda_stream()) == 0


def test_a_stream_that_is_not_the_current_one():
    # inputs made on the current stream, the operators on another after an event
    lib = S.gpu_lib()
    side, n, hw, c = torch.cuda.Stream(), 2, 777, 64
    x, _, gamma, beta = inputs(n, hw, c, "bf16")
    work, size = workspace(lib, n, hw, c, 8)
    y, d = torch.empty_like(x), torch.empty_like(x)
    q = torch.empty(n * hw, c, device="cuda", dtype=torch.int8)
    scale, bias = torch.empty(n * hw, device="cuda"), torch.zeros(c, device="cuda")
    w, ws = quantize(lib, torch.eye(c, device="cuda"), "rows")
    out = torch.empty(n * hw, c, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    s = side.cuda_stream
    code = nb.NPLK_DTYPE_BF16
    assert lib.nplk_group_norm_act(s, n, hw, c, 8, code, x.data_ptr(), c, gamma.data_ptr(),
                                   beta.data_ptr(), 1e-5, 6, 0.0, y.data_ptr(), c, None, None,
                                   work.data_ptr(), size) == 0
    assert lib.nplk_dropout(s, y.numel(), code, y.data_ptr(), d.data_ptr(), 0.5, 3, 1, None) == 0
    assert lib.nplk_quantize_rows(s, n * hw, c, code, d.data_ptr(), c, q.data_ptr(), c,
                                  scale.data_ptr()) == 0
    assert lib.nplk_gemm_i8(s, n * hw, c, c, q.data_ptr(), c, scale.data_ptr(), w.data_ptr(),
                            w.stride(0), ws.data_ptr(), bias.data_ptr(), 0, 0.0, 0,
                            out.data_ptr(), c, None) == 0
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, forward(lib, x, c, 8, gamma, beta, act=6)[0])
    kept = d != 0
    assert torch.equal(d[kept], (y * 2)[kept])
    # rows of the identity are 127 / 127: the product gives the rounded rows back
    want = d.float().view(-1, c)
    assert ((out - want).abs() <= 0.51 * scale[:, None]).all()


@pytest.mark.parametrize("m,n,k", [(40, 1, 64), (40, 1, 4096), (1000, 1, 64), (1, 200, 64)])
def test_the_pitch_of_a_single_row_is_of_no_account(m, n, k):
    lib, far = S.gpu_lib(), 1 << 44
    a, b, sa, sb, bias = operands(m, n, k)
    want = product(lib, a, b, sa, sb, bias)
    c, status = torch.empty_like(want), torch.zeros(1, device="cuda", dtype=torch.int32)
    assert lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, a.data_ptr(), far if m == 1 else k,
                            sa.data_ptr(), b.data_ptr(), far if n == 1 else k, sb.data_ptr(),
                            bias.data_ptr(), 0, 0.1, 0, c.data_ptr(), far if m == 1 else n,
                            status.data_ptr()) == 0
    assert torch.equal(c, want) and status.item() == 0


@pytest.mark.parametrize("c,groups", [(64, 8), (8192, 1)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_the_pitch_of_a_single_pixel_is_of_no_account(c, groups, dtype):
    lib, far = S.gpu_lib(), 1 << 44
    x, dy, gamma, beta = inputs(1, 1, c, dtype)
    y, mean, rstd = forward(lib, x, c, groups, gamma, beta, act=6)
    dx, _, _ = backward(lib, dy, x, c, groups, mean, rstd, gamma, beta, act=6)
    work, size = workspace(lib, 1, 1, c, groups)
    code = {"fp32": 0, "fp16": 1, "bf16": 2}[dtype]
    y2, dx2 = torch.zeros_like(y), torch.zeros_like(dx)
    assert lib.nplk_group_norm_act(S.cuda_stream(), 1, 1, c, groups, code, x.data_ptr(), far,
                                   gamma.data_ptr(), beta.data_ptr(), 1e-5, 6, 0.1, y2.data_ptr(),
                                   far, None, None, work.data_ptr(), size) == 0
    assert lib.nplk_group_norm_act_backward(S.cuda_stream(), 1, 1, c, groups, code, dy.data_ptr(),
                                            far, x.data_ptr(), far, mean.data_ptr(),
                                            rstd.data_ptr(), gamma.data_ptr(), beta.data_ptr(), 6,
                                            0.1, dx2.data_ptr(), far, None, None, work.data_ptr(),
                                            size) == 0
    assert torch.equal(y2, y) and torch.equal(dx2, dx)
