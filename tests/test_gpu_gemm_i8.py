"""8-bit quantisers and matrix product against their definitions: the
quantised values and the integer sums exactly, the results within the fp32
roundings of the scales and one half step of their type."""
import pytest
import torch

import support as S
from support import nb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp32": (torch.float32, 0), "fp16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
CODE = {v[0]: v[1] for v in TYPES.values()}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- quantisers -------------------------------------------------------------------

def quantize(lib, x, axis, ldq=None, q=None):
    rows, cols = x.shape
    lines, length = (rows, cols) if axis == "rows" else (cols, rows)
    ldq = ldq or (length + 15) // 16 * 16
    if q is None:
        q = torch.full((lines, ldq), 111, device="cuda", dtype=torch.int8)
    scale = torch.full((lines,), 9.0, device="cuda")
    rc = getattr(lib, f"nplk_quantize_{axis}")(S.cuda_stream(), rows, cols, CODE[x.dtype],
                                               x.data_ptr(), x.stride(0), q.data_ptr(),
                                               q.stride(0), scale.data_ptr())
    assert rc == 0
    return q, scale


def check_quantized(x, axis, q, scale):
    v = x.float() if axis == "rows" else x.float().t()
    # divided by a tensor: torch divides by a number as a product with its reciprocal
    top = v.abs().amax(1)
    want = (top / torch.full_like(top, 127.0)).clamp(min=2.0 ** -126)
    assert torch.equal(scale, want)
    # the quotient's correctly rounded fp32 value, then to the nearest integer
    assert torch.equal(q[:, :v.shape[1]], torch.round(v / want[:, None]).to(torch.int8))
    assert (q[:, v.shape[1]:] == 111).all()


@pytest.mark.parametrize("axis", ["rows", "cols"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (16, 1), (3, 5), (77, 1000), (7, 4096),
                                       (130, 513), (1, 16384), (2, 40001), (2000, 96),
                                       (4097, 33), (33, 8191)])
def test_quantize_sizes(rows, cols, dtype, axis):
    lib = S.gpu_lib()
    x = torch.randn(rows, cols, device="cuda", generator=gen(rows + cols))
    x = (x * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=gen(1)))).to(
        TYPES[dtype][0])
    check_quantized(x, axis, *quantize(lib, x, axis))


@pytest.mark.parametrize("axis", ["rows", "cols"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_quantize_pitches_and_offsets(dtype, axis):
    lib = S.gpu_lib()
    for pitch, skip, ldq in ((1040, 0, 1024), (1003, 1, 1007), (1008, 3, 1001), (1000, 0, 1003)):
        flat = torch.randn(70 * pitch + 8, device="cuda", generator=gen(pitch)).to(TYPES[dtype][0])
        x = flat[skip:skip + 70 * pitch].view(70, pitch)[:, :1000]
        check_quantized(x, axis, *quantize(lib, x, axis, ldq=ldq))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cols", [7, 8, 9, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257])
def test_quantize_narrow_rows(cols, dtype):
    # rows that share a warp: counts that do not fill the last one, pitches of any size
    lib = S.gpu_lib()
    for rows, pitch in ((1, cols), (15, cols), (16, cols + 8 - cols % 8), (333, cols), (70, 300)):
        flat = torch.randn(rows * pitch, device="cuda", generator=gen(rows + cols))
        x = flat.to(TYPES[dtype][0]).view(rows, pitch)[:, :cols]
        around = torch.full((rows + 2, 320), 111, device="cuda", dtype=torch.int8)
        check_quantized(x, "rows", *quantize(lib, x, "rows", q=around[1:-1]))
        assert (around[0] == 111).all() and (around[-1] == 111).all()


@pytest.mark.parametrize("axis", ["rows", "cols"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("length", [2, 5, 509, 1001, 2049, 4095, 16383, 20479])
def test_quantize_at_any_address(length, dtype, axis):
    # x ends with its allocation; q starts at odd bytes and keeps its surroundings
    lib = S.gpu_lib()
    rows, cols = (5, length) if axis == "rows" else (length, 5)
    for skip in range(0, 8, 1 if length < 5000 else 3):
        flat = torch.randn(skip + rows * cols, device="cuda", generator=gen(length + skip))
        x = flat.to(TYPES[dtype][0])[skip:].view(rows, cols)
        around = torch.full((skip + 5 * (length + 3) + 32,), 111, device="cuda", dtype=torch.int8)
        q = around[skip + 1:skip + 1 + 5 * (length + 3)].view(5, length + 3)
        check_quantized(x, axis, *quantize(lib, x, axis, q=q))
        assert (around[:skip + 1] == 111).all() and (around[-31:] == 111).all()


@pytest.mark.parametrize("axis", ["rows", "cols"])
def test_quantize_borders(axis):
    # quotients a hair from the halves that round either way, in fp32 and bf16
    lib = S.gpu_lib()
    k = torch.arange(-126, 127, device="cuda").float() + 0.5
    for top in (127.0, 100.0, 0.3, 3.0e38, 5e-37):
        base = k * (top / 127.0)
        x = torch.stack([base, torch.nextafter(base, base + 1), torch.nextafter(base, base - 1)])
        x = torch.cat([x, torch.full((3, 1), top, device="cuda")], 1)
        for v in (x, x.bfloat16()):
            v = v if axis == "rows" else v.t().contiguous()
            check_quantized(v, axis, *quantize(lib, v, axis))


@pytest.mark.parametrize("axis", ["rows", "cols"])
@pytest.mark.parametrize("length", [40, 5000])
def test_quantize_special_rows(axis, length):
    lib = S.gpu_lib()
    x = torch.randn(7, length, device="cuda", generator=gen(2))
    x[0] = 0.0
    x[1] = 0.0
    x[1, 3] = -1e-45  # the smallest denormal
    x[2] = 1e-39 * torch.arange(length, device="cuda")
    x[3, 7] = float("nan")
    x[4, length - 1] = float("-inf")
    x[5, 5], x[5, 6] = float("inf"), float("nan")
    v = x if axis == "rows" else x.t().contiguous()
    q, scale = quantize(lib, v, axis)
    good = [0, 1, 2, 6]
    check_quantized(x[good], "rows", q[good], scale[good])
    assert torch.isnan(scale[3]) and scale[4] == float("inf") and torch.isnan(scale[5])
    assert (q[3:6, :length] == 0).all()


@pytest.mark.parametrize("axis", ["rows", "cols"])
@pytest.mark.parametrize("rows,cols", [(40, 40), (3000, 513)])
def test_quantize_captured_and_on_two_streams(rows, cols, axis):
    lib = S.gpu_lib()
    x = [torch.randn(rows, cols, device="cuda", generator=gen(i)) * (3 - i) for i in range(3)]
    want = [quantize(lib, v, axis) for v in x]
    held = x[0].clone()
    q, scale = (torch.empty_like(t) for t in want[0])
    q.fill_(111)

    def call():
        rc = getattr(lib, f"nplk_quantize_{axis}")(S.cuda_stream(), rows, cols, 0, held.data_ptr(),
                                                   cols, q.data_ptr(), q.stride(0),
                                                   scale.data_ptr())
        assert rc == 0

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for v, (wq, ws) in zip(x, want):  # the scales fall from one replay to the next
        held.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, wq) and torch.equal(scale, ws)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for st, v in zip(streams, x):
        with torch.cuda.stream(st):
            got.append(quantize(lib, v, axis))
    torch.cuda.synchronize()
    for (gq, gs), (wq, ws) in zip(got, want):
        assert torch.equal(gq, wq) and torch.equal(gs, ws)


# ---- product ------------------------------------------------------------------------

def act64(z, act, alpha):
    if act == 1:
        return z.clamp(min=0)
    if act == 5:
        return 0.5 * z * (1 + torch.tanh(0.7978845608 * (z + 0.044715 * z ** 3)))
    if act == 6:
        return z * torch.sigmoid(z)
    if act == 7:
        return torch.where(z > 0, z, alpha * z)
    return z


def operands(m, n, k, seed=0, pitch_a=None, pitch_b=None, skip=0):
    def rows(r, pitch, s):
        pitch = pitch or (k + 15) // 16 * 16
        flat = torch.randint(-128, 128, (r * pitch + skip,), device="cuda", dtype=torch.int8,
                             generator=gen(s))
        return flat[skip:].view(r, pitch)[:, :k]

    a, b = rows(m, pitch_a, seed + 1), rows(n, pitch_b, seed + 2)
    sa = torch.rand(m, device="cuda", generator=gen(seed + 3)) / 100 + 1e-3
    sb = (torch.rand(n, device="cuda", generator=gen(seed + 4)) / 100 + 1e-3) / k ** 0.5
    bias = torch.randn(n, device="cuda", generator=gen(seed + 5))
    return a, b, sa, sb, bias


def product(lib, a, b, sa, sb, bias, dtype="fp32", act=0, alpha=0.1, c=None, ldc=None):
    m, n = a.shape[0], b.shape[0]
    t, code = TYPES[dtype]
    if c is None:
        c = torch.full((m, ldc or n), 99.0, device="cuda", dtype=t)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    rc = lib.nplk_gemm_i8(S.cuda_stream(), m, n, a.shape[1], a.data_ptr(), a.stride(0),
                          sa.data_ptr(), b.data_ptr(), b.stride(0), sb.data_ptr(),
                          None if bias is None else bias.data_ptr(), act, alpha, code,
                          c.data_ptr(), c.stride(0), status.data_ptr())
    assert rc == 0 and status.item() == 0
    return c


def sums(a, b):
    """Exact integer sums: products and sums below 2^31 are exact in 64-bit floats."""
    return a.double() @ b.double().t()


def check_product(c, a, b, sa, sb, bias, dtype, act=0, alpha=0.1):
    n = b.shape[0]
    scaled = sums(a, b) * sa.double()[:, None] * sb.double()[None, :]
    z = scaled + (0 if bias is None else bias.double()[None, :])
    ref = act64(z, act, alpha)
    # the sum's conversion and two products round by U each, the bias' sum once
    # more; slopes are at most 1.13, an activation's own error a few steps of |z| + 1
    tol = 1.13 * U * (3 * scaled.abs() + z.abs()) + (24 * U * (1 + z.abs()) if act in (5, 6) else 0)
    eps = torch.finfo(TYPES[dtype][0]).eps if dtype != "fp32" else 0.0
    tol = tol + eps / 2 * (ref.abs() + tol) + (2.0 ** -25 if dtype == "fp16" else 0.0)
    err = (c[:, :n].double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    assert (c[:, n:] == 99.0).all()


SIZES = [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (1, 1000, 130), (2, 77, 513), (7, 130, 257),
         (8, 256, 1024), (9, 300, 96), (16, 1024, 2048), (17, 129, 127), (33, 4096, 640),
         (64, 64, 64), (65, 1000, 1280), (100, 3, 5000), (128, 128, 128), (129, 257, 385),
         (200, 320, 4097), (256, 256, 16), (333, 1000, 1280), (1000, 31, 19), (1024, 1024, 1024),
         (777, 2049, 511), (2048, 1500, 300), (5, 16384, 1), (4100, 17, 33), (1500, 4000, 2000)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_sizes(m, n, k, dtype):
    lib = S.gpu_lib()
    ops = operands(m, n, k)
    act = (m + n + k) % 4
    act = (0, 1, 5, 6)[act]
    check_product(product(lib, *ops, dtype=dtype, act=act), *ops, dtype, act=act)


@pytest.mark.parametrize("m,n,k", [(1, 100, 200), (13, 257, 129), (300, 140, 333), (700, 520, 96)])
@pytest.mark.parametrize("pitch,skip", [(0, 1), (1, 0), (5, 3), (16, 0), (64, 16)])
def test_product_pitches_and_offsets(m, n, k, pitch, skip):
    # operands at odd pitches and addresses, C wider than N at an odd pitch
    lib = S.gpu_lib()
    up = (k + 15) // 16 * 16
    ops = operands(m, n, k, pitch_a=up + pitch, pitch_b=up + 2 * pitch, skip=skip)
    for dtype in sorted(TYPES):
        for ldc in (n, n + 1, n + 8):
            check_product(product(lib, *ops, dtype=dtype, act=1, ldc=ldc), *ops, dtype, act=1)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_product_offset_result(m):
    # C one element past an aligned address
    lib = S.gpu_lib()
    ops = operands(m, 256, 128)
    for dtype in sorted(TYPES):
        flat = torch.full((m * 256 + 1,), 99.0, device="cuda", dtype=TYPES[dtype][0])
        c = product(lib, *ops, dtype=dtype, c=flat[1:].view(m, 256))
        check_product(c, *ops, dtype)
        assert flat[0] == 99.0


@pytest.mark.parametrize("m", [1, 24, 200, 600])
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10])
def test_product_activations_match_the_activation_call(m, act):
    # the epilogue's activation against nplk_activation on the plain product
    lib = S.gpu_lib()
    ops = operands(m, 320, 256, seed=act)
    plain, got = product(lib, *ops), product(lib, *ops, act=act)
    want = torch.empty_like(plain)
    assert lib.nplk_activation(S.cuda_stream(), plain.numel(), plain.data_ptr(), want.data_ptr(),
                               act, 0.1, 0) == 0
    # the same fp32 value goes into the same formula, compiled in two places: a
    # few steps of |z| + 1 (SELU's scale 1.76) either way
    assert ((got - want).abs() <= 48 * U * (1 + plain.abs())).all()


@pytest.mark.parametrize("m,n,k", [(1, 64, 131071), (64, 64, 131071), (300, 300, 131071)])
def test_product_extreme_sums(m, n, k):
    # every product 2^14 and the sum just below 2^31, and its negative
    lib = S.gpu_lib()
    a, b, sa, sb, _ = operands(m, n, k)
    a.fill_(-128)
    b.fill_(-128)
    b[::2] = 127
    sa.fill_(1.0)
    sb.fill_(1.0)
    c = product(lib, a, b, sa, sb, None)
    assert torch.equal(c[:, 1::2], torch.full_like(c[:, 1::2], 16384.0 * k).float())
    assert torch.equal(c[:, ::2], torch.full_like(c[:, ::2], -128.0 * 127 * k).float())


@pytest.mark.parametrize("m", [3, 70, 400])
def test_non_finite_scales_poison_their_row_or_column(m):
    lib = S.gpu_lib()
    a, b, sa, sb, bias = operands(m, 200, 96)
    clean = product(lib, a, b, sa, sb, bias)
    sa, sb, a = sa.clone(), sb.clone(), a.clone()
    sa[1], a[1], sb[7] = float("inf"), 0, float("nan")
    c = product(lib, a, b, sa, sb, bias)
    assert torch.isnan(c[1]).all() and torch.isnan(c[:, 7]).all()
    c[1], c[:, 7] = clean[1], clean[:, 7]
    assert torch.equal(c, clean)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", [1, 5, 6])
@pytest.mark.parametrize("m,n", [(5, 70), (60, 200), (700, 640)])
def test_non_finite_scales_with_an_activation(m, n, act, dtype):
    lib = S.gpu_lib()
    a, b, sa, sb, bias = operands(m, n, 256)
    clean = product(lib, a, b, sa, sb, bias, dtype, act)
    sa, sb = sa.clone(), sb.clone()
    sa[2], sb[n - 3] = float("nan"), float("nan")
    c = product(lib, a, b, sa, sb, bias, dtype, act)
    assert torch.isnan(c[2]).all() and torch.isnan(c[:, n - 3]).all()
    c[2], c[:, n - 3] = clean[2], clean[:, n - 3]
    assert torch.equal(c, clean)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("act", [0, 5, 6, 8])
def test_a_row_does_not_depend_on_its_batch(act, dtype):
    lib = S.gpu_lib()
    a, b, sa, sb, bias = operands(3000, 641, 1100)
    want = product(lib, a, b, sa, sb, bias, dtype, act)
    for first, rows in ((0, 1), (1, 7), (5, 16), (100, 40), (33, 90), (1, 300), (700, 2000)):
        part = slice(first, first + rows)
        got = product(lib, a[part], b, sa[part].clone(), sb, bias, dtype, act)
        assert torch.equal(got, want[part])
    odd = torch.empty(40 * 1101, device="cuda", dtype=torch.int8).view(40, 1101)[:, :1100]
    odd.copy_(a[:40])  # operands that the tensor-core kernels do not take
    assert torch.equal(product(lib, odd, b, sa[:40].clone(), sb, bias, dtype, act), want[:40])


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (50, 640, 512), (600, 800, 400)])
def test_captured_streams_and_repeats(m, n, k):
    lib = S.gpu_lib()
    ops = operands(m, n, k)
    c = torch.empty(m, n, device="cuda")
    code = 0

    def call():
        assert lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, ops[0].data_ptr(), ops[0].stride(0),
                                ops[2].data_ptr(), ops[1].data_ptr(), ops[1].stride(0),
                                ops[3].data_ptr(), ops[4].data_ptr(), 0, 0.0, code, c.data_ptr(),
                                n, None) == 0

    call()
    torch.cuda.synchronize()
    want = c.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want)
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        with torch.cuda.stream(st):
            out = torch.empty(m, n, device="cuda")
            rc = lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, ops[0].data_ptr(), ops[0].stride(0),
                                  ops[2].data_ptr(), ops[1].data_ptr(), ops[1].stride(0),
                                  ops[3].data_ptr(), ops[4].data_ptr(), 0, 0.0, code,
                                  out.data_ptr(), n, None)
            assert rc == 0
            got.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert lib.nplk_read_status(S.cuda_stream()) == 0


@pytest.mark.parametrize("m", [1, 30, 520])
def test_quantised_projection_is_near_the_fp32_one(m):
    # quantise tokens by rows and weights [K][N] by columns, multiply: within the
    # quantisation steps of the exact product
    lib = S.gpu_lib()
    k, n = 640, 384
    x = torch.randn(m, k, device="cuda", generator=gen(m))
    w = torch.randn(k, n, device="cuda", generator=gen(1)) / k ** 0.5
    a, sa = quantize(lib, x, "rows")
    b, sb = quantize(lib, w, "cols")
    c = product(lib, a[:, :k], b[:, :k], sa, sb, None)
    # |x w - (q s)(r t)| <= |x| t/2 + |w| s/2 + s t / 4 for each product (and fp32 roundings)
    bound = (x.abs().double().sum(1)[:, None] * sb.double()[None] / 2
             + w.abs().double().sum(0)[None] * sa.double()[:, None] / 2
             + k * sa.double()[:, None] * sb.double()[None] / 4)
    err = (c.double() - x.double() @ w.double()).abs()
    assert (err <= bound * (1 + 1e-3)).all()


@pytest.mark.parametrize("m,n,k", [(64, 256, 1024), (2048, 2048, 1024)])
def test_expired_wait_is_reported_and_leaves_nothing_behind(m, n, k):
    # the MMA issuer of one armed launch waits 20 ms on a barrier that nothing
    # arrives on: status 102, and the next call is right
    lib = S.gpu_lib()
    ops = operands(m, n, k)
    c = torch.empty(m, n, device="cuda")
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    assert lib.nplk_debug_arm_wait_timeout(nb.NPLK_DEBUG_GEMM, 20_000) == 0
    rc = lib.nplk_gemm_i8(S.cuda_stream(), m, n, k, ops[0].data_ptr(), ops[0].stride(0),
                          ops[2].data_ptr(), ops[1].data_ptr(), ops[1].stride(0),
                          ops[3].data_ptr(), None, 0, 0.0, 0, c.data_ptr(), n,
                          status.data_ptr())
    assert rc == 0 and status.item() == nb.NPLK_STATUS_TIMEOUT_MMA
    assert lib.nplk_debug_arm_wait_timeout(nb.NPLK_DEBUG_GEMM, 0) == 0
    check_product(product(lib, *ops), *ops, "fp32")
