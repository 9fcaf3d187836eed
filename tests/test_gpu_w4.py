"""Weights in 4 bits: the quantiser and the product against their definitions.

Products of small whole numbers and powers of two are compared bit for bit: every sum is
then exact in fp32, whatever its order. Other products: with A = sum |x w| every step of
the sum rounds or cuts by at most 2^-23 A, and a value takes part in at most K / 16 steps of
each of three parts, and in 8 + 16 + K / 32 more for its groups and slices."""
import pytest
import torch

import support as S
from test_gpu_group_norm import act64
from w4 import CODE, TYPES, pack, product, quantize, unpack, weights64

U = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -14, torch.bfloat16: 2.0 ** -126}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- quantiser ----------------------------------------------------------------------

def wanted(w, group, scale_type, zeros):
    n, k = w.shape
    groups = -(-k // group)
    v = torch.zeros(n, groups * group, device=w.device)
    v[:, :k] = w.float()
    v = v.view(n, groups, group)
    # divided by tensors: torch divides by a number as a product with its reciprocal
    if zeros:
        low, high = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
        s = (high - low) / torch.full_like(low, 15.0)
    else:
        s = v.abs().amax(2) / torch.full((), 7.0, device=w.device)
    s = s.to(scale_type).clamp(min=TINY[scale_type])
    q = torch.round(v / s.float()[:, :, None])
    zero = None
    if zeros:
        zero = torch.round(-low / s.float()).clamp(0, 15)
        q = q + zero[:, :, None]
    else:
        q = q + 8
    return q.clamp(0, 15).view(n, -1)[:, :k], s, zero


def check_quantized(w, group, scale_type, q, scale, zero):
    n, k = w.shape
    nibble, s, z = wanted(w, group, scale_type, zero is not None)
    assert torch.equal(scale, s)
    if zero is not None:
        assert torch.equal(zero.float(), z)
    assert torch.equal(unpack(q, k).float(), nibble)
    if k % 2:
        assert (q[:, k // 2] < 16).all()
    assert (q[:, (k + 1) // 2:] == 171).all()


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,k", [(1, 1), (1, 2), (3, 7), (2, 31), (5, 32), (5, 33), (3, 64),
                                 (7, 127), (2, 129), (33, 1281), (300, 256), (1, 40000),
                                 (4099, 65)])
def test_quantizer(n, k, dtype, group, zeros):
    lib = S.gpu_lib()
    w = torch.randn(n, k, device="cuda", generator=gen(n + k))
    w = (w * torch.exp(2 * torch.randn(n, 1, device="cuda", generator=gen(1)))).to(TYPES[dtype][0])
    for scale in {torch.float32, torch.float16, w.dtype}:
        check_quantized(w, group, scale, *quantize(lib, w, group, scale, zeros))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_quantizer_at_any_address_and_pitch(dtype):
    # w ends with its allocation; q keeps its surroundings
    lib, n, k = S.gpu_lib(), 9, 203
    for skip in range(8):
        for pitch, ldq in ((203, 102), (208, 112), (211, 105)):
            flat = torch.randn(skip + (n - 1) * pitch + k, device="cuda", generator=gen(skip))
            w = flat.to(TYPES[dtype][0])[skip:].as_strided((n, k), (pitch, 1))
            around = torch.full((skip + n * ldq + 32,), 171, device="cuda", dtype=torch.uint8)
            q = around[skip:skip + n * ldq].view(n, ldq)
            got = quantize(lib, w, 64, torch.float32, skip % 2 == 0, q=q)
            check_quantized(w, 64, torch.float32, *got)
            assert (around[:skip] == 171).all() and (around[-32:] == 171).all()


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", [torch.float32, torch.float16, torch.bfloat16])
def test_quantizer_borders(scale, zeros):
    # quotients a hair from the halves, by scales that round down and up
    lib = S.gpu_lib()
    k = torch.arange(-7, 7, device="cuda").float() + 0.5
    for top in (7.0, 1.0, 0.3, 3e4, 3e-3, 1e-5, 1e-39):
        s = (torch.tensor(top, device="cuda") / torch.tensor(7.0, device="cuda")).to(scale)
        base = k * s.float().clamp(min=TINY[scale])
        w = torch.stack([base, torch.nextafter(base, base + 1), torch.nextafter(base, base - 1)])
        w = torch.cat([w, torch.full((3, 1), top, device="cuda"),
                       torch.full((3, 1), -top, device="cuda")], 1)
        check_quantized(w, 32, scale, *quantize(lib, w, 32, scale, zeros))


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
def test_quantizer_special_groups(zeros):
    lib, inf, nan = S.gpu_lib(), float("inf"), float("nan")
    w = torch.randn(8, 96, device="cuda", generator=gen(3))
    w[0] = 0.0
    w[1, :32] = 0.5   # one sign: the other limit is 0
    w[2, :32] = -0.5
    w[3, 33] = 1e-45
    w[3, 34:64] = 0.0
    w[3, 32] = 0.0
    w[4, 40] = nan
    w[5, 70] = -inf
    w[6, 0], w[6, 1] = inf, nan
    w[7, 3], w[7, 4] = 3e38, -3e38
    q, scale, zero = quantize(lib, w, 32, torch.float32, zeros)
    bad = torch.zeros(8, 3, device="cuda", dtype=torch.bool)
    for i, j in ((4, 1), (5, 2), (6, 0)):
        bad[i, j] = True
    if zeros:
        bad[7, 0] = True  # the limits' distance is infinite
    nibble, s, z = wanted(torch.where(bad.repeat_interleave(32, 1), 0.0, w), 32, torch.float32,
                          zeros)
    assert torch.equal(scale[~bad], s[~bad])
    got = unpack(q, 96).float()
    assert torch.equal(got[~bad.repeat_interleave(32, 1)], nibble[~bad.repeat_interleave(32, 1)])
    assert torch.isnan(scale[4, 1]) and scale[5, 2] == inf and torch.isnan(scale[6, 0])
    if zeros:
        assert torch.equal(zero.float()[~bad], z[~bad]) and scale[7, 0] == inf
    # equal nibbles and zeros: the group stands for scale * 0
    for i, j in bad.nonzero().tolist():
        at = 8 if zero is None else zero[i, j].float()
        assert (got[i, 32 * j:32 * j + 32] == at).all()


# ---- product ------------------------------------------------------------------------

def whole_operands(m, n, k, group, dtype, scale, zeros, ldx=None, ldq=None, seed=0):
    """Small whole numbers and powers of two: with K <= 16384 no sum needs more than 24 bits."""
    g = gen(seed + m + 3 * n + 5 * k)
    rand = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")  # noqa: E731
    x = torch.full((m, ldx or k), float("nan"), device="cuda", dtype=TYPES[dtype][0])
    x[:, :k] = rand(-2, 3, m, k)
    q = pack(rand(0, 16, n, k), ldq=ldq, behind=0xff)
    groups = -(-k // group)
    sc = torch.pow(2.0, rand(-1, 1, n, groups).float()).to(scale)
    z = rand(0, 256, n, groups).to(torch.uint8) if zeros else None  # the low four bits count
    return x, q, sc, z, rand(-8, 9, n).float()


def check_whole(lib, m, n, k, group, dtype="bf16", scale=torch.float32, zeros=False, ldx=None,
                ldq=None, bias=True, **kw):
    x, q, sc, z, b = whole_operands(m, n, k, group, dtype, scale, zeros, ldx, ldq)
    b = b if bias else None
    c = product(lib, x, q, sc, z, group, n, k, b, **kw)
    w = weights64(q, sc, None if z is None else z & 15, group, k)
    want = x[:, :k].double() @ w.t() + (b.double() if bias else 0.0)
    assert want.abs().max() < 2 ** 22
    assert torch.equal(c[:, :n].double(), want), (c - want).abs().max()


SIZES = [(1, 1, 1), (1, 16, 2), (1, 17, 31), (2, 5, 33), (1, 300, 256), (3, 40, 257), (8, 100, 512),
         (9, 33, 127), (16, 1000, 1281), (17, 100, 300), (5, 64, 4096), (33, 130, 129), (1, 50, 16384),
         (64, 200, 700), (100, 257, 96), (130, 128, 1024), (300, 40, 513), (1, 5000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_whole_numbers_exactly(m, n, k, dtype, group, zeros):
    check_whole(S.gpu_lib(), m, n, k, group, dtype, TYPES[dtype][0], zeros)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 100, 515), (12, 100, 515), (70, 100, 515)])
def test_types_of_scales(m, n, k, dtype, scale):
    check_whole(S.gpu_lib(), m, n, k, 64, dtype, scale, True, bias=False)


@pytest.mark.gpu
@pytest.mark.parametrize("m", range(1, 36))
def test_every_count_of_tokens(m):
    check_whole(S.gpu_lib(), m, 150, 600, 64, "bf16", torch.float32, m % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 2, 15, 16, 30, 32, 34, 63, 64, 65, 96, 128, 160, 250, 255, 256, 258,
                               511, 512, 513, 768, 1000, 2049, 4095, 8193])
@pytest.mark.parametrize("m", [1, 10, 40])
def test_every_kind_of_depth(m, k):
    for group in (32, 128):
        check_whole(S.gpu_lib(), m, 70, k, group, "fp16", torch.float16, k % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m", [1, 7, 16, 40, 150])
def test_any_pitch(m, dtype):
    lib, n, k = S.gpu_lib(), 77, 333
    for ldx, ldq in ((333, 176), (341, 167), (336, 208), (340, 176)):
        check_whole(lib, m, n, k, 32, dtype, torch.bfloat16, True, ldx, ldq)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 40, 150])
def test_any_address_and_the_surroundings_of_c(m):
    lib, n, k, group = S.gpu_lib(), 90, 320, 64
    x, q, sc, z, b = whole_operands(m, n, k, group, "bf16", torch.bfloat16, True)
    want = x.double() @ weights64(q, sc, z & 15, group, k).t() + b.double()
    shifted = lambda t, by: torch.cat([t.new_zeros(by), t.reshape(-1)])[by:].view(t.shape)  # noqa: E731
    for by in (0, 1, 3, 8):
        around = torch.full((m + 2, n + 13), 77.0, device="cuda", dtype=torch.float32)
        c = around[1:-1, by:by + n]
        product(lib, shifted(x, by), shifted(q, by), shifted(sc, by), shifted(z, by), group, n, k,
                shifted(b, by), c=c)
        assert torch.equal(c.double(), want)
        c[:] = 77.0
        assert (around == 77.0).all()


def at_the_end(t):
    """A copy of t whose last byte is the last of a memory segment of its own."""
    room = torch.empty(32 << 20, device="cuda", dtype=torch.uint8)
    size = t.numel() * t.element_size()
    return room[room.numel() - size:].view(t.dtype).view(t.shape).copy_(t)


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group,dtype", [(1, 300, 2048, 32, "bf16"), (9, 48, 640, 64, "fp16"),
                                               (2, 33, 96, 32, "fp32"), (40, 130, 608, 32, "bf16"),
                                               (70, 100, 256, 128, "fp32")])
def test_nothing_behind_the_operands_is_read(m, n, k, group, dtype, zeros):
    lib = S.gpu_lib()
    x, q, sc, z, b = whole_operands(m, n, k, group, dtype, TYPES[dtype][0], zeros)
    want = product(lib, x, q, sc, z, group, n, k, b)
    x, q, sc, b = (at_the_end(t) for t in (x, q, sc, b))
    z = at_the_end(z) if zeros else None
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    assert torch.equal(product(lib, x, q, sc, z, group, n, k, b), want)


def random_operands(m, n, k, group, dtype, zeros, seed=0):
    g = gen(seed + m + n + k)
    x = (torch.randn(m, k, generator=g, device="cuda") * 3).to(TYPES[dtype][0])
    q = pack((torch.randn(n, k, generator=g, device="cuda") * 2.5 + 8).round().clamp(0, 15))
    groups = -(-k // group)
    sc = ((0.5 + torch.rand(n, groups, generator=g, device="cuda")) / (2.5 * k ** 0.5)).to(
        TYPES[dtype][0])
    z = (torch.randint(4, 13, (n, groups), generator=g, device="cuda").to(torch.uint8)
         if zeros else None)
    return x, q, sc, z, 0.1 * torch.randn(n, generator=g, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("act", range(11))
@pytest.mark.parametrize("m,n,k,group,dtype,out", [
    (1, 200, 1000, 64, "bf16", "bf16"), (3, 100, 4096, 128, "fp32", "fp32"),
    (12, 64, 513, 32, "fp16", "fp16"), (40, 130, 640, 128, "bf16", "fp32"),
    (200, 130, 1024, 64, "fp16", "bf16"), (65, 90, 333, 32, "fp32", "fp16")])
def test_activations_and_results(m, n, k, group, dtype, out, act):
    lib, zeros = S.gpu_lib(), act % 2 == 0
    x, q, sc, z, b = random_operands(m, n, k, group, dtype, zeros)
    c = product(lib, x, q, sc, z, group, n, k, b, act=act, out=TYPES[out][0]).double()
    w = weights64(q, sc, z, group, k)
    v = x.double() @ w.t() + b.double()
    size = x.double().abs() @ w.abs().t() + b.double().abs()
    want = act64(v, act)
    steps = 3 * k / 16 + 24 + k / 32
    # slopes up to 1.13 (GELU, swish) and 1.76 (SELU); 2e-5 (1 + |.|) for the formulas
    err = 1.76 * steps * 2 * U * size + 2e-5 * (1 + want.abs())
    half = torch.finfo(TYPES[out][0]).eps / 2
    assert ((c - want).abs() <= err + half * (want.abs() + err) + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 9, 40])
def test_fp32_inputs_keep_all_their_bits(m):
    # one weight of 1 and one of -1 far apart: the difference of two near numbers
    lib, n, k = S.gpu_lib(), 20, 600
    g = gen(m)
    x = torch.randn(m, k, device="cuda", generator=g) * torch.pow(
        2.0, torch.randint(-60, 60, (m, k), device="cuda", generator=g).float())
    x[:, 500] = x[:, 3] * (1 + 2.0 ** -22)
    nibbles = torch.full((n, k), 8, device="cuda", dtype=torch.uint8)
    nibbles[:, 3], nibbles[:, 500] = 9, 7
    sc = torch.ones(n, -(-k // 128), device="cuda")
    c = product(lib, x, pack(nibbles), sc, None, 128, n, k)
    assert torch.equal(c, (x[:, 3] - x[:, 500])[:, None].expand(m, n))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m", [3, 12, 40])
def test_specials_stay_in_their_rows(m, dtype):
    lib, n, k, inf = S.gpu_lib(), 40, 300, float("inf")
    x, q, sc, _, b = random_operands(m, n, k, 64, dtype, False)
    nibbles = unpack(q, k).clone()
    nibbles[:, 7], nibbles[:, 9], nibbles[5, 7] = 10, 3, 3
    q = pack(nibbles)
    clean = product(lib, x, q, sc, None, 64, n, k, b)
    x[0, 11] = float("nan")
    x[1, 7] = inf
    x[2, 7] = -inf
    c = product(lib, x, q, sc, None, 64, n, k, b)
    assert torch.isnan(c[0]).all()
    sign = torch.where(torch.arange(n, device="cuda") == 5, -1.0, 1.0)
    assert torch.equal(c[1], sign * inf) and torch.equal(c[2], -sign * inf)
    assert torch.equal(c[3:], clean[3:])
    # a group's scale that is not finite: its own channel alone
    sc2 = sc.clone()
    sc2[4, 1] = float("nan")
    sc2[6, 0] = inf
    keep = [i for i in range(n) if i not in (4, 6)]
    if m > 3:  # tokens are left
        c = product(lib, x[3:], q, sc2, None, 64, n, k, b)
        again = product(lib, x[3:], q, sc, None, 64, n, k, b)
        assert torch.isnan(c[:, 4]).all() and not torch.isfinite(c[:, 6]).any()
        assert torch.equal(c[:, keep], again[:, keep])


@pytest.mark.gpu
def test_large_values_of_fp32_and_fp16():
    lib = S.gpu_lib()
    top = torch.finfo(torch.float32).max
    x = torch.zeros(2, 64, device="cuda")
    x[0, 1], x[1, 2] = top, -top  # parts by rounding would be infinite
    nib = torch.full((16, 64), 9, device="cuda", dtype=torch.uint8)
    one = torch.ones(16, 2, device="cuda")
    c = product(lib, x, pack(nib), one, None, 32, 16, 64)
    assert (c[0] == top).all() and (c[1] == -top).all()
    h = torch.zeros(1, 64, device="cuda", dtype=torch.float16)
    h[0, 5], h[0, 40] = 2.0 ** -24, 65504.0  # the least and the largest number
    c = product(lib, h, pack(nib), one, None, 32, 16, 64)
    assert (c == 65504.0).all()  # the least one is below the sum's last bit
    h[0, 40] = 0.0
    assert (product(lib, h, pack(nib), one, None, 32, 16, 64) == 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 12, 100])
def test_quantised_weights_come_back(m):
    # the quantiser's weights times the identity's rows: the rounded weights themselves
    lib, n, k = S.gpu_lib(), 70, 333
    w = torch.randn(n, k, device="cuda", generator=gen(m))
    for zeros in (False, True):
        q, sc, z = quantize(lib, w, 32, torch.float32, zeros)
        x = torch.eye(k, device="cuda")[:m]
        c = product(lib, x, q, sc, z, 32, n, k)
        want = weights64(q, sc, z, 32, k)
        assert torch.equal(c.double(), want.float().double().t()[:m])
        # within half a step (of the scale), a whole one where zero and value round apart
        step = sc.repeat_interleave(32, 1)[:, :k].double()
        assert ((want - w.double()).abs() <= (1.0 if zeros else 0.5) * step * (1 + 8 * U)).all()
