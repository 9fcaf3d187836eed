"""Log probabilities of given tokens, entropy and alternatives, and their gradient, against
the definition in 64 bits.

Roundings counted (U = 2^-24). u = l - m rounds once, u * scale * log2 e three times, and
2^t is within 2^-22: an exponential is off by at most |d| 4 U + 2^-22 relative. A sum of V
of them adds a chain of at most V / 512 + 64 roundings: `chain`. So S is off by
(mean |d|) 4 U + 2^-22 + chain, and L by that; the mean of |d| under p is L + (-sum p d)."""
import pytest
import torch

import support as S
from support import nb

U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")
TYPES = {"fp32": (torch.float32, 0), "fp16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
CODE = {v[0]: v[1] for v in TYPES.values()}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def ptr(t):
    return None if t is None else t.data_ptr()


def forward(lib, x, vocab, targets, top=0, scale=1.0, stream=None, parts="les"):
    rows = x.shape[0]
    f = lambda *s: torch.full(s, 99.0, device="cuda")  # noqa: E731
    lp, ent, st = (f(rows) if "l" in parts else None, f(rows) if "e" in parts else None,
                   f(rows, 2) if "s" in parts else None)
    ids = torch.full((rows, top), 77, device="cuda", dtype=torch.int64) if top else None
    tlp = f(rows, top) if top else None
    rc = lib.nplk_token_logprobs(stream or S.cuda_stream(), rows, vocab, CODE[x.dtype],
                                 x.data_ptr(), x.stride(0), scale, ptr(targets), ptr(lp), ptr(ent),
                                 ptr(st), top, ptr(ids), ptr(tlp))
    assert rc == 0
    return lp, ent, st, ids, tlp


def backward(lib, x, vocab, targets, stats, ent, g, h, scale=1.0, out=None, stream=None):
    out = torch.full_like(x, 99.0) if out is None else out
    rc = lib.nplk_token_logprobs_backward(stream or S.cuda_stream(), x.shape[0], vocab,
                                          CODE[x.dtype], x.data_ptr(), x.stride(0), scale,
                                          ptr(targets), ptr(stats), ptr(ent), ptr(g), ptr(h),
                                          out.data_ptr(), out.stride(0))
    assert rc == 0
    return out


def f32(scale):
    return float(torch.tensor(scale, dtype=torch.float32))


def in_fp32_range(v):
    # twice the lowest value of bf16 is below fp32's: its nearest fp32 number is -infinity
    return torch.where(v < -torch.finfo(torch.float32).max, -INF, v)


def check_forward(x, vocab, targets, scale, got, top):
    lp, ent, st, ids, tlp = got
    z = x[:, :vocab].double()
    rows = torch.arange(z.shape[0], device="cuda")
    m = z.amax(1)
    d = (z - m[:, None]) * f32(scale)
    e = torch.exp(d)
    s = e.sum(1)
    big_l = torch.log(s)
    p = e / s[:, None]
    finite = torch.where(e > 0, d, 0.0)
    mean, square = -(p * finite).sum(1), (p * finite * finite).sum(1)
    chain = (vocab / 512 + 64) * U
    err_l = mean * 4 * U + 2.0 ** -22 + chain
    tiny = 2.0 ** -40
    if lp is not None:
        asked = (targets >= 0) & (targets < vocab)
        at = d[rows, targets.clamp(0, vocab - 1)]
        want = in_fp32_range(torch.where(asked, at - big_l, 0.0))
        masked = torch.isinf(want)
        assert torch.equal(lp[masked].double(), want[masked])
        tol = err_l + 4 * U * (at.abs() + big_l) + tiny
        assert ((lp.double() - want).abs() <= tol)[~masked].all(), (lp.double() - want).abs().max()
    if ent is not None:
        # the weighted sum's own terms: |d| times an exponential's error, and the division
        tol = err_l + mean * (err_l + 8 * U + chain) + square * 4 * U + 4 * U * big_l + tiny
        assert ((ent.double() - (big_l + mean)).abs() <= tol).all()
    if st is not None:
        assert torch.equal(st[:, 0].double(), m)
        assert ((st[:, 1].double() - big_l).abs() <= err_l + 2 * U * big_l + tiny).all()
    if top:
        order = torch.sort(z, dim=1, descending=True, stable=True)
        n = min(top, vocab)
        want_ids = torch.full_like(ids, -1)
        want_lp = torch.full_like(tlp, -INF, dtype=torch.float64)
        best = order.values[:, :n]
        want_ids[:, :n] = torch.where(best == -INF, -1, order.indices[:, :n])
        want_lp[:, :n] = in_fp32_range((best - m[:, None]) * f32(scale) - big_l[:, None])
        assert torch.equal(ids, want_ids)
        masked = torch.isinf(want_lp)
        assert torch.equal(tlp[masked].double(), want_lp[masked])
        tol = err_l[:, None] + 4 * U * (want_lp.abs() + 2 * big_l[:, None]) + tiny
        assert ((tlp.double() - want_lp).abs() <= tol)[~masked].all()


def check_backward(x, vocab, targets, stats, ent, g, h, scale, got):
    z = x[:, :vocab].double()
    rows, sc = torch.arange(z.shape[0], device="cuda"), f32(scale)
    u = z - stats[:, :1].double()
    log_p = u * sc - stats[:, 1:].double()
    p = torch.exp(log_p)
    asked = torch.zeros_like(rows, dtype=torch.bool)
    if targets is not None:
        asked = (targets >= 0) & (targets < vocab)
    gg = torch.where(asked, g.double(), 0.0) if g is not None else torch.zeros_like(z[:, 0])
    hot = torch.zeros_like(z)
    if asked.any():
        hot[rows[asked], targets[asked]] = 1.0
    want = gg[:, None] * (hot - p)
    size = gg.abs()[:, None] * (hot + p)
    sure = torch.where(p > 0, log_p, 0.0)
    if h is not None:
        inner = sure + ent.double()[:, None]
        want = want - h.double()[:, None] * p * inner
        size = size + h.double().abs()[:, None] * p * (sure.abs() + ent.double().abs()[:, None])
    want, size = want * sc, size * sc
    # p within its exponent's error, then four roundings
    rel = 4 * U * (sure.abs() + 2 * stats[:, 1:].double().abs() + 2) + 2.0 ** -22
    tol = size * (2 * rel + 8 * U)
    half = torch.finfo(x.dtype).eps / 2
    least = {torch.float32: 2.0 ** -125, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -125}
    err = (got[:, :vocab].double() - want).abs()
    # (2^t below 2^-126 counts as 0: up to scale g 2^-126)
    ok = err <= tol + half * (want.abs() + tol) + least[x.dtype] * (1 + size.amax(1, keepdim=True))
    assert ok.all(), (err - tol)[~ok].max()


def logits(rows, vocab, dtype, seed=0, spread=3.0, ld=None):
    wide = torch.full((rows, ld or vocab), NAN, device="cuda", dtype=TYPES[dtype][0])
    wide[:, :vocab] = torch.randn(rows, vocab, device="cuda", generator=gen(seed + vocab)) * spread
    return wide


def tokens(rows, vocab, seed=0):
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(seed))
    if rows > 2:
        t[1], t[2] = -100, vocab  # no token
    return t


SIZES = [(1, 1), (3, 2), (5, 7), (2, 31), (4, 33), (3, 64), (40, 100), (333, 1000), (2, 4095), (1, 8193),
         (7, 16384), (1, 32000), (20, 50021), (1, 128000), (2, 262147), (600, 37)]


@pytest.mark.gpu
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_forward(rows, vocab, dtype, top):
    lib = S.gpu_lib()
    x, t = logits(rows, vocab, dtype), tokens(rows, vocab)
    for scale in (1.0, 1 / 0.7):
        check_forward(x, vocab, t, scale, forward(lib, x, vocab, t, top, scale), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [s for s in SIZES if s[1] < 200000])
def test_backward(rows, vocab, dtype):
    lib = S.gpu_lib()
    x, t = logits(rows, vocab, dtype), tokens(rows, vocab)
    g = torch.randn(rows, device="cuda", generator=gen(1))
    h = torch.randn(rows, device="cuda", generator=gen(2))
    for scale in (1.0, 1 / 0.7):
        _, ent, st, _, _ = forward(lib, x, vocab, t, 0, scale)
        for gg, hh in ((g, None), (None, h), (g, h)):
            got = backward(lib, x, vocab, t, st, ent if hh is not None else None, gg, hh, scale)
            check_backward(x, vocab, t, st, ent, gg, hh, scale, got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 5), (3, 40), (2, 333)])
def test_gradient_against_differences(rows, vocab):
    # of the definition in 64 bits, and against automatic differentiation of it
    lib, scale = S.gpu_lib(), 1 / 0.7
    x = logits(rows, vocab, "fp32", spread=1.5)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=gen(4))
    g = torch.randn(rows, device="cuda", generator=gen(1))
    h = torch.randn(rows, device="cuda", generator=gen(2))
    _, ent, st, _, _ = forward(lib, x, vocab, t, 0, scale)
    got = backward(lib, x, vocab, t, st, ent, g, h, scale).double()

    def total(z):
        log_p = torch.log_softmax(z * f32(scale), 1)
        lp = log_p[torch.arange(rows, device="cuda"), t]
        return (g.double() * lp).sum() - (h.double()[:, None] * torch.exp(log_p) * log_p).sum()

    z = x.double().requires_grad_()
    auto = torch.autograd.grad(total(z), z)[0]
    # stats and entropy carry fp32 roundings: 2^-22 of terms below 16
    assert ((got - auto).abs() <= 2.0 ** -17).all()
    step = 1e-5
    for r in range(rows):
        for v in range(0, vocab, max(1, vocab // 9)):
            a, b = x.double(), x.double()
            a[r, v] += step
            b[r, v] -= step
            diff = (total(a) - total(b)) / (2 * step)
            assert abs(diff - got[r, v]) <= 2.0 ** -17


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_any_address_and_pitch(dtype):
    lib = S.gpu_lib()
    for skip in range(8):
        for rows, vocab, ld in ((3, 1001, 1001), (5, 517, 520), (4, 300, 1303), (1, 3, 3), (40, 9, 11)):
            flat = torch.full((skip + rows * ld,), NAN, device="cuda", dtype=TYPES[dtype][0])
            x = flat[skip:].view(rows, ld)
            x[:, :vocab] = logits(rows, vocab, dtype, seed=skip)
            t = tokens(rows, vocab)
            got = forward(lib, x, vocab, t, 4)
            check_forward(x, vocab, t, 1.0, got, 4)
            g = torch.randn(rows, device="cuda", generator=gen(1))
            for other in (skip, (skip + 3) % 8):
                for ldd in (ld, ld + 1, vocab):
                    around = torch.full((other + rows * ldd + 8,), 99.0, device="cuda", dtype=x.dtype)
                    dx = around[other:other + rows * ldd].view(rows, ldd)
                    backward(lib, x, vocab, t, got[2], got[1], g, g, out=dx)
                    check_backward(x, vocab, t, got[2], got[1], g, g, 1.0, dx)
                    dx[:, :vocab] = 99.0
                    assert (around == 99.0).all()
            want = backward(lib, x, vocab, t, got[2], got[1], g, g)
            same = flat.clone()
            y = same[skip:].view(rows, ld)
            backward(lib, y, vocab, t, got[2], got[1], g, g, out=y)  # in place
            assert torch.equal(y[:, :vocab], want[:, :vocab])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [64, 1003, 40000])
def test_orders_that_are_hard_on_the_alternatives(vocab, dtype):
    # equal logits, rising, falling, few values, zeros of both signs, all in one place
    lib, top = S.gpu_lib(), 20
    ramp = torch.arange(vocab, device="cuda").float()
    x = torch.stack([torch.zeros_like(ramp), ramp * 8 / vocab, -ramp * 8 / vocab, ramp % 3,
                     torch.where(ramp % 2 == 0, 0.0, -0.0), (ramp >= vocab - 40).float() * 5,
                     (ramp < 40).float() * 5, -(ramp % 7) * 1e-3]).to(TYPES[dtype][0])
    t = torch.full((8,), 3, device="cuda")
    check_forward(x, vocab, t, 1.0, forward(lib, x, vocab, t, top), top)
    one = x[1:2].contiguous()  # a row over a cluster
    check_forward(one, vocab, t[:1], 1.0, forward(lib, one, vocab, t[:1], top), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [40, 1000, 33333])
def test_masks(vocab, dtype):
    lib, top = S.gpu_lib(), 6
    low = torch.finfo(TYPES[dtype][0]).min
    x = logits(8, vocab, dtype)
    x[0] = -INF                       # nothing left
    x[1] = low                        # masked by the type's lowest value: uniform
    x[2, 4:] = -INF                   # four left
    x[3, :-1] = low
    x[4, : vocab // 2] = low
    x[5, ::2] = -INF
    x[6] = -INF
    x[6, vocab - 1] = 3.0             # one left
    x[7, 1:] = -INF
    x[7, 0] = low                     # one left, and that the lowest
    t = torch.tensor([1, 1, 2, 0, vocab - 1, 0, vocab - 1, 0], device="cuda")
    for scale in (1.0, 2.0):
        lp, ent, st, ids, tlp = forward(lib, x, vocab, t, top, scale)
        assert lp[0] == -INF and ent[0] == 0 and (ids[0] == -1).all() and (tlp[0] == -INF).all()
        assert (st[0] == -INF).all()
        assert lp[6] == 0 and ent[6] == 0 and lp[7] == 0 and st[7, 0] == low
        keep = slice(1, 8)
        part = tuple(v[keep] for v in (lp, ent, st, ids, tlp))
        check_forward(x[keep], vocab, t[keep], scale, part, top)
        g = torch.randn(8, device="cuda", generator=gen(1))
        h = torch.randn(8, device="cuda", generator=gen(2))
        dx = backward(lib, x, vocab, t, st, ent, g, h, scale)
        assert (dx[0] == 0).all() and torch.isfinite(dx).all()
        assert (dx[x == -INF] == 0).all() or (x[5, 0] == -INF)
        check_backward(x[keep], vocab, t[keep], st[keep], ent[keep], g[keep], h[keep], scale,
                       dx[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [9, 2000, 40001])
def test_rows_that_hold_a_nan_or_infinity(vocab, dtype):
    lib = S.gpu_lib()
    x = logits(7, vocab, dtype)
    clean = x.clone()
    x[1, 0] = NAN
    x[2, vocab - 1] = INF
    x[3] = NAN
    x[4, vocab // 2], x[4, 0] = INF, -INF
    x[5] = -INF
    x[5, 1] = NAN
    t = torch.zeros(7, device="cuda", dtype=torch.int64)
    lp, ent, st, ids, tlp = forward(lib, x, vocab, t, 5)
    for r in range(1, 6):
        assert lp[r].isnan() and ent[r].isnan() and st[r, 1].isnan(), r
        assert (ids[r] == -1).all() and tlp[r].isnan().all(), r
    want = forward(lib, clean, vocab, t, 5)
    for a, b in zip((lp, ent, st, ids, tlp), want):
        assert torch.equal(a[[0, 6]], b[[0, 6]])
    g = torch.ones(7, device="cuda")
    dx = backward(lib, x, vocab, t, st, ent, g, g)
    assert dx[1:6].isnan().all() and torch.isfinite(dx[[0, 6]]).all()
    # rows of which nothing is asked: zeros, whatever they hold
    g[2:5] = 0.0
    t[1] = -1
    dx = backward(lib, x, vocab, t, st, None, g, None)
    assert (dx[1:5] == 0).all() and dx[5].isnan().all()


@pytest.mark.gpu
def test_parts_that_are_not_asked_for():
    lib, rows, vocab = S.gpu_lib(), 5, 3000
    x, t = logits(rows, vocab, "bf16"), tokens(rows, vocab)
    whole = forward(lib, x, vocab, t, 7)
    for parts in ("l", "e", "s", "le", "es"):
        got = forward(lib, x, vocab, t if "l" in parts else None, 0, parts=parts)
        for name, a, b in zip("les", got, whole):
            assert a is None if name not in parts else torch.equal(a, b)
    ids = forward(lib, x, vocab, None, 7, parts="")[3]
    assert torch.equal(ids, whole[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_likely_tokens_keep_their_small_log_probabilities(dtype):
    # p near 1: logprob = -log(1 + x) with a small x
    lib, vocab = S.gpu_lib(), 5000
    x = torch.zeros(6, vocab, device="cuda")
    x[:, 17] = torch.tensor([10.0, 15.0, 20.0, 25.0, 30.0, 100.0], device="cuda")
    x = x.to(TYPES[dtype][0])
    t = torch.full((6,), 17, device="cuda")
    lp = forward(lib, x, vocab, t)[0].double()
    want = -torch.log1p((vocab - 1) * torch.exp(-x[:, 17].double()))
    assert ((lp - want).abs() <= 2.0 ** -20 * want.abs() + 64 * U).all()


@pytest.mark.gpu
def test_rows_do_not_depend_on_each_other_and_calls_repeat():
    lib, vocab = S.gpu_lib(), 20000
    x, t = logits(700, vocab, "bf16"), tokens(700, vocab)
    a, b = forward(lib, x, vocab, t, 9), forward(lib, x, vocab, t, 9)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    part = forward(lib, x[100:400], vocab, t[100:400], 9)
    for u, v in zip(a, part):
        assert torch.equal(u[100:400], v)
