"""Calls of the language head's operators that their documentation allows beside the plain
one: several streams and graphs at once, a stream that is not the current one, a wait that
runs out, pitches of no account, the largest counts, rows in every form of the kernels."""
import pytest
import torch

import support as S
import w4
from support import nb
from test_gpu_token_logprobs import (INF, NAN, TYPES, backward, check_backward, check_forward,
                                     forward, gen, logits, tokens)
from test_gpu_w4 import check_whole, random_operands, whole_operands

pytestmark = pytest.mark.gpu

# few tokens, tensor-core tiles by TMA and not, tokens' tiles of each size, K shared by a
# cluster, rows of weights at odd addresses
PRODUCTS = [(1, 4096, 4096, 128, "bf16"), (7, 1000, 1281, 32, "fp32"), (16, 300, 512, 64, "fp16"),
            (20, 1000, 4096, 128, "bf16"), (64, 2000, 640, 32, "fp16"), (40, 500, 1000, 64, "fp32"),
            (300, 1024, 2048, 128, "bf16"), (513, 700, 257, 128, "bf16")]
ROWS = [(1, 128000, "bf16", 20), (3, 50021, "fp16", 5), (400, 9000, "bf16", 5), (64, 1000, "fp32", 0),
        (2, 300001, "fp16", 32)]


def product_of(lib, ops, case, c=None, stream=None):
    m, n, k, group, dtype = case
    return w4.product(lib, *ops[:4], group, n, k, ops[4], act=6, out=TYPES[dtype][0], c=c,
                      stream=stream)


def test_all_kernels_at_once_and_replayed():
    # each on a stream of its own, as launches and as graphs, the inputs read by all
    lib = S.gpu_lib()
    ops = [random_operands(*case, zeros=i % 2 == 0) for i, case in enumerate(PRODUCTS)]
    want = [product_of(lib, o, case) for o, case in zip(ops, PRODUCTS)]
    rows = []
    for n, vocab, dtype, top in ROWS:
        x, t = logits(n, vocab, dtype), tokens(n, vocab)
        g, h = torch.randn(2, n, device="cuda", generator=gen(n))
        out = forward(lib, x, vocab, t, top)
        rows.append((x, vocab, t, top, g, h, out, backward(lib, x, vocab, t, out[2], out[1], g, h)))
    torch.cuda.synchronize()

    def calls(i, stream):
        with torch.cuda.stream(stream):
            if i < len(PRODUCTS):
                return [product_of(lib, ops[i], PRODUCTS[i])]
            x, vocab, t, top, g, h, _, _ = rows[i - len(PRODUCTS)]
            out = forward(lib, x, vocab, t, top)
            return [*out, backward(lib, x, vocab, t, out[2], out[1], g, h)]

    wanted = [[w] for w in want] + [[*r[6], r[7]] for r in rows]
    streams = [torch.cuda.Stream() for _ in wanted]
    got = [[] for _ in wanted]
    for _ in range(6):
        for i, stream in enumerate(streams):
            got[i].append(calls(i, stream))
    torch.cuda.synchronize()
    graphs, replayed = [], []
    for i, stream in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            replayed.append(calls(i, stream))
        graphs.append(graph)
    for _ in range(6):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for i, w in enumerate(wanted):
        for results in got[i] + [replayed[i]]:
            for a, b in zip(results, w):
                assert a is b is None or torch.equal(a, b), i
    assert lib.nplk_read_status(S.cuda_stream()) == 0


def test_a_stream_that_is_not_the_current_one():
    lib, side = S.gpu_lib(), torch.cuda.Stream()
    m, n, k, group = 33, 500, 1024, 64
    w = torch.randn(n, k, device="cuda", generator=gen(4))
    want_q, want_s, want_z = w4.quantize(lib, w, group, torch.float16, True)
    x = torch.randn(m, k, device="cuda", generator=gen(5))
    want = w4.product(lib, x, want_q, want_s, want_z, group, n, k)
    t = tokens(m, n)
    wanted = forward(lib, want, n, t, 4)
    g = torch.ones(m, device="cuda")
    want_dx = backward(lib, want, n, t, wanted[2], None, g, None)
    q, s, z = (torch.zeros_like(v) for v in (want_q, want_s, want_z))
    c, dx = torch.zeros_like(want), torch.zeros_like(want)
    lp, ent, st, ids, tlp = (torch.zeros_like(v) for v in wanted)
    torch.cuda.synchronize()
    raw = side.cuda_stream
    assert lib.nplk_quantize_w4(raw, n, k, group, 0, w.data_ptr(), k, q.data_ptr(), q.stride(0), 1,
                                s.data_ptr(), k // group, z.data_ptr(), k // group) == 0
    w4.product(lib, x, q, s, z, group, n, k, c=c, stream=raw)
    assert lib.nplk_token_logprobs(raw, m, n, 0, c.data_ptr(), n, 1.0, t.data_ptr(), lp.data_ptr(),
                                   ent.data_ptr(), st.data_ptr(), 4, ids.data_ptr(),
                                   tlp.data_ptr()) == 0
    assert lib.nplk_token_logprobs_backward(raw, m, n, 0, c.data_ptr(), n, 1.0, t.data_ptr(),
                                            st.data_ptr(), None, g.data_ptr(), None, dx.data_ptr(),
                                            n) == 0
    side.synchronize()
    for a, b in zip((q[:, :k // 2], s, z, c, lp, ent, st, ids, tlp, dx),
                    (want_q[:, :k // 2], want_s, want_z, want, *wanted, want_dx)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m,n,k,dtype", [(20, 256, 4096, "bf16"), (48, 20000, 256, "fp16"),
                                         (300, 512, 1024, "bf16"), (40, 300, 1000, "fp32"),
                                         (17, 100, 100, "fp16")])
def test_expired_wait_is_reported_and_leaves_nothing_behind(m, n, k, dtype):
    # the MMA issuer of one armed launch waits 20 ms on a barrier that nothing arrives on
    lib = S.gpu_lib()
    x, q, sc, z, b = whole_operands(m, n, k, 32, dtype, torch.bfloat16, True)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    assert lib.nplk_debug_arm_wait_timeout(nb.NPLK_DEBUG_GEMM, 20_000) == 0
    w4.product(lib, x, q, sc, z, 32, n, k, b, status=status)
    assert status.item() == nb.NPLK_STATUS_TIMEOUT_MMA
    assert lib.nplk_debug_arm_wait_timeout(nb.NPLK_DEBUG_GEMM, 0) == 0
    check_whole(lib, m, n, k, 32, dtype, torch.bfloat16, True)
    assert lib.nplk_read_status(S.cuda_stream()) == 0


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m", [1, 20])
def test_the_pitch_of_a_single_row_is_of_no_account(m, dtype):
    lib, k, group = S.gpu_lib(), 96, 32
    x, q, sc, z, b = whole_operands(m, 1, k, group, dtype, torch.float32, True)
    want = x.double() @ w4.weights64(q, sc, z & 15, group, k).t() + b.double()
    for ldx in ((k, k + 1, 1 << 40) if m == 1 else (k,)):
        for ldq in (k // 2, k // 2 + 3, 1 << 41):
            c = torch.empty(m, 1, device="cuda")
            assert lib.nplk_gemm_w4(S.cuda_stream(), m, 1, k, group, TYPES[dtype][1], x.data_ptr(),
                                    ldx, q.data_ptr(), ldq, 0, sc.data_ptr(), 1 << 42, z.data_ptr(),
                                    1 << 42, b.data_ptr(), 0, 0.0, 0, c.data_ptr(), 1, None) == 0
            assert torch.equal(c.double(), want)


@pytest.mark.parametrize("m,n,k,dtype", [(100000, 5, 33, "bf16"), (70001, 130, 64, "fp32"),
                                         (2, 1 << 20, 64, "fp16"), (20, 1200000, 32, "bf16"),
                                         (3, 17, 200000, "bf16"), (18, 40, 150000, "fp32")])
def test_many_tokens_channels_and_values(m, n, k, dtype):
    # (few enough that no whole-number sum needs more than 24 bits: |x w| <= 2 * 15 at most,
    # and by chance much less; the sum itself is checked against 2^22)
    check_whole(S.gpu_lib(), m, n, k, 32, dtype, torch.float32, True)


@pytest.mark.parametrize("rows,vocab,dtype", [(1 << 20, 3, "bf16"), (300000, 130, "fp32"),
                                              (70000, 1100, "fp16")])
def test_many_rows(rows, vocab, dtype):
    lib = S.gpu_lib()
    x, t = logits(rows, vocab, dtype), tokens(rows, vocab)
    got = forward(lib, x, vocab, t, 4)
    check_forward(x, vocab, t, 1.0, got, 4)
    g, h = torch.randn(2, rows, device="cuda", generator=gen(2))
    dx = backward(lib, x, vocab, t, got[2], got[1], g, h)
    check_backward(x, vocab, t, got[2], got[1], g, h, 1.0, dx)


def hard_rows(vocab, dtype):
    ramp = torch.arange(vocab, device="cuda").float()
    return torch.stack([torch.zeros_like(ramp), ramp * 8 / vocab, -ramp * 8 / vocab, ramp % 3,
                        torch.where(ramp % 2 == 0, 0.0, -0.0), (ramp >= vocab - 40).float() * 5,
                        (ramp < 40).float() * 5, -(ramp % 7) * 1e-3,
                        torch.where(ramp < vocab - 3, -INF, ramp)]).to(TYPES[dtype][0])


# one warp a row, four (more rows than fill the GPU with wider ones), sixteen, clusters with
# more than one look at their maxima
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("times,vocab", [(1, 500), (40, 9001), (40, 33333), (20, 70000), (1, 600011),
                                         (20, 300007)])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_hard_orders_in_every_form(times, vocab, dtype, top):
    lib, x = S.gpu_lib(), hard_rows(vocab, dtype)
    n = x.shape[0]
    t = torch.full((n,), vocab - 1, device="cuda")
    x, t = x.repeat(times, 1), t.repeat(times)
    got = forward(lib, x, vocab, t, top)
    whole = ~(x == INF).any(1)  # (past 65504 the last row's logits are infinite in fp16)
    check_forward(x[whole], vocab, t[whole], 1.0, tuple(v[whole] for v in got), top)
    assert all(v[~whole].isnan().all() for v in got if v.is_floating_point() and v.dim() == 1)
    assert (got[3][~whole] == -1).all() and got[4][~whole].isnan().all()
    # equal rows at equal places of 16 bytes: equal bits (the order of a row's sums goes by its
    # alignment, which with an odd count of 2-byte values comes back every eighth time)
    for v in got:
        assert torch.equal(v[8 * n:].nan_to_num(7.0), v[:-8 * n].nan_to_num(7.0)) or times < 9


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [(640, 500), (640, 20001), (16, 300007)])
def test_masks_and_nan_in_every_form(rows, vocab, dtype):
    lib, top = S.gpu_lib(), 3
    low = torch.finfo(TYPES[dtype][0]).min
    x, t = logits(rows, vocab, dtype), tokens(rows, vocab)
    nothing, lowest, nan, inf = (slice(i, None, 8) for i in (1, 3, 4, 6))
    x[nothing], x[lowest] = -INF, low
    x[nan, vocab // 3], x[inf, vocab - 1] = NAN, INF
    lp, ent, st, ids, tlp = got = forward(lib, x, vocab, t, top)
    asked = (t >= 0) & (t < vocab)
    assert (lp[nothing] == torch.where(asked, -INF, 0.0)[nothing]).all() and (ent[nothing] == 0).all()
    assert (ids[nothing] == -1).all() and (tlp[nothing] == -INF).all()
    for r in (nan, inf):
        assert ent[r].isnan().all() and (ids[r] == -1).all() and tlp[r].isnan().all()
    rest = torch.ones(rows, device="cuda", dtype=torch.bool)
    for r in (nothing, nan, inf):
        rest[r] = False
    check_forward(x[rest], vocab, t[rest], 1.0, tuple(v[rest] for v in got), top)
    g, h = torch.randn(2, rows, device="cuda", generator=gen(2))
    dx = backward(lib, x, vocab, t, st, ent, g, h)
    assert (dx[nothing] == 0).all() and dx[nan].isnan().all() and dx[inf].isnan().all()
    check_backward(x[rest], vocab, t[rest], st[rest], ent[rest], g[rest], h[rest], 1.0, dx[rest])


@pytest.mark.parametrize("scale", [2.0 ** 126, 1e30, 1e-30, 1e-44])
def test_the_largest_and_smallest_scales(scale):
    # all on the largest logit, and all alike: the limits of softmax
    lib, rows, vocab = S.gpu_lib(), 3, 1000
    x = torch.randint(-50, 50, (rows, vocab), device="cuda", generator=gen(6)).float()
    x[:, 7] = 60.0
    t = torch.tensor([7, 8, 7], device="cuda")
    lp, ent, st, ids, tlp = forward(lib, x, vocab, t, 2, scale)
    if scale > 1:
        d = torch.full_like(lp, -scale) * (60.0 - x[:, 8])
        assert torch.equal(lp, torch.where(t == 7, torch.zeros_like(lp), d))
        assert (ent == 0).all() and (st[:, 1] == 0).all() and (tlp[:, 0] == 0).all()
    else:
        # a thousand equal terms: log 1000 within the sums' roundings
        uniform = torch.full((), vocab, dtype=torch.float64).log().item()
        assert ((ent.double() - uniform).abs() <= 2.0 ** -18).all()
        assert ((lp.double() + uniform).abs() <= 2.0 ** -18).all()
    assert (ids[:, 0] == 7).all()


# as much of x as a CTA holds for a few tokens, just under and just over
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group,dtype", [
    (4, 100, 11008, 128, "bf16"), (8, 70, 6200, 32, "fp16"), (8, 40, 2100, 64, "fp32"),
    (3, 1000, 16000, 64, "bf16"), (1, 33, 51200, 128, "bf16"), (1, 33, 51201, 32, "fp16"),
    (8, 100, 6400, 128, "bf16"), (8, 100, 6432, 32, "bf16"), (16, 100, 2048, 128, "fp16"),
    (16, 100, 2080, 32, "fp16"), (9, 50, 3640, 32, "bf16")])
def test_long_rows_of_few_tokens(m, n, k, group, dtype, zeros):
    check_whole(S.gpu_lib(), m, n, k, group, dtype, TYPES[dtype][0], zeros)
