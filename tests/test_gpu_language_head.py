"""A language model's head, served and trained, as npl_b200.workloads composes it, against
the same steps in 64 bits."""
import pytest
import torch

import support as S
import w4
from npl_b200 import workloads as W
from test_gpu_token_logprobs import TYPES, U, check_backward, check_forward, gen, tokens

pytestmark = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("m,k,vocab,group,dtype,zeros", [
    (1, 256, 1000, 128, "fp32", False), (5, 500, 4099, 32, "bf16", True),
    (16, 1024, 2000, 64, "fp16", False), (40, 333, 513, 32, "fp32", True),
    (130, 512, 5000, 128, "bf16", True)])
def test_served(m, k, vocab, group, dtype, zeros, captured):
    lib, top, temperature = S.gpu_lib(), 5, 0.5
    randn = lambda *s: torch.randn(*s, generator=gen(m + k), device="cuda")  # noqa: E731
    x, gamma, beta = randn(m, k) * 2 + 0.3, 1 + 0.2 * randn(k), 0.1 * randn(k)
    q, scale, zero = w4.quantize(lib, randn(vocab, k) / k ** 0.5, group, torch.float32, zeros)
    y, logits = torch.empty_like(x), torch.empty(m, vocab, device="cuda", dtype=TYPES[dtype][0])
    t = tokens(m, vocab)
    lp, ent = torch.empty(2, m, device="cuda")
    ids = torch.empty(m, top, device="cuda", dtype=torch.int64)
    tlp = torch.empty(m, top, device="cuda")

    def run():
        assert W.score_tokens_w4(lib, S.cuda_stream(), x, gamma, beta, y, q, scale, zero, group,
                                 logits, t, lp, ent, ids, tlp, temperature) == 0

    run()
    if captured:
        want = [v.clone() for v in (logits, lp, ent, ids, tlp)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for v in (y, logits, lp, ent, ids, tlp):
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((logits, lp, ent, ids, tlp), want))
    # each step against the one before it: the product's sum of K terms rounds at most K + 4
    # times on its way (and once to its type), its inputs are exact
    x64 = x.double()
    d = x64 - x64.mean(1, keepdim=True)
    norm = d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gamma.double() + beta.double()
    assert ((y.double() - norm).abs() <= 2e-5 * (1 + norm.abs())).all()
    weights = w4.weights64(q, scale, zero, group, k)
    exact = y.double() @ weights.t()
    bound = (k + 4) * U * (y.double().abs() @ weights.abs().t())
    tol = bound + half_step(logits.dtype) * (exact.abs() + bound)
    assert ((logits.double() - exact).abs() <= tol + 2.0 ** -25).all()
    check_forward(logits, vocab, t, 1.0 / temperature, (lp, ent, None, ids, tlp), top)
    assert lib.nplk_read_status(S.cuda_stream()) == 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows,vocab,dtype,entropy", [(1, 50, "fp32", True), (33, 1000, "bf16", False),
                                                      (400, 4001, "fp16", True), (5, 40000, "bf16", True)])
def test_trained(rows, vocab, dtype, entropy, in_place):
    lib, temperature = S.gpu_lib(), 2.0
    x = (torch.randn(rows, vocab, generator=gen(rows), device="cuda") * 4).to(TYPES[dtype][0])
    t, kept = tokens(rows, vocab), x.clone()
    lp, ent, g = torch.empty(3, rows, device="cuda")
    stats, g = torch.empty(rows, 2, device="cuda"), g.fill_(-1.0 / rows)
    h = torch.randn(rows, generator=gen(1), device="cuda") if entropy else None
    dx = x if in_place else torch.full_like(x, 99.0)
    assert W.token_loss(lib, S.cuda_stream(), x, t, lp, ent, stats, g, h, dx, temperature) == 0
    check_forward(kept, vocab, t, 1.0 / temperature, (lp, ent, stats, None, None), 0)
    check_backward(kept, vocab, t, stats, ent, g, h, 1.0 / temperature, dx)


def test_a_step_of_training_the_head():
    # the loss's gradient against differences along random directions of the hidden rows:
    # logits = hidden @ weights, d_hidden = dlogits @ weights^T (the framework's own product)
    lib, rows, k, vocab = S.gpu_lib(), 12, 64, 300
    randn = lambda *s: torch.randn(*s, generator=gen(9), device="cuda")  # noqa: E731
    q, scale, zero = w4.quantize(lib, randn(vocab, k) / 8, 32, torch.float32, True)
    weights = w4.weights64(q, scale, zero, 32, k)
    hidden, t = randn(rows, k), torch.randint(0, vocab, (rows,), generator=gen(3), device="cuda")
    g = torch.full((rows,), -1.0 / rows, device="cuda")

    def loss(h64):
        z = h64 @ weights.t()
        return -torch.log_softmax(z, 1)[torch.arange(rows, device="cuda"), t].mean()

    logits = w4.product(lib, hidden, q, scale, zero, 32, vocab, k)
    lp, ent = torch.empty(2, rows, device="cuda")
    stats, dx = torch.empty(rows, 2, device="cuda"), torch.empty_like(logits)
    assert W.token_loss(lib, S.cuda_stream(), logits, t, lp, ent, stats, g, None, dx) == 0
    assert abs(-lp.double().mean() - loss(hidden.double())) <= 2e-5
    d_hidden, dense = torch.zeros_like(hidden), weights.float().contiguous()
    assert lib.nplk_gemm(S.cuda_stream(), rows, k, vocab, 1.0, dx.data_ptr(), vocab,
                         dense.data_ptr(), k, 0.0, d_hidden.data_ptr(), k, None, 0, 0.0, 0, None, 0,
                         None) == 0
    for i in range(4):
        way = torch.randn(rows, k, generator=gen(20 + i), device="cuda").double()
        eps = 1e-5  # central differences in 64 bits: off by some eps^2
        slope = (loss(hidden.double() + eps * way) - loss(hidden.double() - eps * way)) / (2 * eps)
        # dlogits within 2^-16 of sizes that add up to 2 / rows a row, in fp32 products
        tol = 2.0 ** -16 * 2 * (way @ weights.t()).abs().amax()
        assert abs((d_hidden.double() * way).sum() - slope) <= tol
