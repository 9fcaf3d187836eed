"""The language head's operators on tensors whose elements lie past 2^32: few values in very
wide rows, against the same call on packed rows (the same kernels, so the same bits)."""
import pytest
import torch

import support as S
import w4
from test_gpu_token_logprobs import backward, forward, tokens
from test_gpu_w4 import random_operands

pytestmark = pytest.mark.gpu

PITCH = 32784  # elements, or bytes; a multiple of 16


def far(packed, pitch):
    """packed, its rows `pitch` elements apart in a buffer otherwise unset."""
    rows, cols = packed.shape
    assert (rows - 1) * pitch > 1 << 32
    wide = torch.empty(rows * pitch, device="cuda", dtype=packed.dtype).view(rows, pitch)[:, :cols]
    return wide.copy_(packed)


@pytest.mark.parametrize("m,odd", [(1, 0), (5, 0), (20, 0), (20, 1)])
def test_product_with_far_weights(m, odd):
    lib, n, k, group = S.gpu_lib(), 140000, 160, 32
    x, q, sc, z, b = random_operands(m, n, k, group, "bf16", True)
    if odd:  # the form for rows of any address
        q = torch.cat([q, q[:, :1]], 1)
    want = w4.product(lib, x, q, sc, z, group, n, k, b)
    by = PITCH + odd
    assert torch.equal(w4.product(lib, x, far(q, by), far(sc, by), far(z, by), group, n, k, b), want)


@pytest.mark.parametrize("m,pitch", [(3, (1 << 31) + 8), (16, 1 << 29), (34, 1 << 27), (300, 1 << 24)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_product_with_far_tokens(m, pitch, dtype):
    lib, n, k, group = S.gpu_lib(), 70, 300, 64
    x, q, sc, z, b = random_operands(m, n, k, group, dtype, False)
    want = w4.product(lib, x, q, sc, z, group, n, k, b, out=torch.bfloat16)
    c = far(torch.zeros_like(want), pitch)
    assert torch.equal(w4.product(lib, far(x, pitch), q, sc, z, group, n, k, b, c=c), want)


def test_quantiser():
    lib, n, k, group = S.gpu_lib(), 140000, 70, 32
    w = torch.randn(n, k, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    q, sc, z = w4.quantize(lib, w, group, torch.float16, True)
    a, b, c = far(torch.zeros_like(q), PITCH), far(torch.zeros_like(sc), PITCH), far(
        torch.zeros_like(z), PITCH)
    wide = far(w, PITCH)
    assert lib.nplk_quantize_w4(S.cuda_stream(), n, k, group, 2, wide.data_ptr(), PITCH, a.data_ptr(),
                                PITCH, 1, b.data_ptr(), PITCH, c.data_ptr(), PITCH) == 0
    assert torch.equal(a[:, :k // 2], q[:, :k // 2])
    assert torch.equal(b, sc) and torch.equal(c, z)


@pytest.mark.parametrize("rows,vocab,pitch", [(140000, 40, PITCH), (3, 5000, (1 << 31) + 8),
                                              (700, 9001, 1 << 23)])
def test_log_probabilities_and_gradient(rows, vocab, pitch):
    lib, t = S.gpu_lib(), tokens(rows, vocab)
    g = torch.Generator("cuda").manual_seed(2)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 3).bfloat16()
    d = torch.randn(2, rows, device="cuda", generator=g)
    wide = far(x, pitch)

    def run(v):
        got = forward(lib, v, vocab, t, 4)
        return [*got, backward(lib, v, vocab, t, got[2], got[1], d[0], d[1], out=v)]

    near = torch.zeros(rows, -(-vocab // 8) * 8, device="cuda", dtype=x.dtype)[:, :vocab]
    near.copy_(x)  # rows of the same alignment: the order of a row's sums goes by it
    for a, b in zip(run(wide), run(near)):
        assert torch.equal(a, b)
