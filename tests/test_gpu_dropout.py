"""Dropout against its definition: the same elements kept, every kept value
scaled and rounded once."""
import numpy as np
import pytest
import torch

import support as S
from philox import dropout_bits
from support import nb

pytestmark = pytest.mark.gpu

TYPES = {"fp32": (torch.float32, 0), "fp16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def dropout(lib, x, p, seed, offset, y=None, at=None, n=None):
    code = {v[0]: v[1] for v in TYPES.values()}[x.dtype]
    y = torch.full_like(x, 99.0) if y is None else y
    rc = lib.nplk_dropout(S.cuda_stream(), x.numel() if n is None else n, code, x.data_ptr(),
                          y.data_ptr(), p, seed, offset, None if at is None else at.data_ptr())
    assert rc == 0
    return y


def expected(x, p, seed, offset):
    t = int(np.floor(np.float64(np.float32(p)) * 65536 + 0.5))
    keep = torch.from_numpy(dropout_bits(x.numel(), seed, offset) >= t).cuda().view(x.shape)
    # one fp32 product, rounded to the type: the same two roundings everywhere
    scale = 0.0 if t == 65536 else float(np.float32(65536) / np.float32(65536 - t))
    return torch.where(keep, x.float() * scale, torch.zeros_like(x.float())).to(x.dtype), keep


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 255, 1001, 4096, 65537, 3000001])
@pytest.mark.parametrize("offset", [0, 3, 8, (1 << 35) + 5, (1 << 64) - 13])
def test_sizes_and_offsets(dtype, n, offset):
    lib = S.gpu_lib()
    x = torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(
        TYPES[dtype][0])
    seed = 0x123456789ABCDEF0 + n
    want, _ = expected(x, 0.3, seed, offset)
    got = dropout(lib, x, 0.3, seed, offset)
    assert torch.equal(got, want)
    same = x.clone()
    assert torch.equal(dropout(lib, same, 0.3, seed, offset, y=same), want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("skip_x,skip_y", [(1, 0), (0, 1), (1, 1), (3, 3), (4, 4), (2, 6)])
def test_misaligned_pointers(dtype, skip_x, skip_y):
    lib = S.gpu_lib()
    base = torch.randn(5008, device="cuda").to(TYPES[dtype][0])
    x, y = base[skip_x:skip_x + 5000], torch.full_like(base, 99.0)
    want, _ = expected(x, 0.5, 77, 6)
    dropout(lib, x, 0.5, 77, 6, y=y[skip_y:], n=5000)
    assert torch.equal(y[skip_y:skip_y + 5000], want)
    assert (y[:skip_y] == 99.0).all() and (y[skip_y + 5000:] == 99.0).all()


@pytest.mark.parametrize("p", [0.0, 1.0, 1e-6, 0.999999, 0.1, 0.75])
def test_probabilities(p):
    lib = S.gpu_lib()
    x = torch.randn(100003, device="cuda")
    want, keep = expected(x, p, 5, 0)
    got = dropout(lib, x, p, 5, 0)
    assert torch.equal(got, want)
    if p in (0.0, 1e-6):
        assert torch.equal(got, x)
    if p in (1.0, 0.999999):
        assert (got == 0).all()
    # five deviations of a binomial share
    share = keep.double().mean().item()
    assert abs(share - (1 - p)) <= 5 * (p * (1 - p) / x.numel()) ** 0.5 + 2.0 ** -16


def test_non_finite_values():
    lib = S.gpu_lib()
    x = torch.full((1000,), float("nan"), device="cuda")
    x[::2] = float("inf")
    got = dropout(lib, x, 0.5, 3, 0)
    _, keep = expected(torch.ones_like(x), 0.5, 3, 0)
    assert (got[~keep] == 0).all()
    assert torch.isinf(got[::2][keep[::2]]).all() and torch.isnan(got[1::2][keep[1::2]]).all()


def test_gradient_is_the_same_call():
    # y is linear in x, so dx = mask * dy * scale: the call on dy with the same
    # seed and offset; and a difference of two calls gives the same slope
    lib = S.gpu_lib()
    x, dy = torch.randn(2, 5001, device="cuda")
    dx = dropout(lib, dy, 0.25, 9, 100)
    up, down = (dropout(lib, x + s * dy, 0.25, 9, 100) for s in (0.5, -0.5))
    # three roundings of values below |x| + |dy| and the scale 4/3
    assert ((up - down - dx).abs() <= 6 * 2.0 ** -24 * 4 / 3 * (x.abs() + dy.abs())).all()


def test_captured_replays_draw_new_masks():
    lib = S.gpu_lib()
    n = 4099
    x = torch.randn(n, device="cuda")
    at = torch.zeros(1, device="cuda", dtype=torch.int64)
    y = torch.empty_like(x)
    dropout(lib, x, 0.5, 21, 2, y=y, at=at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dropout(lib, x, 0.5, 21, 2, y=y, at=at)
        at += n
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expected(x, 0.5, 21, 2 + k * n)[0])


def test_count_past_32_bits():
    # 2^32 + 9 elements: positions and indexes beyond 32 bits
    lib = S.gpu_lib()
    n = (1 << 32) + 9
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    dropout(lib, x, 0.5, 4, 11, y=x)
    for start in (0, (1 << 32) - 1000):
        part = x[start:start + 1009]
        want, _ = expected(torch.ones(part.numel(), device="cuda", dtype=x.dtype), 0.5, 4,
                           11 + start)
        assert torch.equal(part, want)
