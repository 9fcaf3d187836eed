"""The 4-bit product's forms one by one: few tokens, tiles of each size with x by TMA and by
threads, K shared by a cluster, weights at odd addresses."""
import pytest
import torch

import support as S
from test_gpu_group_norm import act64
from test_gpu_head_calls import PRODUCTS
from test_gpu_w4 import U, check_whole, gen, random_operands
from w4 import TYPES, pack, product, weights64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [0, 1])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m", [1, 12, 40, 70])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_a_group_is_scaled_in_one_rounding(m, dtype, group, odd):
    # one group, whole numbers: its sum is exact, the result is its product with the scale,
    # rounded once, for scales of 24 bits and for scales next to fp32's limits
    lib, n, k = S.gpu_lib(), 90, group
    g = gen(m + group)
    x = torch.randint(-2, 3, (m, k), device="cuda", generator=g).to(TYPES[dtype][0])
    q = pack(torch.randint(0, 16, (n, k), device="cuda", generator=g), ldq=k // 2 + 16 + odd)
    z = torch.randint(0, 16, (n, 1), device="cuda", generator=g).to(torch.uint8)
    sc = 1.0 + torch.rand(n, 1, device="cuda", generator=g)
    sc[::5] *= 2.0 ** 126  # times 8 alone infinite
    sc[1::5] *= 2.0 ** -126
    for zero in (None, z):
        c = product(lib, x, q, sc, zero, group, n, k)
        want = (x.double() @ weights64(q, sc, zero, group, k).t()).float()
        # Weights as bf16 are quarters, their sums a quarter of the group's, exactly. The scale
        # times that is a multiple of 2^-149 below 2^-126, off by 2^-150 at most; four times it,
        # by 2^-148 below 2^-124, where the wanted number is itself off by 2^-150.
        near = want.abs() < 2.0 ** -124
        assert torch.equal(c[~near], want[~near])
        assert ((c - want).abs() <= 2.0 ** -148)[near].all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m,n,k,group", [(1, 130, 513, 32), (7, 65, 1000, 64), (70, 200, 2049, 128)])
def test_weights_at_odd_addresses_with_scales_of_24_bits(m, n, k, group, dtype):
    lib, g, groups = S.gpu_lib(), gen(k), -(-k // group)
    x = torch.randn(m, k, device="cuda", generator=g).to(TYPES[dtype][0])
    q = pack(torch.randint(0, 16, (n, k), device="cuda", generator=g), ldq=(k + 1) // 2 | 1)
    z = torch.randint(0, 16, (n, groups), device="cuda", generator=g).to(torch.uint8)
    sc = 0.5 + torch.rand(n, groups, device="cuda", generator=g)
    c = product(lib, x, q, sc, z, group, n, k).double()
    w = weights64(q, sc, z, group, k)
    # a value is in at most `group` sums within its group, and in one with each group's scale
    size = x.double().abs() @ w.abs().t()
    assert ((c - x.double() @ w.t()).abs() <= (group + groups + 1) * U * size).all()


# tiles of 32, 48 (groups of 128), 64 and 128 tokens with x by TMA; one stage of K, an odd count
# of them, a share of every CTA of a cluster, and no cluster
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [17, 24, 32, 33, 48, 49, 57, 64, 65, 128])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_tiles_by_tma(m, group, dtype, zeros):
    lib = S.gpu_lib()
    for n, k in ((130, 96), (300, 640), (70, 1024), (200, 4096), (20001, 384)):
        check_whole(lib, m, n, k, group, dtype, TYPES[dtype][0], zeros)


@pytest.mark.parametrize("case", PRODUCTS)
def test_against_64_bits(case):
    # the calls of test_gpu_head_calls.PRODUCTS, which are compared with their own repetition there
    m, n, k, group, dtype = case
    lib = S.gpu_lib()
    x, q, sc, z, b = random_operands(*case, zeros=True)
    for zero in (None, z):
        c = product(lib, x, q, sc, zero, group, n, k, b, act=6).double()
        w = weights64(q, sc, zero, group, k)
        v = x.double() @ w.t() + b.double()
        want = act64(v, 6)
        # steps of a sum as in test_gpu_w4; the slope of swish is up to 1.1, 2e-5 for its formula
        err = 1.1 * (3 * k / 16 + 24 + k / 32) * 2 * U * (x.double().abs() @ w.abs().t() + b.abs())
        assert ((c - want).abs() <= err + 2e-5 * (1 + want.abs())).all()
