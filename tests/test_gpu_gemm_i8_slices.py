"""The 8-bit product where a cluster shares K and its tokens end inside a batch of
the slices' sums: every count of slices and tokens a batch, bit by bit against the
same rows of a larger product."""
import pytest
import torch

import support as S
from test_gpu_gemm_i8 import TYPES, check_product, operands, product

pytestmark = pytest.mark.gpu

# By (tokens of a tile, slices), on 148 SMs: n and k. Tokens: the tile's counts off by
# one to three, a lone one in a second tile.
SPLITS = {(32, 2): (9000, 1024), (32, 4): (300, 512), (32, 8): (300, 1024),
          (64, 2): (4096, 2048), (64, 4): (1500, 4096), (64, 8): (1500, 4096),
          (128, 2): (4096, 4096), (128, 4): (4096, 4096), (128, 8): (1500, 8192)}
TOKENS = {32: (17, 18, 19, 29, 31, 33), 64: (62, 63, 65, 67, 99, 126, 130),
          128: (65, 67, 90, 99, 127, 130, 131, 190, 253)}


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tile", sorted(SPLITS))
def test_tokens_that_end_inside_a_batch(tile, dtype):
    lib = S.gpu_lib()
    n, k = SPLITS[tile]
    a, b, sa, sb, bias = operands(512, n, k)
    want = product(lib, a, b, sa, sb, bias, dtype)
    check_product(want, a, b, sa, sb, bias, dtype)
    for m in TOKENS[tile[0]]:
        c = torch.full((m + 3, n), 99.0, device="cuda", dtype=TYPES[dtype][0])
        product(lib, a[:m], b, sa[:m].clone(), sb, bias, dtype, c=c[:m])
        assert torch.equal(c[:m], want[:m]) and (c[m:] == 99.0).all()
