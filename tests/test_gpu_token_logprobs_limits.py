"""Log probabilities at the limits of what the header allows, in every form of the kernel:
one warp, four and sixteen warps a row, a row over a cluster."""
import pytest
import torch

import support as S
from test_gpu_token_logprobs import INF, NAN, TYPES, backward, forward, logits

pytestmark = pytest.mark.gpu

FORMS = [(7, 9), (7, 1003), (600, 3001), (7, 12001), (7, 40001), (320, 20001)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_both_stats_of_a_row_with_a_nan_or_infinity(rows, vocab, dtype):
    lib = S.gpu_lib()
    x = logits(rows, vocab, dtype)
    clean = x.clone()
    x[1, 0] = NAN
    x[2, vocab - 1] = INF
    x[3] = NAN
    x[4, vocab // 2], x[4, 0] = INF, -INF
    x[5] = -INF
    x[5, 1] = NAN
    bad = slice(1, 6)
    t = torch.zeros(rows, device="cuda", dtype=torch.int64)
    lp, ent, st, ids, tlp = forward(lib, x, vocab, t, 3)
    assert st[bad].isnan().all() and lp[bad].isnan().all() and ent[bad].isnan().all()
    assert (ids[bad] == -1).all() and tlp[bad].isnan().all()
    want = forward(lib, clean, vocab, t, 3)
    for a, b in zip((lp, ent, st, ids, tlp), want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[6:], b[6:])
    # a row without a token has log probability 0, whatever it holds
    t[1:4] = torch.tensor([-100, vocab, -1], device="cuda")
    lp, ent, st, _, _ = forward(lib, x, vocab, t, 0)
    assert (lp[1:4] == 0).all() and lp[4:6].isnan().all() and st[bad].isnan().all()
    g = torch.ones(rows, device="cuda")
    dx = backward(lib, x, vocab, t, st, None, g, None)
    assert (dx[1:4] == 0).all() and dx[4:6].isnan().all()
    dx = backward(lib, x, vocab, t, st, ent, g, g)
    assert dx[bad].isnan().all() and torch.isfinite(dx[0]).all() and torch.isfinite(dx[6:]).all()
