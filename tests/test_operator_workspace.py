"""The group norm's workspace: what is asked for is what the calls use, and it
suffices at every type and alignment and for fewer images."""
import pytest

from support import nb


@pytest.fixture(scope="module")
def lib():
    return nb.load()


@pytest.mark.parametrize("n,hw,c,groups", [(8, 4096, 320, 32), (64, 4096, 320, 32),
                                           (256, 1024, 1280, 32), (1, 64, 1280, 32)])
def test_images_kept_on_the_chip_need_the_channel_sums_only(lib, n, hw, c, groups):
    # the gradient's sums per image and channel, two floats each
    size = lib.nplk_group_norm_workspace_size(n, hw, c, groups)
    assert 8 * n * c <= size <= 8 * n * c + 256


@pytest.mark.parametrize("n,hw,c,groups", [(1, 262144, 128, 32), (4, 16384, 512, 32),
                                           (2, 1500, 2560, 32), (1, 5, 8192, 1)])
def test_passes_over_memory_need_the_sums_of_their_runs(lib, n, hw, c, groups):
    # at most 3 runs of rows for each of 148 SMs and image: the channels' sums and four
    # floats a group, beside four per image and group
    size = lib.nplk_group_norm_workspace_size(n, hw, c, groups)
    runs = n * max(1, min(3 * 148, (hw + 7) // 8))
    assert 0 < size <= runs * (8 * c + 16 * groups) + 16 * n * groups + 256


@pytest.mark.parametrize("hw,c,groups", [(1, 1, 1), (9, 4098, 2), (961, 510, 30), (1024, 640, 32),
                                         (4096, 320, 32), (1500, 2560, 32), (16384, 512, 32),
                                         (20000, 130, 10), (262144, 128, 32)])
def test_more_images_never_need_less(lib, hw, c, groups):
    counts = list(range(1, 70)) + [100, 147, 148, 149, 295, 296, 297, 443, 444, 445, 1000]
    sizes = [lib.nplk_group_norm_workspace_size(n, hw, c, groups) for n in counts]
    assert sizes == sorted(sizes) and sizes[0] > 0


GUARD = 4096


def guarded(torch, size):
    """A 256-byte aligned buffer of `size` bytes and the buffer around it."""
    around = torch.full((size + 2 * GUARD,), 171, device="cuda", dtype=torch.uint8)
    assert around.data_ptr() % 256 == 0
    return around[GUARD:GUARD + size], around


# kept, in clusters and not; in passes, one batch of images and several; odd packs
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,hw,c,groups", [(5, 1, 6, 3), (3, 961, 510, 30), (7, 1024, 64, 8),
                                           (2, 1500, 2560, 32), (3, 16400, 256, 32),
                                           (9, 30000, 128, 4), (3, 40000, 33, 3), (2, 9, 4098, 2)])
def test_the_reported_size_suffices(lib, n, hw, c, groups, dtype):
    import torch

    import test_gpu_group_norm as G

    size = lib.nplk_group_norm_workspace_size(n, hw, c, groups)
    plenty = torch.empty(8 * size + (64 << 20), device="cuda", dtype=torch.uint8)
    x, dy, gamma, beta = G.inputs(n, hw, c, dtype)
    for skip in (0, 1, 2, 4):  # elements past an aligned address: every width of packs
        move = lambda t: torch.cat([t.new_zeros(skip), t.reshape(-1)])[skip:].view(t.shape)  # noqa: E731
        for images in sorted({n, 1, (n + 1) // 2}, reverse=True):
            xs, ds = move(x[:images]), move(dy[:images])
            work, around = guarded(torch, size)
            mine, big = (work, size), (plenty, plenty.numel())
            y, mean, rstd = G.forward(lib, xs, c, groups, gamma, beta, 6, y=move(torch.zeros_like(xs)),
                                      work=mine)
            got = G.backward(lib, ds, xs, c, groups, mean, rstd, gamma, beta, 6,
                             dx=move(torch.zeros_like(xs)), work=mine)
            assert (around[:GUARD] == 171).all() and (around[GUARD + size:] == 171).all()
            want = G.forward(lib, xs, c, groups, gamma, beta, 6, y=move(torch.zeros_like(xs)),
                             work=big)
            more = G.backward(lib, ds, xs, c, groups, mean, rstd, gamma, beta, 6,
                              dx=move(torch.zeros_like(xs)), work=big)
            for a, b in zip((y, mean, rstd) + got, want + more):
                assert torch.equal(a, b)
