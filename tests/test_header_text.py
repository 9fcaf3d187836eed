"""The public headers' comments: the definitions that callers have are whole."""
import re

import pytest

from support import REPO

HEADERS = sorted((REPO / "include").glob("*.h"))


@pytest.mark.parametrize("header", HEADERS, ids=lambda h: h.name)
def test_comment_lines_are_whole(header):
    # every line of a comment after its first starts with its star: a line that lost its
    # beginning does not
    text = header.read_text()
    for comment in re.finditer(r"/\*.*?\*/", text, re.S):
        first = text[:comment.start()].count("\n") + 1
        for i, line in enumerate(comment.group(0).split("\n")[1:], 1):
            assert re.match(r"\s*\*", line), f"{header.name}:{first + i}: {line!r}"


def test_dropout_defines_its_threshold_and_types():
    text = (REPO / "include" / "npl_kernels.h").read_text()
    comment = text[text.index("---- dropout ----"):text.index("nplk_dropout(void")]
    comment = re.sub(r"[\s*]+", " ", comment)
    assert "elements of type `dtype`" in comment
    assert "t is p 65536 rounded to the nearest integer (p in [0, 1], as fp32; halves up)" in comment


@pytest.mark.gpu
@pytest.mark.parametrize("k", [0, 1, 6, 13107, 65534])
def test_the_threshold_rounds_halves_up(k):
    import numpy as np
    import torch

    import support as S
    from philox import dropout_bits

    # (k + 1/2) / 65536 is exact in fp32: t is k + 1
    p, n = (k + 0.5) / 65536, 1 << 20
    x, y = torch.ones(n, device="cuda"), torch.empty(n, device="cuda")
    assert S.gpu_lib().nplk_dropout(S.cuda_stream(), n, 0, x.data_ptr(), y.data_ptr(), p, 7, 0,
                                    None) == 0
    bits = dropout_bits(n, 7, 0)
    assert (bits == k).any()  # what tells k + 1 from k
    scale = float(np.float32(65536) / np.float32(65535 - k))
    want = np.where(bits >= k + 1, scale, 0.0).astype(np.float32)
    assert np.array_equal(y.cpu().numpy(), want)
