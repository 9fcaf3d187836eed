"""The dropout tests' generator against its authors' published answers."""
import numpy as np

from philox import philox

ANSWERS = [
    ([0] * 4, [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
]


def test_published_answers():
    for counter, key, want in ANSWERS:
        got = philox([np.array([c], dtype=np.uint64) for c in counter], key)
        assert [int(w[0]) for w in got] == want
