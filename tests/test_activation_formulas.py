"""Each activation's derivative is written down once in the kernel sources."""
import re

from support import PKG

CODES = range(11)


def cases(text, name):
    """The case labels of function `name`."""
    at = re.search(rf"\b{name}\((?!x, act)", text).start()
    return [int(v) for v in re.findall(r"case (\d+):", text[at:text.index("\n}\n", at)])]


def test_one_derivative_for_each_activation():
    sources = {p.name: p.read_text() for p in (PKG / "csrc" / "kernels").iterdir()}
    assert "act_slope(" not in "".join(sources.values())
    text = sources["act_epilogue.cuh"]
    found = cases(text, "act_slope_array") + cases(text, "act_slope_call")
    assert "default:  // 10" in text
    assert sorted(found + [10]) == list(CODES)
