"""The barriers that end kernels whose CTAs use each other's shared memory, read
from the source: such a fault (a CTA gone while another still reads it) must not be
looked for by running it."""
import re

import pytest

from support import PKG

KERNELS = PKG / "csrc" / "kernels"


def body(text, name):
    """The text of kernel `name` from its name to the end of its function."""
    at = text.index(name + "(")
    return text[at:text.index("\n}\n", at)]


@pytest.mark.parametrize("source,kernel", [("gemm_i8.cu", "gemm_i8_split_kernel"),
                                           ("gemm_i8.cu", "gemm_i8_pair_kernel"),
                                           ("conv_window_pair.cu", "conv_window_pair_kernel")])
def test_the_last_cluster_barrier_orders_what_came_before(source, kernel):
    barriers = re.findall(r"\bcluster_sync\w*\(", body((KERNELS / source).read_text(), kernel))
    assert barriers and barriers[-1] == "cluster_sync("


def test_no_load_from_another_cta_goes_unused():
    # the slices' sums: tokens that are loaded are those that are added up
    text = (KERNELS / "gemm_i8.cu").read_text()
    adder = text[text.index("void i8_add_slices("):]
    adder = adder[:adder.index("\n}\n")]
    load = adder.index("ld_shared_cluster_v4")
    assert "if (b < here)" in adder[:load] and "if (b >= here) break" in adder[load:]
    assert re.search(r"here = min\(kBatch, p\.M - m0 - tok\)", adder)


def test_a_pair_waits_for_the_arrivals_of_its_mma_commits():
    # the leader's commits arrive in both CTAs: each producer ends with a wait for the
    # last one on every stage, so none reaches a CTA that has ended
    text = body((KERNELS / "gemm_i8.cu").read_text(), "gemm_i8_pair_kernel")
    producer = text[text.index("TMA producer"):text.index("MMA issuer")]
    tail = producer[producer.index("tma_load_2d_pair(&map_x"):]
    assert "mbar_wait_pair_async(&empty[s]" in tail


@pytest.mark.parametrize("kernel", ["gemm_i8_split_kernel", "gemm_i8_pair_kernel"])
def test_a_warp_reads_its_accumulator_as_a_whole_or_not_at_all(kernel):
    # a wait that expires may end differently from lane to lane
    text = re.sub(r"\s+", " ", body((KERNELS / "gemm_i8.cu").read_text(), kernel))
    waits = re.findall(r"(__all_sync\(0xffffffffu, )?mbar_wait(?:_pair_async)?\(&?acc_full", text)
    assert waits and all(waits)
