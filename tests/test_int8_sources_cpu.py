"""What the sources of the 8-bit operators have to keep to, where a run cannot show it."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "llama2_b200" / "csrc"


def code(path):
    """A source without its comments."""
    return re.sub(r"//[^\n]*", "", path.read_text())


# Kernels that wait for the kernel before them while they run (griddepcontrol.wait)
DEPENDENT = sorted(p.name for p in CSRC.glob("*.cu") if "pdl_wait()" in code(p))


@pytest.mark.parametrize("name", DEPENDENT)
def test_dependent_launches_read_through_the_coherent_path(name):
    """Such a kernel's inputs are written while it runs. The non-coherent path is
    for data that nobody writes during the kernel: a read of it may be moved above
    the wait, or answered from a line that an earlier kernel left in L1."""
    text = code(CSRC / name)
    assert not re.findall(r"__ldg\w*|ldg_keep|ldg_stream|ld\.global\.nc|__restrict__", text)


def test_the_dependent_launches_are_found():
    assert DEPENDENT == ["gemm_int8_tc.cu", "int8_rows.cu"]
    body = code(CSRC / "common.cuh").split("ldg_coherent(const void *p)")[1].split("}")[0]
    assert "asm volatile" in body and "ld.global.v4" in body


def test_a_failed_rank_drains_the_cluster_reduction():
    """After an expired wait a rank of a split tile still waits, with a limit, until
    the reductions into its shared memory have landed, and the other ranks learn of
    the failure before they store: the wait for the reductions does not look at the
    rank's own failure, and comes after each peer's has been read."""
    text = code(CSRC / "gemm_int8_tc.cu")
    tile = text[text.index("linear_int8_tile_kernel("):text.index("linear_int8_pair_kernel(")]
    waits = re.findall(r"mbar_wait\(bar_red, 0, (&?\w+)\)", tile)
    assert waits == ["&quiet"]
    reduction = tile[tile.rindex("cluster_barrier();"):]
    order = [reduction.index(s) for s in ("bulk_add_s32(", "ld_cluster_u32(cluster_addr(abort_addr", "mbar_arrive(bar_red)",
                                          "mbar_wait(bar_red", "store8<T>(", "cluster_barrier_relaxed();")]
    assert order == sorted(order)
    # each peer's warp arrives, beside the one arrival with the byte count
    assert re.search(r"mbar_init\(bar_red, split\)", tile)
