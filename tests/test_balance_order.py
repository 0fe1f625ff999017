"""csrc/balance.cu read from the source (no GPU needed): the order of shared memory within a warp, and what is built."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "smel-ft_b200", "csrc", "balance.cu")


def test_a_warps_counts_are_zero_before_another_lane_adds_to_them():
    """Votes and shuffles order no memory: between the zeroing of a warp's table, its additions and its reads there is a
    __syncwarp each."""
    with open(SOURCE) as f:
        text = f.read()
    body = text[text.index("void warp_run("):text.index("enum TileKind")]
    zero, add, read = body.index("h[e] = 0;"), body.index("atomicAdd(&h["), body.index("= h[e];")
    assert zero < add < read
    assert re.search(r"__syncwarp\(\);", body[zero:add]) and re.search(r"__syncwarp\(\);", body[add:read])


def test_the_usage_kernels_are_the_ones_that_are_launched():
    """The usage statistics are of one sequence: the finishing kernel is built for them at 8 experts to a block alone."""
    with open(SOURCE) as f:
        text = f.read()
    launched = set(re.findall(r"balance_finish_kernel<(\w+), (\d+)><<<", text))
    assert launched == {("USAGE", "8"), ("false", "32")}
