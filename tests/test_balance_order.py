"""The order of shared-memory accesses within a warp of csrc/balance.cu, read from the source (no GPU needed)."""
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
