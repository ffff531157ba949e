"""Attention over a paged cache at head sizes that the matrix-core forms do not take (above
128, no multiples of 16), over long texts of which one position takes most of the weight."""
import numpy as np
import pytest

from test_gpu_paged_ops import attn_case, check, check_peaked, f16, half, peaked

pytestmark = pytest.mark.gpu


def with_mean(c):
    """Values around half of the largest, so that weights which are lost do not cancel."""
    v = c["pages"].v
    v[...] = f16(half(v) * 0.5 + 1.0) if c["pages"].type == "fp16" else (v.view(np.int8) // 2 + 64).astype(np.int8).view(np.uint8)
    return c


@pytest.mark.parametrize("type", ["fp16", "int8"])
@pytest.mark.parametrize("H,KVH,hd", [(5, 1, 7), (5, 1, 40), (2, 1, 131), (2, 1, 250), (1, 1, 256), (1, 1, 512),
                                      (14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("gap", [4.6, 7.0])
@pytest.mark.parametrize("at", [0.0, 0.5])
def test_small_weights_beside_a_large_one(type, H, KVH, hd, gap, at):
    """32000 positions share a hundredth or a thousandth of the weight: none of them is lost
    beside the one that has the rest.  (One by one onto a sum of it they are less than a
    step each: 2e-4 of the outputs.)  In sums of 16 and of 256 positions they are 125
    roundings of half a step, 2^-24 of the outputs each, independent ones, and 31 more in
    front of those in the sums of the one's own 256 positions: within the bound's 2^-20."""
    check_peaked(with_mean(peaked(int(10 * gap), type, H, KVH, hd, [32000], [2], at, gap)), [(0, 0), (0, 1)])


@pytest.mark.parametrize("hd", [7, 131, 250, 256, 512])
@pytest.mark.parametrize("past", [0, 1, 14, 15, 16, 17, 31, 255, 256, 257, 271, 272, 273, 511, 600])
def test_ends_of_the_sums(hd, past):
    """Texts that end anywhere in a sum of 16 positions, or of 256."""
    c = attn_case(past, "int8", 2, 1, hd, 16, [past + 1, past], [1, 2])
    check(c)
    check(c, 16, 2)
