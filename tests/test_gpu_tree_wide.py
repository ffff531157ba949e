"""Tree attention at head sizes that the matrix-core form does not take (above 128, no
multiples of 32), over long texts of which one position takes most of the weight."""
import pytest

from test_gpu_tree_ops import attn_case, check_attention
from test_gpu_tree_values import check, peaked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KVH,hd", [(5, 1, 7), (5, 1, 40), (2, 1, 131), (2, 1, 250), (1, 1, 256), (1, 1, 512)])
@pytest.mark.parametrize("gap", [4.6, 7.0])
@pytest.mark.parametrize("at", [0.0, 0.5])
def test_small_weights_beside_a_large_one(H, KVH, hd, gap, at):
    """32000 positions share a hundredth or a thousandth of the weight: none of them is lost
    beside the one that has the rest (whose value is a fiftieth of theirs, or as theirs).  In
    sums of 16 and of 256 positions they are 125 roundings of half a step, 2^-24 of the outputs
    each, independent ones, and 31 more in front of those in the sums of the one's own 256
    positions: within the bound's 2^-20."""
    for value in (0.02, 1.0):
        check(peaked(int(10 * gap), H, KVH, hd, 1, 2, 32000, at, gap, value=value), [(0, 0), (0, 1)])


@pytest.mark.parametrize("hd", [7, 131, 250, 256, 512])
def test_ends_of_the_sums(hd):
    """Texts that end anywhere in a sum of 16 positions, or of 256; nodes that are not seen."""
    past = [0, 1, 13, 14, 15, 16, 17, 31, 249, 250, 255, 256, 257, 271, 272, 273, 511, 600]
    c = attn_case(hd, 2, 1, hd, len(past), 7, past)
    check_attention(c)
    check_attention(c, 16)
