"""How a call of paged attention is cut, as far as its scratch shows it."""
import pytest

from promptcache_amd import _blocks as B


def few(groups, cols, dim, n_tiles):
    """Scratch of work shared out in blocks of few columns: the tiles' sums, two results of every workgroup."""
    return -(-(n_tiles + 2) // 4) * 4 + 2 * groups * cols * (dim + 2)


@pytest.mark.parametrize("rows, keys, blocks_of_128", [(32, 2032, False), (16, 8016, True), (16, 6016, False), (32, 6032, True), (16, 12016, True)])
def test_long_units_of_heads_of_128_take_the_blocks_of_128(rows, keys, blocks_of_128):
    """32 heads of 128 on 8: (32, 2 032) measured 17.5 us in blocks of 32 columns and 22.2 in blocks of 128, (16, 8 016) 23.5 and 20.2.  The scratch is the larger one of the two element
    types'; fp32 takes the blocks of 128 from fewer keys on, and their results of a few key runs are the smaller scratch."""
    steps = -(-keys // 64)
    units = rows * 4 // 32 * 8
    floats = B.attn_pages_part(rows, 32, 8, 128, 1, rows, keys)
    shared = few(min(512, -(-units * steps // 4)), 32, 128, 1)
    assert (floats < shared / 2) == blocks_of_128, (floats, shared)
