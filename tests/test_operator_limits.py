"""Limits of the operators beside the step that follow from other limits: refused on the host, by the name of what is too large."""
import pytest

from turbogpt_amd import bridge

A = 4096  # an aligned address that nothing reads: every call here is refused


def refused(call, needle):
    assert call == -1
    assert needle in bridge.library().tgk_error(), bridge.library().tgk_error()


@pytest.mark.parametrize("N", [(1 << 22) + 8, 1 << 30])
def test_columns_beyond_the_largest_leading_dimension(N):
    """Y's leading dimension is at least N and at most 2^22: N is too."""
    refused(bridge.library().tgk_gemm_q8(None, 4, N, 256, A, 256, A, 4, A, 256, A, 2, A, N, None, 0), b"N a multiple of 8 and at most 2^22")


# A launch holds fewer than 2^32 work items, 256 a block: a block takes 32 rows of 512 columns, or a tile of 128 x 128.
@pytest.mark.parametrize("rows,columns", [(1 << 29, 8), ((1 << 31) - 1, 8), (1 << 29, 512), (1 << 28, 520), (1 << 20, 1 << 20)])
def test_rows_to_codes_of_more_blocks_than_a_launch_holds(rows, columns):
    refused(bridge.library().tgk_quantize_rows(None, rows, columns, A, columns, A, columns, A, rows), b"2^24 blocks")


@pytest.mark.parametrize("rows,columns", [((1 << 31) - 1, 136), ((1 << 30) + 1, 256), (1 << 20, 1 << 20)])
def test_weights_to_codes_of_more_blocks_than_a_launch_holds(rows, columns):
    tiles = -(-columns // 128)
    refused(bridge.library().tgk_quantize_tiles(None, rows, columns, A, columns, A, columns, A, tiles), b"2^24 blocks")
