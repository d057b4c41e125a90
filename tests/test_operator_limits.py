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
