"""Every form of the block-scaled products where its rings wrap and its tiles end inside: which form a size runs by is asserted beside its values."""
import pytest

from savanna_b200.ops import cuda_ops

pytestmark = pytest.mark.gpu

def _takes_few(T, N):
    return bool(cuda_ops.require().sb_gemm_fp8_block_takes_few(T, N))


def test_wide_products_of_more_than_31_tokens_go_by_tiles():
    """Where the tiles' kernel was the faster one."""
    assert not any(_takes_few(T, 12288) for T in (32, 33, 64))
    assert all(_takes_few(T, 12288) for T in (1, 16, 17, 31)) and all(_takes_few(T, 8192) for T in (1, 32, 64))
