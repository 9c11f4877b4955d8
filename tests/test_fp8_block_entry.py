"""The library's entry for block-scaled products refuses on the host what none of its kernels does."""
import ctypes

import pytest

from savanna_b200.ops import cuda_ops


@pytest.mark.parametrize("bias,residual", [(1, 0), (0, 1), (1, 1)])
def test_a_weight_gradient_takes_no_bias_and_no_residual(bias, residual):
    """Stored in boxes it would come out without them.  Nothing behind these addresses is read."""
    fn = ctypes.CDLL(cuda_ops._LIB_PATH).sb_gemm_fp8_block
    P, I, LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
    fn.argtypes = [P, P, LL, LL, P, P, LL, LL, I, P, P, P, I, I, I, LL, LL, LL, LL, I, I, I, I, P, P]
    args = [16, 16, 1, 128, 16, 16, 1, 128, 1, 16, 16 if bias else None, 16 if residual else None, 128, 128, 128, 128, 128, 128, 128, 1, 1, 0, 0, None, None]
    assert fn(*args) == -3
