"""What the product's entry points make of their arguments before anything is launched."""
import ctypes as C

import pytest
import torch

from autoresearch_b200.ops import kernels as K

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not a GPU's")


def _code(splitk, batch=1, stride_c=0):
    """Return code of an fp32 store; without a GPU the checks end where the first tensor map is made."""
    one = C.c_void_p(1 << 20)
    return K.lib().arb_gemm_bf16(one, one, one, None, 256, 256, 512, batch, 512, 512, 256, 256 * 512, 256 * 512, stride_c, 0, 0, K.EPI_STORE_F32,
                                 splitk, 0.0, 0.0, 1.0, None, None)


@pytest.mark.parametrize("batch,stride_c", [(1, 0), (1, 256 * 256), (3, 256 * 256)])
def test_a_split_is_nothing_that_an_fp32_store_is_refused_for(batch, stride_c):
    assert _code(2, batch, stride_c) == _code(1, batch, stride_c) != -3
