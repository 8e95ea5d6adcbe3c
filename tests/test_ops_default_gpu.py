"""The operators around the product as a user gets them: the library's own choice, 8-bit operands in their default position."""
import ctypes
import math

import pytest
import torch

import decode_matmul_amd as dmm
from decode_matmul_amd import capi
from gpu_util import DEV
from ops_util import (ACTS, assert_within, check_routing, combine64, decode64, fused_inputs, grouped64, grouped_inputs, product64, weights)

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def dev(*ts):
    return [t.to(DEV) if t is not None else None for t in ts]


@pytest.fixture(autouse=True)
def default_choice():
    lib = capi.lib()
    before = lib.dmm_set_gemv_8bit(1)
    yield
    lib.dmm_set_ops_kernel(-1)
    lib.dmm_set_gemv_8bit(before)


@pytest.mark.parametrize("M,N,K,gated", [(2, 4096, 4096, False), (2, 4100, 2048, False), (1, 4096, 4088 - 8, False), (2, 8192, 4096, False),
                                         (2, 2048, 4096, True), (2, 40000, 1024, False)])
def test_few_tiles_keep_16_bit_operands(M, N, K, gated):
    """Where 8-bit operands save no time, one and two rows have the sums of exact products: what they have with the switch off."""
    x, codes, grid, _, _ = fused_inputs(M, N, K, gated, None, None, M + N + K)
    args = dev(x, codes, grid)
    y = dmm.decode_matmul_fused(*args, 1 / math.sqrt(K), gated=gated)
    capi.lib().dmm_set_gemv_8bit(0)
    assert torch.equal(y, dmm.decode_matmul_fused(*args, 1 / math.sqrt(K), gated=gated))
