"""The residual as the output itself, on every kernel of the product with an epilogue: each element is read once, by the thread
that writes it, and stored once."""
import ctypes
import math

import pytest
import torch

from decode_matmul_amd import capi
from gpu_util import DEV
from ops_util import assert_within, decode64, fused_inputs, product64

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
TYPE = {F16: 0, F32: 1}


@pytest.fixture(autouse=True)
def default_choice():
    lib = capi.lib()
    before = lib.dmm_set_gemv_8bit(1)
    yield
    lib.dmm_set_ops_kernel(-1)
    lib.dmm_set_gemv_8bit(before)


def in_place(x, codes, grid, scale, bias, act, gated, r):
    """y = the call's result, computed in the residual's own memory."""
    M, K = x.shape
    N = codes.shape[0] // 2 if gated else codes.shape[0]
    xd, cd, gd, y = (t.to(DEV) for t in (x, codes, grid, r.clone()))
    bd = None if bias is None else bias.to(DEV)
    lib = capi.lib()
    ep = capi.Epilogue(bias=None if bd is None else bd.data_ptr(), residual=y.data_ptr(), bias_type=0 if bd is None else TYPE[bd.dtype],
                       residual_type=TYPE[r.dtype], out_type=TYPE[r.dtype], activation={"none": 0, "silu": 2}[act], gated=int(gated),
                       scale=scale, scale_up=scale)
    need = lib.dmm_fused_workspace_bytes(M, N, K, int(gated))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    capi.check("fused", lib.dmm_decode_matmul_fused(xd.data_ptr(), cd.data_ptr(), gd.data_ptr(), ctypes.byref(ep), y.data_ptr(), M, N, K,
                                                    ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return y


def test_more_jobs_than_the_redo_has_numbers_for():
    """20000 segments of two rows on 8-bit operands, some 78 jobs per workgroup, a late one with an infinity: the rows beside it
    must not get their residual twice."""
    M, N, K = 40000, 16, 256
    x, codes, grid, _, r = fused_inputs(M, N, K, False, None, F16, 3, coarse=True)
    bad = [M - 1, M // 2, 140]
    x[bad, 100] = math.inf
    capi.lib().dmm_set_ops_kernel(4)
    y = in_place(x, codes, grid, 0.05, None, "none", False, r)
    want, tol = product64(x.double(), decode64(codes, grid), (0.05, 0.05), None, False, "none", r, F16)
    keep = torch.ones(M, dtype=torch.bool)
    keep[bad] = False
    assert_within(y.cpu()[keep], want[keep], tol[keep])
    assert not torch.isfinite(y[bad]).any()


# one row: the streaming body, the batch-1 body on 8-bit operands, one job and many on 8-bit operands; two rows
@pytest.mark.parametrize("M,N,K,gated", [(1, 4096, 512, False), (1, 16400, 512, False), (1, 5504, 512, True), (1, 40004, 512, False),
                                         (1, 20000, 256, True), (2, 4096, 512, False), (2, 14000, 4096, False), (2, 40004, 512, False)])
@pytest.mark.parametrize("what", ["finite", "infinity", "grid"])
def test_one_and_two_rows(M, N, K, gated, what):
    """As the library chooses; what 8-bit operands cannot do is done again in the same launch."""
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, F16, F16, M + N, fp8=what != "grid", coarse=True)
    if what == "infinity":
        x[M - 1, K // 2] = math.inf
    act, s = ("silu" if gated else "none"), 1 / math.sqrt(K)
    y = in_place(x, codes, grid, s, b, act, gated, r)
    want, tol = product64(x.double(), decode64(codes, grid), (s, s), b, gated, act, r, F16)
    if what == "infinity":
        assert not torch.isfinite(y[M - 1]).all()
        y, want, tol = y[:M - 1], want[:M - 1], tol[:M - 1]
    assert_within(y, want, tol)


@pytest.mark.parametrize("kernel", [-1, 0, 1, 2, 3, 5], ids=["auto", "generic", "rows", "gemm", "split", "mid"])
@pytest.mark.parametrize("M", [1, 2, 5, 12, 40, 130, 700])
@pytest.mark.parametrize("N,K,gated,types", [(100, 768, True, F16), (515, 512, False, F32), (272, 2048, False, F16)])
def test_every_kernel(M, N, K, gated, types, kernel):
    capi.lib().dmm_set_gemv_8bit(0)       # sums of exact products
    capi.lib().dmm_set_ops_kernel(kernel)
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, F32, types, M + N + K)
    s = 1 / math.sqrt(K)
    y = in_place(x, codes, grid, s, b, "silu", gated, r)
    assert_within(y, *product64(x.double(), decode64(codes, grid), (s, s), b, gated, "silu", r, types))
