"""Activations relative to their result, far into the tails: on the host, and on the GPU through kernels of every form of epilogue."""
import math

import pytest
import torch

import decode_matmul_amd as dmm
from decode_matmul_amd import capi
from gpu_util import DEV
from ops_util import EPS32, weights

F16, F32 = torch.float16, torch.float32


def arguments():
    z = torch.cat([torch.linspace(-14, 14, 1401), torch.linspace(-100, -14, 200), torch.tensor([14.5, 20, 87, 90, 200, 6e4, 3e38, math.inf]),
                   -torch.tensor([14.5, 200, 6e4, 3e38]), 10.0 ** torch.linspace(-30, -1, 100), -(10.0 ** torch.linspace(-30, -1, 100))])
    return z.to(F32)


def want_and_tol(z, act):
    """The activation in 64 bits from forms in which nothing cancels, and what an fp32 form may be off by.

    silu, z / (1 + exp(-z)): an exponential and a reciprocal of one step (2 EPS32) each, their arguments' and three more roundings: 8
    relative.  gelu: ten half steps of the tail by an emulation of its roundings, and the subtraction: 16.  gelu_tanh: as silu, with an
    argument of 2u = 1.5958 (z + 0.044715 z^3) that carries four roundings of its own, which the exponential turns into relative
    errors of the result, on the side where it does not saturate.  A factor below 2^-126 may be 0."""
    z = z.double()
    if act == "silu":
        return z / (1 + torch.exp(-z)), 8 * EPS32, z.abs()
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2)), 16 * EPS32, z.abs()
    u2 = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    return z / (1 + torch.exp(-u2)), (8 + 4 * (-u2).clamp(0, 100)) * EPS32, z.abs()


def check(y, z, act):
    want, rel, size = want_and_tol(z, act)
    tol = rel * want.abs() + 2.0 ** -126 * (1 + size)
    got = y.cpu().double()
    bad = ~(((got - want).abs() <= tol) | (got == want))
    if bad.any():
        i = int(torch.nonzero(bad)[0])
        raise AssertionError("%s: %d of %d, z = %r: got %r want %r" % (act, int(bad.sum()), len(z), z[i].item(), got[i].item(), want[i].item()))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_on_host(act):
    z = arguments()
    codes, grid = weights(torch.Generator().manual_seed(1), len(z), 1)
    y = dmm.decode_matmul_fused(torch.zeros(1, 8, dtype=F16), codes, grid, 1.0, bias=z, activation=act, out_dtype=F32)
    check(y[0], z, act)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_minus_infinity_and_nan_on_host(act):
    z = torch.tensor([-math.inf, math.nan])
    codes, grid = weights(torch.Generator().manual_seed(1), 2, 1)
    y = dmm.decode_matmul_fused(torch.zeros(1, 8, dtype=F16), codes, grid, 1.0, bias=z, activation=act, out_dtype=F32)
    assert torch.isnan(y).all()          # -inf times 0


# generic, few rows (a thread's four outputs; one after the other), matrix-matrix, split, tens of rows
@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("kernel,M", [(-1, 1), (0, 2), (1, 1), (1, 4), (1, 9), (2, 40), (3, 40), (5, 40)])
def test_on_gpu(act, kernel, M):
    z = arguments()
    codes, grid = weights(torch.Generator().manual_seed(1), len(z), 32)
    x = torch.zeros(M, 256, dtype=F16, device=DEV)
    capi.lib().dmm_set_ops_kernel(kernel)
    try:
        y = dmm.decode_matmul_fused(x, codes.to(DEV), grid.to(DEV), 1.0, bias=z.to(DEV), activation=act, out_dtype=F32)
        assert all(torch.equal(row, y[0]) for row in y)
        check(y[0], z, act)
        ends = torch.tensor([-math.inf, math.nan] * 8, device=DEV)
        y = dmm.decode_matmul_fused(x, codes[:16].contiguous().to(DEV), grid.to(DEV), 1.0, bias=ends, activation=act, out_dtype=F32)
        assert torch.isnan(y).all()
    finally:
        capi.lib().dmm_set_ops_kernel(-1)
