"""The inputs for the kernels on 8-bit operands see every part of the arithmetic: planted in the emulation, on the CPU."""
import numpy as np
import pytest
import torch

import decode_matmul_amd as dmm
from ops_terms import Case, cancelling, means, terms
from ops_util import decode64


def test_terms_and_means_of_halves():
    x = np.random.default_rng(0).standard_normal((3, 64)).astype(np.float16)
    x[0, :4] = [65504, -65504, 0.0, 1 + 2.0 ** -10]
    assert np.array_equal(sum(terms(x)), x.astype(np.float64))
    hi, lo = means(x)
    exact = x.astype(np.float64).reshape(3, 8, 8).mean(-1)
    assert np.all(np.abs(hi + lo - exact) <= 2.0 ** -22 * np.abs(exact) + 2.0 ** -24)


# (K, first code, codes): all of K; and a window of 256 k at the start, inside, and at the end of a long one
WINDOWS = [(256, 0, None), (64, 0, None), (2048, 0, None), (8192, 0, 32), (8192, 500, 32), (8192, 992, 32), (4096, 0, None)]


@pytest.mark.parametrize("K,first,count", WINDOWS)
@pytest.mark.parametrize("M", [1, 2])
def test_a_dropped_term_shows(M, K, first, count):
    c = Case(M, 12, K, K + first + M, first, count)
    w = decode64(c.codes, c.grid)
    assert torch.equal(c.x.double() @ w.t(), c.sum.expand(M, -1))          # the same products, in one piece
    b, left = cancelling(c)
    assert torch.all((c.emulate() + b - left).abs() <= c.tol())
    for drop in ("t0", "t1", "t2", "t3", "hi", "lo"):
        if c.used > {"lo": 256, "t3": 2048}.get(drop, 1 << 30):
            continue                                                     # below the bound of so long a sum
        off = (c.emulate(drop) + b - left).abs()
        assert torch.all(off > 1.15 * c.tol()), (drop, float((off / c.tol()).min()))
    # the host route has sums of exact products
    y = dmm.decode_matmul_fused(c.x, c.codes, c.grid, 1.0, bias=b, out_dtype=torch.float32)
    assert torch.all((y.double() - left).abs() <= c.tol())
