"""The operators around the product on host tensors, and everything that is refused: no GPU."""
import ctypes
import math

import pytest
import torch

import decode_matmul_amd as dmm
from decode_matmul_amd import capi
from ops_util import ACTS, assert_within, check_routing, combine64, decode64, fused_inputs, grouped64, grouped_inputs, product64

F16, F32 = torch.float16, torch.float32


# ----------------------------------------------------------------- the product with an epilogue
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K,bias,residual,out", [(1, 5, 8, None, None, F16), (3, 16, 64, F16, F32, F32), (2, 7, 264, F32, F16, F16),
                                                     (4, 1, 0, F32, None, F32)])
def test_fused_on_host(M, N, K, bias, residual, out, gated, act):
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, bias, residual, seed=M + N + K)
    scale = (0.125, 0.25) if gated else 0.125
    y = dmm.decode_matmul_fused(x, codes, grid, scale, bias=b, activation=act, gated=gated, residual=r, out_dtype=out)
    want, tol = product64(x.double(), decode64(codes, grid), scale if gated else (scale, scale), b, gated, act, r, out)
    assert y.dtype == out
    assert_within(y, want, tol)


def test_fused_without_epilogue_is_the_plain_product():
    x, codes, grid, _, _ = fused_inputs(3, 33, 520, False, None, None, seed=2)
    assert torch.equal(dmm.decode_matmul_fused(x, codes, grid, 0.1), dmm.decode_matmul(x, codes, grid, 0.1))


def test_fused_refusals():
    x, codes, grid, b, r = fused_inputs(2, 8, 64, False, F16, F16, seed=1)
    f = dmm.decode_matmul_fused
    for kw, match in (({"bias": b[:4]}, "bias"), ({"bias": b.double()}, "bias"), ({"residual": r[:1]}, "residual"),
                      ({"residual": r.to(torch.bfloat16)}, "residual"), ({"activation": "tanh"}, "activation"),
                      ({"out_dtype": torch.bfloat16}, "out_dtype"), ({"residual": r.t().contiguous().t()}, "contiguous")):
        with pytest.raises(RuntimeError, match=match):
            f(x, codes, grid, 1.0, **kw)
    with pytest.raises(RuntimeError, match="pair of scales"):
        f(x, codes, grid, (1.0, 2.0))
    with pytest.raises(RuntimeError, match="gated"):
        f(x, codes[:7].contiguous(), grid, 1.0, gated=True)
    with pytest.raises(RuntimeError, match="8 \\* codes"):
        f(x[:, :56].contiguous(), codes, grid, 1.0)
    with pytest.raises(RuntimeError, match="float16"):
        f(x.float(), codes, grid, 1.0)
    with pytest.raises(RuntimeError, match="contiguous"):
        f(x.repeat(1, 2)[:, ::2], codes, grid, 1.0)
    with pytest.raises(RuntimeError, match="gradient"):
        f(x, codes, grid, 1.0, bias=b.requires_grad_())
    with torch.no_grad():
        assert not f(x, codes, grid, 1.0, bias=b).requires_grad


# ----------------------------------------------------------------- by expert
@pytest.mark.parametrize("gated,act,gather,scale_kind", [(False, "none", False, "number"), (True, "silu", True, "per expert"),
                                                         (True, "gelu", False, "gate and up"), (False, "relu", True, "per expert")])
@pytest.mark.parametrize("counts", [(3,), (0, 2, 0, 1, 5), (0, 0), (1, 0)])
def test_grouped_on_host(counts, gated, act, gather, scale_kind):
    x, codes, grid, offsets, rows, b = grouped_inputs(counts, 6, 9, 72, gated, F32, gather, seed=len(counts), behind=2)
    E = len(counts)
    scale = {"number": 0.2, "per expert": torch.linspace(0.1, 0.3, E), "gate and up": torch.linspace(0.1, 0.4, 2 * E).view(E, 2)}[scale_kind]
    R = x.shape[0] if rows is None else rows.shape[0]
    out = torch.full((R, 9), math.nan, dtype=F16)
    y = dmm.decode_matmul_grouped(x, codes, grid, scale, offsets, rows=rows, bias=b, activation=act, gated=gated, out=out)
    assert y.data_ptr() == out.data_ptr()
    want, tol = grouped64(x, codes, grid, scale, offsets, rows, b, gated, act, F16, 9)
    assert_within(y, want, tol)            # rows that belong to no expert are still NaN


def test_grouped_lists_that_lead_out_of_the_buffers():
    x, codes, grid, offsets, rows, _ = grouped_inputs((2, 3), 4, 8, 64, False, None, True, seed=3)
    rows[1], rows[4] = -7, 4                                  # outside x: rows of zeros
    y = dmm.decode_matmul_grouped(x, codes, grid, 0.1, offsets, rows=rows)
    want, tol = grouped64(x, codes, grid, 0.1, offsets, rows, None, False, "none", F16, 8)
    assert_within(y, want, tol)
    assert torch.all(y[1] == 0) and torch.all(y[4] == 0)
    for broken in ([-3, 2, 5], [0, 9, 5], [0, 2, 500], [4, 1, 3], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        out = torch.zeros(5 + 2, 8, dtype=F16)
        dmm.decode_matmul_grouped(x, codes, grid, 0.1, torch.tensor(broken, dtype=torch.int32), rows=rows, out=out[1:6])
        assert torch.all(out[0] == 0) and torch.all(out[6] == 0)


def test_grouped_refusals():
    x, codes, grid, offsets, rows, b = grouped_inputs((2, 3), 4, 8, 64, False, F16, True, seed=3)
    f = dmm.decode_matmul_grouped
    for off in (offsets.long(), offsets[:2].contiguous(), offsets.view(1, -1)):
        with pytest.raises(RuntimeError, match="offsets"):
            f(x, codes, grid, 1.0, off, rows=rows)
    with pytest.raises(RuntimeError, match="rows"):
        f(x, codes, grid, 1.0, offsets, rows=rows.long())
    with pytest.raises(RuntimeError, match="scale"):
        f(x, codes, grid, torch.ones(3), offsets, rows=rows)
    with pytest.raises(RuntimeError, match="scale"):
        f(x, codes, grid, torch.ones(2, 2), offsets, rows=rows)       # a pair is for gated calls
    with pytest.raises(RuntimeError, match="bias"):
        f(x, codes, grid, 1.0, offsets, rows=rows, bias=b[0].contiguous())
    with pytest.raises(RuntimeError, match="codes must be \\[E"):
        f(x, codes[0].contiguous(), grid, 1.0, offsets, rows=rows)
    with pytest.raises(RuntimeError, match="out must be"):
        f(x, codes, grid, 1.0, offsets, rows=rows, out=torch.empty(5, 7, dtype=F16))
    with pytest.raises(RuntimeError, match="out must be"):
        f(x, codes, grid, 1.0, offsets, rows=rows, out=torch.empty(5, 8, dtype=F16), out_dtype=F32)
    with pytest.raises(RuntimeError, match="share memory"):
        f(x, codes, grid, 1.0, offsets, rows=rows, out=x.view(-1)[200:240].view(5, 8))
    with pytest.raises(RuntimeError, match="scale"):
        f(x, codes, grid, torch.ones(()), offsets, rows=rows)
    with pytest.raises(RuntimeError, match="gradient"):
        f(x, codes, grid, torch.ones(2, requires_grad=True), offsets, rows=rows)


# ----------------------------------------------------------------- choice of experts
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, F32), (5, 8, 2, F16), (70, 65, 7, torch.bfloat16), (0, 4, 2, F32), (3, 12, 12, F32)])
def test_route_on_host(T, E, k, dtype, scoring, normalize):
    gen = torch.Generator().manual_seed(T + E)
    logits = (torch.randn(T, E, generator=gen) * 2).to(dtype)
    if T > 4:
        logits[1] = -math.inf                 # a padded row
        logits[2, : E - 1] = -math.inf        # one expert left
        logits[3] = 0.5                       # all equal
        logits[4, ::2] = torch.finfo(dtype).min   # a mask of the type's lowest value is a number
    check_routing(dmm.route_experts(logits, k, scoring=scoring, normalize=normalize), logits, k, scoring, normalize)


def test_route_zeros_of_both_signs_are_equal_and_nan_shows():
    z = torch.tensor([[0.0, -0.0, 0.0, -1.0], [-0.0, 0.0, -0.0, 3.0]])
    assert dmm.route_experts(z, 3).experts.tolist() == [[0, 1, 2], [3, 0, 1]]
    r = dmm.route_experts(torch.tensor([[1.0, math.nan, 2.0], [1.0, 0.0, 2.0]]), 3)
    assert r.experts.tolist() == [[2, 0, -1], [2, 0, 1]]
    assert torch.isnan(r.weights[0]).all() and torch.isfinite(r.weights[1]).all()


def test_route_sigmoids_too_small_for_a_float_still_have_shares():
    gen = torch.Generator().manual_seed(7)
    z = torch.randn(6, 9, generator=gen) * 5 - torch.tensor([0.0, 60, 90, 200, 400, 600]).view(6, 1)
    check_routing(dmm.route_experts(z, 4, scoring="sigmoid"), z, 4, "sigmoid", True)
    for dtype in (F16, F32, torch.bfloat16):        # a row that a mask of the type's lowest value covers: equal shares
        w = dmm.route_experts(torch.full((2, 5), torch.finfo(dtype).min, dtype=dtype), 4, scoring="sigmoid").weights
        assert torch.equal(w, torch.full((2, 4), 0.25))


def test_route_refusals():
    z = torch.zeros(3, 8)
    for k in (0, 9, -1):
        with pytest.raises(RuntimeError, match="k must"):
            dmm.route_experts(z, k)
    with pytest.raises(RuntimeError, match="k must"):
        dmm.route_experts(torch.zeros(2, 1025), 2)
    with pytest.raises(RuntimeError, match="scoring"):
        dmm.route_experts(z, 2, scoring="top")
    with pytest.raises(RuntimeError, match="logits"):
        dmm.route_experts(z.double(), 2)
    with pytest.raises(RuntimeError, match="contiguous"):
        dmm.route_experts(z.t(), 2)
    with pytest.raises(RuntimeError, match="tokens"):
        dmm.route_experts(torch.zeros(2 ** 24 + 1, 1, dtype=F16), 1)
    with pytest.raises(RuntimeError, match="gradient"):
        dmm.route_experts(z.requires_grad_(), 2)


# ----------------------------------------------------------------- weighted sum
@pytest.mark.parametrize("y_type,residual,out", [(F16, None, F16), (F16, F16, F32), (F32, F32, F16)])
@pytest.mark.parametrize("T,k,N,R", [(1, 1, 1, 1), (5, 3, 37, 11), (4, 2, 8, 0), (2, 0, 5, 3), (0, 2, 5, 3)])
def test_combine_on_host(T, k, N, R, y_type, residual, out):
    gen = torch.Generator().manual_seed(T * 10 + N)
    y = torch.randn(R, N, generator=gen).to(y_type)
    slots = torch.randint(-2, R + 2, (T, k), generator=gen, dtype=torch.int32)      # some outside y
    w = torch.rand(T, k, generator=gen)
    w[slots < 0] = math.inf                   # the weight of a slot outside is not looked at
    r = torch.randn(T, N, generator=gen).to(residual) if residual else None
    got = dmm.combine_experts(y, slots, w, residual=r, out_dtype=out)
    assert got.dtype == out
    assert_within(got, *combine64(y, slots, w, r, out))


def test_combine_refusals():
    y, s, w = torch.zeros(4, 8, dtype=F16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    f = dmm.combine_experts
    with pytest.raises(RuntimeError, match="slots"):
        f(y, s.long(), w)
    with pytest.raises(RuntimeError, match="weights"):
        f(y, s, w.half())
    with pytest.raises(RuntimeError, match="weights"):
        f(y, s, torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="residual"):
        f(y, s, w, residual=torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="y must"):
        f(y.to(torch.bfloat16), s, w)
    with pytest.raises(RuntimeError, match="gradient"):
        f(y, s, w.requires_grad_())


# ----------------------------------------------------------------- the C ABI's own checks: a status, before any GPU call
def test_status_codes_of_the_operators_around_the_product():
    lib = capi.lib()
    buf = (ctypes.c_uint16 * 4096)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    odd = ctypes.c_void_p(p.value + 1)

    def ep(**kw):
        e = capi.Epilogue(scale=1.0, scale_up=1.0)
        for name, v in kw.items():
            setattr(e, name, v)
        return ctypes.byref(e)

    fused = lib.dmm_decode_matmul_fused
    assert fused(p, p, p, ep(), p, 1, 4, 12, None, 0, None) == -2            # K % 8
    assert fused(p, p, p, ep(), p, -1, 4, 16, None, 0, None) == -2
    assert fused(p, p, p, None, p, 1, 4, 16, None, 0, None) == -1
    assert fused(p, p, None, ep(), p, 1, 4, 16, None, 0, None) == -1
    assert fused(p, p, p, ep(), None, 1, 4, 16, None, 0, None) == -1
    assert fused(odd, p, p, ep(), p, 1, 4, 16, None, 0, None) == -3
    assert fused(p, p, p, ep(bias=odd.value), p, 1, 4, 16, None, 0, None) == -3
    assert fused(p, p, p, ep(out_type=1), ctypes.c_void_p(p.value + 2), 1, 4, 16, None, 0, None) == -3
    assert fused(p, p, p, ep(activation=5), p, 1, 4, 16, None, 0, None) == -2
    assert fused(p, p, p, ep(out_type=2), p, 1, 4, 16, None, 0, None) == -2  # bfloat16 is for logits only
    assert fused(p, p, p, ep(), p, 1, 1 << 31, 16, None, 0, None) == -4
    assert fused(p, p, p, ep(), p, (1 << 30) + 1, 4, 16, None, 0, None) == -4
    assert fused(p, p, p, ep(), p, 1, 4, 16, ctypes.c_void_p(p.value + 4), 64, None) == -3
    assert fused(p, p, p, ep(), p, 1, 4, 16, p, -1, None) == -2
    assert fused(None, None, None, ep(), None, 0, 4, 16, None, 0, None) == 0
    grouped = lib.dmm_decode_matmul_grouped
    assert grouped(p, 3, p, p, p, None, 1, p, ep(residual=p.value), p, 4, 2, 4, 16, None) == -2
    assert grouped(p, 3, None, p, p, None, 1, p, ep(), p, 4, 2, 4, 16, None) == -2      # no rows: T has to be R
    assert grouped(p, 3, p, p, p, p, 2, p, ep(), p, 4, 2, 4, 16, None) == -2            # a pair of scales, not gated
    assert grouped(p, 3, p, p, p, None, 1, None, ep(), p, 4, 2, 4, 16, None) == -1
    assert grouped(p, 3, p, p, p, None, 1, odd, ep(), p, 4, 2, 4, 16, None) == -3
    assert grouped(p, 3, p, p, p, None, 1, p, ep(), p, 4, 65536, 4, 16, None) == -4
    assert grouped(p, 3, p, p, p, None, 1, p, ep(), p, (1 << 30) + 1, 2, 4, 16, None) == -4
    assert grouped(p, (1 << 30) + 1, p, p, p, None, 1, p, ep(), p, 4, 2, 4, 16, None) == -4
    assert grouped(None, 0, None, None, None, None, 1, None, ep(), None, 0, 2, 4, 16, None) == 0
    route = lib.dmm_route_experts
    assert route(p, 1, 3, 8, 9, 0, 1, p, p, p, p, p, None, 0, None) == -2
    assert route(p, 3, 3, 8, 2, 0, 1, p, p, p, p, p, None, 0, None) == -2
    assert route(p, 1, 3, 8, 2, 2, 1, p, p, p, p, p, None, 0, None) == -2
    assert route(p, 1, 3, 2000, 2, 0, 1, p, p, p, p, p, None, 0, None) == -4
    assert route(p, 1, 3, 8, 2, 0, 1, p, p, None, p, p, None, 0, None) == -1
    assert route(p, 1, 3, 8, 2, 0, 1, odd, p, p, p, p, None, 0, None) == -3
    assert route(p, 1, (1 << 24) + 1, 8, 2, 0, 1, p, p, p, p, p, None, 0, None) == -4
    need = lib.dmm_route_workspace_bytes(100, 8)
    assert need > 0 and lib.dmm_route_workspace_bytes(64, 8) == 0 and lib.dmm_route_workspace_bytes(-1, 8) == 0
    assert route(p, 1, 100, 8, 2, 0, 1, p, p, p, p, p, None, 0, None) == -1
    assert route(p, 1, 100, 8, 2, 0, 1, p, p, p, p, p, p, need - 1, None) == -8
    combine = lib.dmm_combine_experts
    assert combine(p, 2, p, p, None, 0, p, 0, 4, 3, 2, 8, None) == -2
    assert combine(p, 0, p, p, None, 0, None, 0, 4, 3, 2, 8, None) == -1
    assert combine(p, 0, odd, p, None, 0, p, 0, 4, 3, 2, 8, None) == -3
    assert combine(p, 0, p, p, odd, 0, p, 0, 4, 3, 2, 8, None) == -3
    assert combine(p, 0, p, p, None, 0, p, 0, -4, 3, 2, 8, None) == -2
    assert combine(None, 0, None, None, None, 0, None, 0, 4, 0, 2, 8, None) == 0
    assert lib.dmm_fused_workspace_bytes(-1, 8, 64, 0) == 0


def test_no_vector_instruction_is_written_as_inline_assembly():
    """The compiler keeps the distance between a matrix instruction and a vector one that writes its C operand only
    for instructions that it knows; four of the library's kernels had none left between the two."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(capi.LIB_PATH), "csrc")
    for name in sorted(os.listdir(csrc)):
        text = open(os.path.join(csrc, name)).read()
        assert not re.search(r'asm\s*(volatile)?\s*\(\s*"\s*v_', text), name
