"""Calls of the operators around the product that the library refuses, or has to take, before any GPU call."""
import ctypes
import math

import pytest
import torch

import decode_matmul_amd as dmm
from decode_matmul_amd import capi
from ops_util import assert_within, combine64, decode64, fused_inputs, grouped64, grouped_inputs, product64

F16, F32 = torch.float16, torch.float32
OVERLAP = -10


# ----------------------------------------------------------------- a residual that overlaps the output
def test_residual_that_overlaps_the_output_is_refused():
    lib = capi.lib()
    buf = (ctypes.c_uint16 * 8192)()
    p = ctypes.addressof(buf)
    M, N, K = 4, 8, 16
    assert b"residual" in lib.dmm_status_string(OVERLAP)

    def fused(fn, residual, residual_type, y, out_type):
        e = capi.Epilogue(residual=residual, residual_type=residual_type, out_type=out_type, scale=1.0, scale_up=1.0)
        tail = (None, 0, None) if fn is lib.dmm_decode_matmul_fused else ()
        return fn(p, p + 1024, p + 2048, ctypes.byref(e), y, M, N, K, *tail)

    def combine(fn, residual, residual_type, out, out_type):
        tail = (None,) if fn is lib.dmm_combine_experts else ()
        return fn(p, 0, p + 1024, p + 2048, residual, residual_type, out, out_type, 4, M, 2, N, *tail)

    y = p + 8192
    for call, fns in ((fused, (lib.dmm_decode_matmul_fused, lib.dmm_decode_matmul_fused_host)),
                      (combine, (lib.dmm_combine_experts, lib.dmm_combine_experts_host))):
        for fn in fns:
            assert call(fn, y, 0, y, 1) == OVERLAP              # half elements under float ones
            assert call(fn, y, 1, y, 0) == OVERLAP
            assert call(fn, y + 2, 0, y, 0) == OVERLAP          # one element further on
            assert call(fn, y - 2 * M * N + 2, 0, y, 0) == OVERLAP
            assert call(fn, y + 4 * M * N - 2, 0, y, 1) == OVERLAP
        host = fns[1]
        assert call(host, y, 0, y, 0) == 0                      # the output itself
        assert call(host, y, 1, y, 1) == 0
        assert call(host, y + 2 * M * N, 0, y, 0) == 0          # side by side
        assert call(host, y - 2 * M * N, 0, y, 1) == 0


# ----------------------------------------------------------------- scales
def test_a_scale_that_is_nan_shows_in_the_result():
    x, codes, grid, _, _ = fused_inputs(2, 8, 64, False, None, None, seed=1)
    assert torch.isnan(dmm.decode_matmul_fused(x, codes, grid, math.nan)).all()
    y = dmm.decode_matmul_fused(x, codes, grid, (math.nan, 1.0), gated=True)
    assert torch.isnan(y).all() and y.shape == (2, 4)


def test_a_pair_of_scales_is_for_a_gated_call_whatever_its_values():
    x, codes, grid, _, _ = fused_inputs(2, 8, 64, False, None, None, seed=1)
    for pair in ((0.5, 0.5), [0.5, 0.25], (math.nan, math.nan)):
        with pytest.raises(RuntimeError, match="pair of scales is for a gated call"):
            dmm.decode_matmul_fused(x, codes, grid, pair)
    for bad in ((0.5,), (0.5, 0.5, 0.5), ()):
        with pytest.raises(RuntimeError, match="pair of scales is"):
            dmm.decode_matmul_fused(x, codes, grid, bad, gated=True)
    for pair in ((0.5, 0.25), [0.5, 0.25]):
        y = dmm.decode_matmul_fused(x, codes, grid, pair, gated=True, out_dtype=F32)
        assert_within(y, *product64(x.double(), decode64(codes, grid), pair, None, True, "none", None, F32))


# ----------------------------------------------------------------- gradients
def calls():
    """(name of the input, call with it replaced): every input that could carry a gradient."""
    x, codes, grid, b, r = fused_inputs(2, 8, 64, False, F16, F16, seed=1)
    gx, gcodes, ggrid, offsets, rows, gb = grouped_inputs((2, 3), 4, 8, 64, False, F16, True, seed=3)
    y, slots, w, res = torch.ones(4, 8, dtype=F16), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, 2), torch.ones(3, 8)
    fused = {"x": x, "grid": grid, "bias": b, "residual": r}
    for name, t in fused.items():
        def call(v, n=name):
            a = dict(fused, **{n: v})
            return dmm.decode_matmul_fused(a["x"], codes, a["grid"], 0.1, bias=a["bias"], residual=a["residual"])
        yield "fused", name, t, call
    grouped = {"x": gx, "grid": ggrid, "bias": gb, "scale": torch.ones(2), "out": torch.zeros(5, 8, dtype=F16)}
    for name, t in grouped.items():
        def call(v, n=name):
            a = dict(grouped, **{n: v})
            return dmm.decode_matmul_grouped(a["x"], gcodes, a["grid"], a["scale"], offsets, rows=rows, bias=a["bias"], out=a["out"])
        yield "grouped", name, t, call
    yield "route", "logits", torch.ones(3, 8), lambda v: dmm.route_experts(v, 2)
    combine = {"y": y, "weights": w, "residual": res}
    for name, t in combine.items():
        def call(v, n=name):
            a = dict(combine, **{n: v})
            return dmm.combine_experts(a["y"], slots, a["weights"], residual=a["residual"])
        yield "combine", name, t, call


CALLS = list(calls())


@pytest.mark.parametrize("op,name,t,call", CALLS, ids=["%s-%s" % c[:2] for c in CALLS])
def test_an_input_that_asks_for_a_gradient_is_refused(op, name, t, call):
    import torch.autograd.forward_ad as fwd
    call(t)
    with pytest.raises(RuntimeError, match="%s requires a gradient" % name):
        call(t.clone().requires_grad_())
    with torch.no_grad():
        call(t.clone().requires_grad_())
    with fwd.dual_level():
        dual = fwd.make_dual(t.clone(), torch.ones_like(t))
        with pytest.raises(RuntimeError, match="%s carries a tangent" % name):
            call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="%s carries a tangent" % name):      # tangents live on under it
            call(dual)
        call(fwd.unpack_dual(dual).primal)
        with torch.inference_mode():                                                                  # where they do not
            call(dual)
    if name != "out":                                          # torch.func's transforms: an error, never a wrong gradient
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda v: call(v), (t,), (torch.ones_like(t),))


def test_a_scale_tensor_that_asks_for_a_gradient_is_refused():
    import torch.autograd.forward_ad as fwd
    x, codes, grid, _, _ = fused_inputs(2, 8, 64, False, None, None, seed=1)
    s = torch.tensor(0.5, requires_grad=True)
    want = dmm.decode_matmul_fused(x, codes, grid, 0.5)
    for scale, gated in ((s, False), ((s, 0.5), True), ((0.5, s), True)):
        with pytest.raises(RuntimeError, match="scale requires a gradient"):
            dmm.decode_matmul_fused(x, codes, grid, scale, gated=gated)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="scale carries a tangent"):
        dmm.decode_matmul_fused(x, codes, grid, fwd.make_dual(s.detach(), torch.tensor(1.0)))
    with torch.no_grad():
        assert torch.equal(dmm.decode_matmul_fused(x, codes, grid, s), want)
    assert torch.equal(dmm.decode_matmul_fused(x, codes, grid, s.detach()), want)


def test_grouped_takes_a_pair_of_scales_as_fused_does():
    x, codes, grid, offsets, rows, b = grouped_inputs((2, 0, 3), 4, 8, 64, True, F16, True, seed=3)
    pair = (0.25, 0.125)
    y = dmm.decode_matmul_grouped(x, codes, grid, pair, offsets, rows=rows, bias=b, activation="silu", gated=True, out_dtype=F32)
    assert_within(y, *grouped64(x, codes, grid, torch.tensor([pair] * 3), offsets, rows, b, True, "silu", F32, 8))
    assert torch.equal(y, dmm.decode_matmul_grouped(x, codes, grid, torch.tensor([pair] * 3), offsets, rows=rows, bias=b, activation="silu", gated=True,
                                                    out_dtype=F32))
    with pytest.raises(RuntimeError, match="decode_matmul_grouped: a pair of scales is for a gated call"):
        dmm.decode_matmul_grouped(x, codes, grid, pair, offsets, rows=rows)
    with pytest.raises(RuntimeError, match="pair of scales is"):
        dmm.decode_matmul_grouped(x, codes, grid, (0.5,) * 3, offsets, rows=rows, gated=True)
    with pytest.raises(RuntimeError, match="scale must be"):
        dmm.decode_matmul_grouped(x, codes, grid, torch.ones(2), offsets, rows=rows, gated=True)


def test_grouped_out_counts_as_written():
    """A product that saved `out` for its gradient: an error afterwards, not a gradient of other values."""
    x, codes, grid, offsets, rows, _ = grouped_inputs((2, 3), 4, 8, 64, False, None, True, seed=3)
    out, w = torch.ones(5, 8, dtype=F16), torch.ones(5, 8, dtype=F16, requires_grad=True)
    product = (w * out).sum()
    dmm.decode_matmul_grouped(x, codes, grid, 0.1, offsets, rows=rows, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():
        out = torch.ones(5, 8, dtype=F16)
    dmm.decode_matmul_grouped(x, codes, grid, 0.1, offsets, rows=rows, out=out)          # has no version


def test_workspace_of_sizes_that_are_refused():
    """No split, so no workspace, for sizes the call itself refuses; their products do not fit 64 bits."""
    need = capi.lib().dmm_fused_workspace_bytes
    assert need(300, 4096, 11008, 0) > 0
    for M, N, K, gated in ((40, 16, 1 << 60, 1), (40, 16, (1 << 62) + 64, 0), (32, 1 << 62, 64, 1), (64, 1 << 31, 1 << 40, 0), (1 << 40, 64, 64, 0), (17, 16, 1 << 62, 1)):
        assert need(M, N, K, gated) == 0
