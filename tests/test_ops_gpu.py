"""The operators around the product on the GPU, against 64 bits, at the sizes and lists where they can go wrong."""
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
def sixteen_bit_operands():
    """Sums of exact products unless a test asks for 8-bit operands."""
    before = capi.lib().dmm_set_gemv_8bit(0)
    yield
    capi.lib().dmm_set_gemv_8bit(before)


@pytest.fixture(params=[-1, 1, 2, 3, 4, 5], ids=["auto", "rows", "gemm", "split", "rows8", "mid"])
def kernel(request):
    """The library's choice, and every kernel in its place where it can take the call."""
    lib = capi.lib()
    lib.dmm_set_ops_kernel(request.param)
    yield request.param
    lib.dmm_set_ops_kernel(-1)


def check_fused(M, N, K, gated=False, act="none", bias=None, residual=None, out=F16, seed=0, fp8=True, scale=None, kernel=-1):
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, bias, residual, seed + M + N + K, fp8=fp8, coarse=kernel == 4)
    s = 1.0 / math.sqrt(max(K, 1)) if scale is None else scale
    xd, cd, gd, bd, rd = dev(x, codes, grid, b, r)
    y = dmm.decode_matmul_fused(xd, cd, gd, s, bias=bd, activation=act, gated=gated, residual=rd, out_dtype=out)
    torch.cuda.synchronize()
    assert y.dtype == out and tuple(y.shape) == (M, N)
    want, tol = product64(x.double(), decode64(codes, grid), s if isinstance(s, tuple) else (s, s), b, gated, act, r, out)
    assert_within(y, want, tol, "M=%d N=%d K=%d" % (M, N, K))
    return y


# ----------------------------------------------------------------- the product with an epilogue
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (2, 5, 24), (3, 33, 264), (5, 7, 0)])
@pytest.mark.parametrize("gated", [False, True])
def test_fused_any_shape(M, N, K, gated):
    check_fused(M, N, K, gated, "silu", F32, F16, F32)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bias,residual,out", [(None, None, F16), (F16, F32, F16), (F32, F16, F32), (None, F16, F16)])
def test_fused_epilogues(act, gated, bias, residual, out, kernel):
    check_fused(1, 272, 512, gated, act, bias, residual, out, kernel=kernel)
    check_fused(7, 272, 512, gated, act, bias, residual, out, kernel=kernel)
    check_fused(40, 272, 512, gated, act, bias, residual, out, kernel=kernel)


@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("N,K,gated", [(64, 256, False), (100, 768, True), (17, 320, False), (1030, 1024, True), (515, 2112, False)])
def test_fused_rows(M, N, K, gated, kernel):
    check_fused(M, N, K, gated, "gelu_tanh", F16, None, F16, kernel=kernel)


def test_fused_gate_and_up_scales():
    check_fused(3, 64, 256, True, "silu", F32, None, F32, scale=(0.06, 0.11))
    check_fused(50, 64, 256, True, "silu", F32, None, F32, scale=(0.06, 0.11))


@pytest.mark.parametrize("M", [1, 3, 40])
def test_fused_grid_that_does_not_fit_8_bits(M, kernel):
    check_fused(M, 4240, 512, False, "relu", F16, F16, F16, fp8=False)
    check_fused(M, 2128, 512, True, "silu", F16, F16, F16, fp8=False)
    check_fused(M, 40000, 256, False, "none", None, None, F16, fp8=False)


@pytest.mark.parametrize("M,N,K,gated", [(1, 4096, 4096, False), (2, 4128, 11008, False), (1, 5504, 4096, True), (2, 40004, 512, False),
                                         (1, 20000, 512, True), (2, 8200, 320, True), (1, 16400, 8192, False)])
@pytest.mark.parametrize("coarse", [True, False])
def test_fused_on_8_bit_operands(M, N, K, gated, coarse):
    """The library's own choice for one or two rows: the exact products' bound where every sum is exact on 8-bit operands
    too, the plain product's tolerance on them (1e-2 of z and of its unit) for normal x."""
    capi.lib().dmm_set_gemv_8bit(1)
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, F16, F16, M + N + K, coarse=coarse)
    s = 1.0 / math.sqrt(K)
    xd, cd, gd, bd, rd = dev(x, codes, grid, b, r)
    y = dmm.decode_matmul_fused(xd, cd, gd, s, bias=bd, activation="silu" if gated else "none", gated=gated, residual=rd)
    want, tol = product64(x.double(), decode64(codes, grid), (s, s), b, gated, "silu" if gated else "none", r, F16)
    if not coarse:
        z = (x.double() @ decode64(codes, grid).t() * s + b.double()).abs()
        e = 1e-2 * (1 + z)
        tol = tol + (1.13 * e[:, :N] * (z[:, N:] + e[:, N:]) + z[:, :N] * e[:, N:] if gated else e)
    assert_within(y, want, tol)


def test_grouped_on_8_bit_operands_and_x_that_is_not_finite():
    """Many jobs per workgroup, some with an infinity: those rows, and no others, are not finite."""
    capi.lib().dmm_set_gemv_8bit(1)
    capi.lib().dmm_set_ops_kernel(4)
    try:
        for gated in (False, True):
            counts = (1, 0, 2, 3, 1)
            x, codes, grid, offsets, rows, b = grouped_inputs(counts, 4, 9000, 768, gated, F16, True, 5, coarse=True)
            x[2, 700] = math.inf
            rows[:7] = torch.tensor([0, 1, 2, 3, 2, 0, 1], dtype=torch.int32)
            y = dmm.decode_matmul_grouped(*dev(x, codes, grid), 0.03, offsets.to(DEV), rows=rows.to(DEV), bias=b.to(DEV), gated=gated)
            want, tol = grouped64(x, codes, grid, 0.03, offsets, rows, b, gated, "none", F16, 9000)
            bad = rows == 2
            assert_within(y[~bad.to(DEV)], want[~bad], tol[~bad])
            assert not torch.isfinite(y[bad.to(DEV)]).any()
            assert torch.equal(torch.isnan(y[bad.to(DEV)]).cpu(), torch.isnan(want[bad]))
    finally:
        capi.lib().dmm_set_ops_kernel(-1)


@pytest.mark.parametrize("M", [1, 4, 16, 40])
def test_fused_x_that_is_not_finite_stays_in_its_row(M, kernel):
    x, codes, grid, _, _ = fused_inputs(M, 4240, 512, False, None, None, seed=5, coarse=kernel == 4)
    x[M - 1, 500] = math.inf
    y = dmm.decode_matmul_fused(*dev(x, codes, grid), 0.05)
    want, tol = product64(x.double(), decode64(codes, grid), (0.05, 0.05), None, False, "none", None, F16)
    tol[M - 1] = math.inf
    assert_within(y, want, tol)
    assert not torch.isfinite(y[M - 1]).any()      # inf times a weight: inf, or NaN for a weight of 0


def test_fused_activations_at_the_ends():
    """z from the bias alone (x = 0): large, infinite and tiny arguments of every activation."""
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-4, -1e-4, 5.0, -5.0, 20.0, -20.0, 87.0, -87.0, 90.0, -90.0, 200.0, -200.0, 6e4,
                      -6e4, 3e38, math.inf], dtype=F32)
    K = 256
    codes, grid = weights(torch.Generator().manual_seed(1), len(z), K // 8)
    x = torch.zeros(2, K, dtype=F16)
    for act in ACTS:
        y = dmm.decode_matmul_fused(*dev(x, codes, grid), 1.0, bias=z.to(DEV), activation=act, out_dtype=F32).cpu()
        zz = z.double()
        want = {"none": zz, "relu": zz.clamp(min=0), "silu": zz / (1 + torch.exp(-zz)), "gelu": zz * 0.5 * torch.erfc(-zz / math.sqrt(2)),
                "gelu_tanh": 0.5 * zz * (1 + torch.tanh(math.sqrt(2 / math.pi) * (zz + 0.044715 * zz ** 3)))}[act]
        # 8 roundings of the argument's size; results below the smallest normal number may be 0
        assert_within(y[0], want, 8 * 2.0 ** -24 * zz.abs().clamp(max=1e300) + 2.0 ** -120, act)
        assert torch.equal(y[0], y[1])


def test_fused_residual_may_be_the_output():
    x, codes, grid, b, r = fused_inputs(5, 48, 256, False, F16, F16, seed=9)
    xd, cd, gd, bd, rd = dev(x, codes, grid, b, r)
    want = dmm.decode_matmul_fused(xd, cd, gd, 0.1, bias=bd, activation="gelu", residual=rd)
    ep = capi.Epilogue(bias=bd.data_ptr(), residual=rd.data_ptr(), activation=3, scale=0.1, scale_up=0.1)
    capi.check("fused", capi.lib().dmm_decode_matmul_fused(xd.data_ptr(), cd.data_ptr(), gd.data_ptr(), ctypes.byref(ep), rd.data_ptr(),
                                                           5, 48, 256, None, 0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(rd, want)


@pytest.mark.parametrize("M,N,K", [(1, 64, 256), (12, 64, 256), (70, 64, 256)])
def test_fused_buffers_at_odd_places(M, N, K):
    """Views that start two bytes (half) or four (float) into their storage."""
    x, codes, grid, b, r = fused_inputs(M, N, K, False, F32, F16, seed=4)
    want, tol = product64(x.double(), decode64(codes, grid), (0.1, 0.1), b, False, "silu", r, F16)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:].copy_(t.flatten())
        return flat[1:].view(t.shape)

    for which in range(5):
        args = [shifted(t) if i == which else t.to(DEV) for i, t in enumerate((x, codes, grid, b, r))]
        y = dmm.decode_matmul_fused(*args[:3], 0.1, bias=args[3], activation="silu", residual=args[4])
        assert_within(y, want, tol, "operand %d" % which)


# ----------------------------------------------------------------- by expert
def check_grouped(counts, T, N, K, gated=False, act="none", bias=None, gather=True, behind=0, out=F16, scale=None, seed=0,
                  kernel=-1):
    x, codes, grid, offsets, rows, b = grouped_inputs(counts, T, N, K, gated, bias, gather, seed + N + K, behind, coarse=kernel == 4)
    s = 1.0 / math.sqrt(K) if scale is None else scale
    R = x.shape[0] if rows is None else rows.shape[0]
    y = torch.full((R, N), math.nan, dtype=out, device=DEV)
    dmm.decode_matmul_grouped(*dev(x, codes, grid), s.to(DEV) if isinstance(s, torch.Tensor) else s, offsets.to(DEV), rows=dev(rows)[0],
                              bias=dev(b)[0], activation=act, gated=gated, out=y)
    torch.cuda.synchronize()
    want, tol = grouped64(x, codes, grid, s, offsets, rows, b, gated, act, out, N)
    assert_within(y, want, tol, "counts=%s N=%d K=%d" % (str(counts)[:60], N, K))


COUNTS = [(1,), (0, 1), (3, 0, 0, 4, 1), (0, 0, 0), (17, 1, 0, 33, 5, 16), (1,) * 70, (0,) * 65 + (9,) + (0,) * 66, (100, 3, 70),
          (300, 0, 1, 130)]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("N,K,gated", [(64, 256, False), (36, 512, True), (21, 320, False), (272, 1024, True)])
def test_grouped(counts, N, K, gated, kernel):
    check_grouped(counts, 11, N, K, gated, "silu" if gated else "none", F16 if gated else None, gather=True, behind=3, kernel=kernel)


@pytest.mark.parametrize("counts", [(3, 0, 0, 4, 1), (40, 0, 25)])
@pytest.mark.parametrize("K", [8, 24, 264, 64, 4096])
def test_grouped_row_order_and_types(counts, K, kernel):
    E = len(counts)
    check_grouped(counts, 5, 20, K, False, "gelu", F32, gather=False, behind=1, out=F32, scale=torch.linspace(0.02, 0.05, E), kernel=kernel)
    check_grouped(counts, 5, 20, K, True, "relu", F16, gather=True, out=F32, scale=torch.linspace(0.02, 0.05, 2 * E).view(E, 2), kernel=kernel)


def test_grouped_many_tiles_per_workgroup(kernel):
    check_grouped((2, 0, 1, 19), 9, 8200, 256, False, "none", None, kernel=kernel)
    check_grouped((2, 0, 1, 19), 9, 4100, 512, True, "silu", None, kernel=kernel)
    check_grouped((1,), 3, 33000, 256, False, "none", None, kernel=kernel)


def test_grouped_lists_that_lead_out_of_the_buffers(kernel):
    for counts in ((2, 3), (90, 60)):
        x, codes, grid, offsets, rows, _ = grouped_inputs(counts, 4, 64, 256, False, None, True, seed=3, coarse=kernel == 4)
        R = rows.shape[0]
        rows[1], rows[R - 1] = -7, 4                               # outside x: rows of zeros
        xd, cd, gd, od, rd = dev(x, codes, grid, offsets, rows)
        y = dmm.decode_matmul_grouped(xd, cd, gd, 0.1, od, rows=rd)
        want, tol = grouped64(x, codes, grid, 0.1, offsets, rows, None, False, "none", F16, 64)
        assert_within(y, want, tol)
        for broken in ([-3, 2, R], [0, 9 * R, R], [0, 2, 500000], [4, 1, 3], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
            out = torch.zeros(R + 2, 64, dtype=F16, device=DEV)
            dmm.decode_matmul_grouped(xd, cd, gd, 0.1, torch.tensor(broken, dtype=torch.int32, device=DEV), rows=rd, out=out[1:R + 1])
            torch.cuda.synchronize()
            assert torch.all(out[0] == 0) and torch.all(out[-1] == 0)


def test_grouped_rows_of_others_may_hold_anything():
    """NaN and infinities in the rows of x of one expert and behind the last one reach no other expert's rows."""
    for counts in ((3, 2, 5), (40, 3, 70), (300, 10, 200)):
        for kernel in (-1, 1, 2, 4, 5):
            capi.lib().dmm_set_ops_kernel(kernel)
            try:
                x, codes, grid, offsets, _, _ = grouped_inputs(counts, 0, 52, 320, False, None, False, seed=8, behind=9, coarse=True)
                lo, hi = int(offsets[1]), int(offsets[2])
                x[lo:hi] = math.nan
                x[int(offsets[3]):] = math.inf
                y = dmm.decode_matmul_grouped(*dev(x, codes, grid), 0.1, offsets.to(DEV))
                want, tol = grouped64(x, codes, grid, 0.1, offsets, None, None, False, "none", F16, 52)
                keep = torch.ones(x.shape[0], dtype=torch.bool)
                keep[lo:hi] = False
                keep[int(offsets[3]):] = False
                assert_within(y.cpu()[keep], want[keep], tol[keep], "kernel %d" % kernel)
                assert torch.isnan(y[lo:hi]).all()
            finally:
                capi.lib().dmm_set_ops_kernel(-1)


def test_grouped_empty():
    x, codes, grid, offsets, rows, _ = grouped_inputs((0, 0), 4, 64, 256, False, None, True, seed=3)
    assert dmm.decode_matmul_grouped(*dev(x, codes, grid), 0.1, offsets.to(DEV), rows=rows.to(DEV)).shape == (0, 64)
    e = torch.empty(0, 256, dtype=F16, device=DEV)
    rows = torch.zeros(3, dtype=torch.int32, device=DEV)           # x has no rows: every entry points outside
    y = dmm.decode_matmul_grouped(e, *dev(codes, grid), 0.1, torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV), rows=rows)
    assert torch.all(y == 0)


# ----------------------------------------------------------------- choice of experts
@pytest.mark.parametrize("scoring,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("T,E,k,dtype", [(1, 1, 1, F32), (5, 8, 2, F16), (64, 64, 6, F32), (65, 65, 7, torch.bfloat16), (3, 12, 12, F32),
                                         (200, 128, 8, F16), (300, 257, 5, F32), (70, 1000, 64, F16), (130, 600, 3, F32),
                                         (90, 16, 16, F16), (67, 30, 17, F32), (61, 200, 16, F32), (63, 100, 40, F16), (66, 40, 4, F16)])
def test_route(T, E, k, dtype, scoring, normalize):
    gen = torch.Generator().manual_seed(T + E)
    logits = (torch.randn(T, E, generator=gen) * 2).to(dtype)
    if T > 4:
        logits[1] = -math.inf
        logits[2, : E - 1] = -math.inf
        logits[3] = 0.5
        logits[4, ::2] = torch.finfo(dtype).min
    check_routing(dmm.route_experts(logits.to(DEV), k, scoring=scoring, normalize=normalize), logits, k, scoring, normalize)


def test_route_sigmoids_too_small_for_a_float_still_have_shares():
    gen = torch.Generator().manual_seed(7)
    for E, k in ((9, 4), (300, 20)):
        z = torch.randn(6, E, generator=gen) * 5 - torch.tensor([0.0, 60, 90, 200, 400, 600]).view(6, 1)
        check_routing(dmm.route_experts(z.to(DEV), k, scoring="sigmoid"), z, k, "sigmoid", True)
    for dtype in (F16, F32, torch.bfloat16):
        w = dmm.route_experts(torch.full((2, 5), torch.finfo(dtype).min, dtype=dtype, device=DEV), 4, scoring="sigmoid").weights
        assert torch.equal(w.cpu(), torch.full((2, 4), 0.25))


def test_grouped_lists_that_give_every_expert_all_rows(kernel):
    """A list that does not increase: rows of several experts, written by each of them; every one stays inside y."""
    R, E, N, K = 70, 40, 52, 320
    x, codes, grid, _, rows, _ = grouped_inputs((2,) * 35 + (0,) * 5, 9, N, K, True, None, True, seed=5, coarse=True)
    out = torch.zeros(R + 2, N, dtype=F16, device=DEV)
    broken = torch.tensor(([0, R] * E)[:E + 1], dtype=torch.int32, device=DEV)
    dmm.decode_matmul_grouped(*dev(x, codes, grid), 0.1, broken, rows=rows.to(DEV), gated=True, out=out[1:R + 1])
    torch.cuda.synchronize()
    assert torch.all(out[0] == 0) and torch.all(out[-1] == 0)
    # which matrix gives an element its value is not said: one of those whose range is not empty.  Both sides are rounded once
    # (2 x 2^-11); the fp32 sums of a few hundred products, of either order, are far nearer than 1e-3.
    got, near = out[1:R + 1].float(), torch.zeros(R, N, dtype=torch.bool, device=DEV)
    for c in codes.to(DEV)[::2]:
        want = dmm.decode_matmul_fused(x.to(DEV)[rows.to(DEV).long()], c, grid.to(DEV), 0.1, gated=True).float()
        near |= (got - want).abs() <= 2.0 ** -10 * want.abs() + 1e-3
    assert near.all()


def test_route_many_tokens_against_the_host_route():
    """More than one block, one and several words per expert's mask; the lists equal the host's bit for bit."""
    for T, E, k in ((5000, 16, 2), (33000, 40, 3), (140000, 8, 2)):
        gen = torch.Generator().manual_seed(T)
        logits = torch.randn(T, E, generator=gen)
        logits[torch.randperm(T, generator=gen)[: T // 9]] = -math.inf
        want, got = dmm.route_experts(logits, k), dmm.route_experts(logits.to(DEV), k)
        for name in ("experts", "offsets", "rows", "slots"):
            assert torch.equal(getattr(got, name).cpu(), getattr(want, name)), (T, name)


def test_route_no_tokens_zeros_of_both_signs_and_nan():
    r = dmm.route_experts(torch.zeros(0, 9, device=DEV), 2)
    assert r.offsets.tolist() == [0] * 10 and r.weights.shape == (0, 2)
    z = torch.tensor([[0.0, -0.0, 0.0, -1.0], [-0.0, 0.0, -0.0, 3.0]], device=DEV)
    assert dmm.route_experts(z, 3).experts.tolist() == [[0, 1, 2], [3, 0, 1]]
    for scoring in ("softmax", "sigmoid"):
        r = dmm.route_experts(torch.tensor([[1.0, math.nan, 2.0], [1.0, 0.0, 2.0]], device=DEV), 3, scoring=scoring)
        assert r.experts.tolist() == [[2, 0, -1], [2, 0, 1]]
        assert torch.isnan(r.weights[0]).all() and torch.isfinite(r.weights[1]).all()


# ----------------------------------------------------------------- weighted sum
@pytest.mark.parametrize("y_type,residual,out", [(F16, None, F16), (F16, F16, F32), (F32, F32, F16), (F16, F16, F16)])
@pytest.mark.parametrize("T,k,N,R", [(1, 1, 1, 1), (5, 3, 37, 11), (4, 2, 8, 0), (2, 0, 5, 3), (33, 8, 4096, 100), (3, 2, 2050, 6), (0, 2, 5, 3),
                                     (70000, 1, 3, 10)])
def test_combine(T, k, N, R, y_type, residual, out):
    gen = torch.Generator().manual_seed(T * 10 + N)
    y = torch.randn(R, N, generator=gen).to(y_type)
    slots = torch.randint(-2, R + 2, (T, k), generator=gen, dtype=torch.int32)
    w = torch.rand(T, k, generator=gen)
    w[slots < 0] = math.inf
    r = torch.randn(T, N, generator=gen).to(residual) if residual else None
    yd, sd, wd, rd = dev(y, slots, w, r)
    got = dmm.combine_experts(yd, sd, wd, residual=rd, out_dtype=out)
    torch.cuda.synchronize()
    assert_within(got, *combine64(y, slots, w, r, out))


# ----------------------------------------------------------------- together, as a layer uses them
def moe_layer(x, logits, k, up, down, grid, N, H):
    r = dmm.route_experts(logits, k)
    h = dmm.decode_matmul_grouped(x, up, grid, 1 / math.sqrt(H), r.offsets, rows=r.rows, activation="silu", gated=True)
    o = dmm.decode_matmul_grouped(h, down, grid, 1 / math.sqrt(N), r.offsets)
    return r, h, o, dmm.combine_experts(o, r.slots, r.weights, residual=x)


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (24, 8, 2), (200, 16, 3)])
def test_a_layer_of_experts_with_padded_tokens(T, E, k):
    H, N = 512, 768
    gen = torch.Generator().manual_seed(T)
    up, grid = weights(gen, E, 2 * N, H // 8)
    down, _ = weights(gen, E, H, N // 8)
    x = torch.randn(T, H, generator=gen).half()
    logits = torch.randn(T, E, generator=gen)
    if T > 3:
        logits[-3:] = -math.inf
    xd, ld, ud, dd, gd = dev(x, logits, up, down, grid)
    r, h, o, y = moe_layer(xd, ld, k, ud, dd, gd, N, H)
    check_routing(r, logits, k, "softmax", True)
    off, live = r.offsets.cpu(), int(r.offsets[-1])
    want, tol = grouped64(x, up, grid, 1 / math.sqrt(H), off, r.rows.cpu(), None, True, "silu", F16, N)
    assert_within(h[:live], want[:live], tol[:live])
    want, tol = grouped64(h.cpu(), down, grid, 1 / math.sqrt(N), off, None, None, False, "none", F16, H)
    assert_within(o[:live], want[:live], tol[:live])
    assert_within(y, *combine64(o.cpu(), r.slots.cpu(), r.weights.cpu(), x, F16))
    if T > 3:
        assert torch.equal(y[-3:].cpu(), x[-3:])          # padded tokens: the residual alone


@pytest.mark.parametrize("T", [1, 24, 200])
def test_captured_layer_follows_its_inputs(T):
    """The layer in one graph: replays with other tokens and other choices give what eager calls give, bit for bit."""
    E, k, H, N = 8, 2, 512, 768
    gen = torch.Generator().manual_seed(T)
    up, grid = weights(gen, E, 2 * N, H // 8)
    down, _ = weights(gen, E, H, N // 8)
    wq, _ = weights(gen, 2 * H, H // 8)
    ud, dd, gd, wd = dev(up, down, grid, wq)
    x, logits = torch.empty(T, H, dtype=F16, device=DEV), torch.empty(T, E, device=DEV)

    def layer():
        y = moe_layer(x, logits, k, ud, dd, gd, N, H)[3]
        return dmm.decode_matmul_fused(y, wd, gd, 0.04, activation="gelu", gated=True, residual=y)

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(T, H, generator=g))
        logits.copy_(torch.randn(T, E, generator=g))

    capi.check("dmm_init", capi.lib().dmm_init(-1))
    fill(0)
    layer()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = layer()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2, 3, 4):
        fill(seed)
        want = layer()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), seed


def test_calls_on_another_stream_and_twice_at_once():
    x, codes, grid, b, r = fused_inputs(40, 528, 2048, True, F16, F16, seed=3)
    args = dev(x, codes, grid)
    bd, rd = dev(b, r)
    want = dmm.decode_matmul_fused(*args, 0.02, bias=bd, activation="silu", gated=True, residual=rd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(dmm.decode_matmul_fused(*args, 0.02, bias=bd, activation="silu", gated=True, residual=rd))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_routing_results_stand_alone():
    """The five results share one allocation and nothing else: each is contiguous, may be written, and outlives the others."""
    logits = torch.randn(70, 12, device=DEV)
    r = dmm.route_experts(logits, 3)
    kept = [t.clone() for t in r]
    for t in r:
        assert t.is_contiguous() and not t.requires_grad and t.data_ptr() % 16 == 0
    r.weights.zero_()
    r.rows.fill_(-5)
    assert torch.equal(r.experts, kept[1]) and torch.equal(r.offsets, kept[2]) and torch.equal(r.slots, kept[4])
    slots = r.slots
    del r
    torch.empty(1 << 20, device=DEV).fill_(3)
    assert torch.equal(slots, kept[4])


def test_mixed_devices_are_refused():
    x, codes, grid, b, _ = fused_inputs(2, 8, 64, False, F16, None, seed=1)
    with pytest.raises(RuntimeError, match="must be on"):
        dmm.decode_matmul_fused(x.to(DEV), codes, grid.to(DEV), 1.0)
    with pytest.raises(RuntimeError, match="must be on"):
        dmm.decode_matmul_fused(*dev(x, codes, grid), 1.0, bias=b)
    with pytest.raises(RuntimeError, match="same device"):
        dmm.combine_experts(torch.zeros(2, 8, dtype=F16, device=DEV), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, device=DEV))


# ----------------------------------------------------------------- past 32 bits
def test_grouped_codes_past_4_gib(kernel):
    E, N, K = 2100, 1024, 8192                                     # 2 MiB of codes per expert
    who, counts = [0, 1049, E - 1], (5, 40, 25)
    x, some, grid, ends, rows, b = grouped_inputs(counts, 9, N, K, False, F32, True, seed=4, coarse=kernel == 4)
    codes = torch.zeros(E, N, K // 8, dtype=torch.int16, device=DEV)
    bias = torch.zeros(E, N, dtype=F32, device=DEV)
    sizes = torch.zeros(E, dtype=torch.int64)
    for i, e in enumerate(who):
        codes[e], bias[e], sizes[e] = some[i].to(DEV), b[i].to(DEV), counts[i]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).int()
    y = dmm.decode_matmul_grouped(x.to(DEV), codes, grid.to(DEV), 0.01, offsets.to(DEV), rows=rows.to(DEV), bias=bias)
    assert_within(y, *grouped64(x, some, grid, 0.01, ends, rows, b, False, "none", F16, N))


@pytest.mark.parametrize("kernel", [-1, 0, 1, 5])
def test_results_past_4_gib(kernel):
    M, N, K = 70000, 32768, 64
    x, codes, grid, _, _ = fused_inputs(M, N, K, False, None, None, 6)
    lib = capi.lib()
    lib.dmm_set_ops_kernel(kernel)
    try:
        y = dmm.decode_matmul_fused(*dev(x, codes, grid), 0.1, activation="relu")
        torch.cuda.synchronize()
    finally:
        lib.dmm_set_ops_kernel(-1)
    pick = torch.tensor([0, 1, 35000, 65535, 65536, 69997, 69999])
    want, tol = product64(x[pick].double(), decode64(codes, grid), (0.1, 0.1), None, False, "relu", None, F16)
    assert_within(y[pick.to(DEV)], want, tol)
    slots = torch.tensor([[M - 1, 65536], [0, M - 2], [M, 35000]], dtype=torch.int32)
    w = torch.tensor([[0.5, 0.25], [1.5, -1.0], [3.0, 2.0]])
    got = dmm.combine_experts(y, slots.to(DEV), w.to(DEV))
    near = torch.tensor([[0, 1], [2, 3], [9, 4]], dtype=torch.int32)            # the same rows in a small y
    few = y[torch.tensor([M - 1, 65536, 0, M - 2, 35000]).to(DEV)].cpu()
    assert_within(got, *combine64(few, near, w, None, F16))
