"""The operators around the product as a user gets them: the library's own choice, 8-bit operands in their default position."""
import math

import pytest
import torch

import decode_matmul_amd as dmm
from decode_matmul_amd import capi
from gpu_util import DEV
from ops_terms import Case, cancelling, grouped8
from ops_util import assert_within, check_routing, combine64, decode64, fused_inputs, grouped64, grouped_inputs, product64, weights

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


# ----------------------------------------------------------------- every term of x and both halves of the means
def check_cancelled(y, left, tol):
    """y = what a bias leaves of the sums: left up to tol, in fp32 (two roundings of the sum and the bias are in tol), rounded to half."""
    bound = tol + 2.0 ** -11 * (left.abs() + tol) + 2.0 ** -25
    err = (y.detach().cpu().double() - left).abs()
    assert torch.all(err <= bound), "%d of %d outside, worst %.3g of the bound" % (int((err > bound).sum()), err.numel(), float((err / bound).max()))


def check_terms(M, N, K, gated, first=0, count=None):
    if not gated:
        c = Case(M, N, K, M + N + K + first, first, count)
        b, left = cancelling(c)
        y = dmm.decode_matmul_fused(*dev(c.x, c.codes, c.grid), 1.0, bias=b.to(DEV))
        assert y.dtype == F16
        check_cancelled(y, left.expand(M, N), c.tol())
        return
    c = Case(M, 2 * N, K, M + N + K + first, first, count)
    for who in (0, 1):      # one factor's sums cancel, the other factor is 64
        keep = torch.full((2 * N,), 64.0, dtype=torch.float64)
        keep[who * N:(who + 1) * N] = 0
        b, left = cancelling(c, keep)
        y = dmm.decode_matmul_fused(*dev(c.x, c.codes, c.grid), 1.0, bias=b.to(DEV), gated=True)
        gate, up = left[:N], left[N:]
        t = c.tol()
        check_cancelled(y, (gate * up).expand(M, N), (t * (gate.abs() + up.abs() + t) + 2.0 ** -24 * (gate * up).abs()).expand(M, N))


# tiles per compute unit (256 of them): gemv_q8d's body with 2, 4, 6 and 8 tiles, plain and in pairs, tails of all kinds
@pytest.mark.parametrize("N,gated", [(4095, False), (8192, False), (12288, False), (16383, False), (16386, False), (24575, False),
                                     (24580, False), (32766, False), (2049, True), (4096, True), (8189, True), (11008, True),
                                     (12285, True), (16382, True)])
@pytest.mark.parametrize("K,first,count", [(256, 0, None), (2048, 0, None), (8192, 0, 32), (8192, 500, 32), (8192, 992, 32)])
def test_one_row_sees_every_term(N, K, first, count, gated):
    check_terms(1, N, K, gated, first, count)


# the jobs' kernel: one job and many, one row and two, K that is not whole steps
@pytest.mark.parametrize("M,N,gated", [(1, 40004, False), (1, 20001, True), (2, 14000, False), (2, 33001, False), (2, 8197, True), (2, 20001, True)])
@pytest.mark.parametrize("K,first,count", [(2304, 0, 32), (4352, 400, 32), (4352, 512, 32), (2064, 256, 2), (2064, 240, 18), (8192, 992, 32)])
def test_one_and_two_rows_in_jobs_see_every_term(M, N, gated, K, first, count):
    check_terms(M, N, K, gated, first, count)


# forced where the choice would not take it: short K, few tiles, many segments
@pytest.mark.parametrize("M,N,gated", [(1, 17, False), (2, 16, True), (1, 5000, False), (2, 9001, True)])
@pytest.mark.parametrize("K", [16, 64, 240, 256])
def test_short_k_in_jobs_sees_every_term(M, N, gated, K):
    capi.lib().dmm_set_ops_kernel(4)
    check_terms(M, N, K, gated)


def grouped_terms(counts, N, K, seed, first=0, count=None):
    """Every expert its own case; up to two rows each, as tokens in an order of their own; the biases cancel all sums."""
    cases = [Case(max(n, 1), N, K, seed + e, first, count) for e, n in enumerate(counts)]
    T = sum(counts)
    order = torch.randperm(T, generator=torch.Generator().manual_seed(seed))
    x = torch.zeros(T, K, dtype=F16)
    x[order] = torch.cat([c.x[:n] for c, n in zip(cases, counts) if n > 0])
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    b, left = zip(*(cancelling(c) for c in cases))
    want = torch.cat([v.expand(n, -1) for v, n in zip(left, counts)])
    tol = torch.cat([torch.full((n, N), c.tol(), dtype=torch.float64) for c, n in zip(cases, counts)])
    return x, torch.stack([c.codes for c in cases]), cases[0].grid, offsets, order.int(), torch.stack(b), want, tol


# by expert, by the library's own rule: up to two rows in all, and a quarter as many rows as experts, on 20 MB of codes and more
@pytest.mark.parametrize("counts,N,K,first,count", [((0, 1, 0, 1), 10300, 4096, 0, 32), ((0, 0, 2), 22000, 4096, 300, 32),
                                                    ((0, 1), 21001, 4352, 512, 32), ((0, 2, 0, 0, 0, 0, 1, 0) + (0,) * 5 + (1, 0, 0), 5500, 4096, 480, 32)])
def test_grouped_sees_every_term(counts, N, K, first, count):
    x, codes, grid, offsets, rows, b, want, tol = grouped_terms(counts, N, K, 7, first, count)
    args = dev(x, codes, grid)
    kw = dict(rows=rows.to(DEV), bias=b.to(DEV))
    y = dmm.decode_matmul_grouped(*args, 1.0, offsets.to(DEV), **kw)
    check_cancelled(y, want, tol)


@pytest.mark.parametrize("counts,N,K", [((1, 2, 0, 2, 1, 1), 9001, 256), ((2,) * 70, 200, 256), ((0,) * 66 + (2, 0, 1), 777, 256), ((1, 2), 40, 112)])
def test_grouped_many_jobs_see_every_term(counts, N, K):
    capi.lib().dmm_set_ops_kernel(4)
    x, codes, grid, offsets, rows, b, want, tol = grouped_terms(counts, N, K, 11)
    y = dmm.decode_matmul_grouped(*dev(x, codes, grid), 1.0, offsets.to(DEV), rows=rows.to(DEV), bias=b.to(DEV))
    check_cancelled(y, want, tol)


@pytest.mark.parametrize("N,gated", [(4095, False), (8192, False), (16383, False), (24575, False), (32766, False), (2049, True), (8189, True),
                                     (11008, True), (16382, True)])
@pytest.mark.parametrize("what", ["grid", "infinity", "nan"])
def test_one_row_that_8_bit_operands_cannot_do(N, gated, what):
    """The batch-1 body hands the launch over to 16 bits: the sums of exact products, and an infinity only where it belongs."""
    K = 512
    x, codes, grid, b, r = fused_inputs(1, N, K, gated, F16, F16, N, fp8=what != "grid")
    if what != "grid":
        x[0, 300] = math.inf if what == "infinity" else math.nan
    y = dmm.decode_matmul_fused(*dev(x, codes, grid), 0.05, bias=b.to(DEV), gated=gated, residual=r.to(DEV))
    want, tol = product64(x.double(), decode64(codes, grid), (0.05, 0.05), b, gated, "none", r, F16)
    if what == "grid":
        assert_within(y, want, tol)
        return
    got = y.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    live = ~torch.isnan(want)
    assert torch.equal(got[live], want[live])        # infinities of the right sign


# ----------------------------------------------------------------- together, as a layer uses them
def layer_weights(E, H, N, seed):
    gen = torch.Generator().manual_seed(seed)
    up, grid = weights(gen, E, 2 * N, H // 8)
    down, _ = weights(gen, E, H, N // 8)
    dense, _ = weights(gen, 2 * N, H // 8)
    back, _ = weights(gen, H, N // 8)
    return up, down, dense, back, grid


def layer(x, logits, up, down, dense, back, grid, H, N, k=2):
    """Routed experts and a shared dense MLP whose result is the residual of their sum."""
    h = dmm.decode_matmul_fused(x, dense, grid, 1 / math.sqrt(H), gated=True, activation="silu")
    shared = dmm.decode_matmul_fused(h, back, grid, 1 / math.sqrt(N), residual=x)
    r = dmm.route_experts(logits, k)
    g = dmm.decode_matmul_grouped(x, up, grid, 1 / math.sqrt(H), r.offsets, rows=r.rows, activation="silu", gated=True)
    o = dmm.decode_matmul_grouped(g, down, grid, 1 / math.sqrt(N), r.offsets)
    return r, h, shared, g, o, dmm.combine_experts(o, r.slots, r.weights, residual=shared)


@pytest.mark.parametrize("T", [1, 2, 5])
def test_a_decode_step_through_a_layer(T):
    """4096 -> 2 x 5376, two of four experts and a shared MLP: one token takes every kernel on 8-bit operands."""
    H, N, E, k = 4096, 5376, 4, 2
    up, down, dense, back, grid = layer_weights(E, H, N, T)
    gen = torch.Generator().manual_seed(T + 100)
    x, logits = torch.randn(T, H, generator=gen).half(), torch.randn(T, E, generator=gen)
    r, h, shared, g, o, y = layer(*dev(x, logits, up, down, dense, back, grid), H, N)
    check_routing(r, logits, k, "softmax", True)
    all_rows, one = torch.arange(T, dtype=torch.int32), torch.tensor([0, T])
    assert_within(h, *grouped8(x, dense[None], grid, 1 / math.sqrt(H), one, all_rows, True, "silu", F16, N))
    want, tol = grouped8(h.cpu(), back[None], grid, 1 / math.sqrt(N), one, all_rows, False, "none", F16, H)
    want = want + x.double()
    assert_within(shared, want, tol + 2.0 ** -11 * want.abs())
    assert_within(g, *grouped8(x, up, grid, 1 / math.sqrt(H), r.offsets.cpu(), r.rows.cpu(), True, "silu", F16, N))
    assert_within(o, *grouped8(g.cpu(), down, grid, 1 / math.sqrt(N), r.offsets.cpu(), torch.arange(T * k, dtype=torch.int32), False, "none", F16, H))
    assert_within(y, *combine64(o.cpu(), r.slots.cpu(), r.weights.cpu(), shared.cpu(), F16))


@pytest.mark.parametrize("T", [1, 2, 24])
def test_captured_decode_step_follows_its_inputs(T):
    """Replays with other tokens, other choices, an infinity, and a grid that does not fit 8 bits give what eager calls give."""
    H, N, E = 4096, 5376, 4
    up, down, dense, back, grid = dev(*layer_weights(E, H, N, 3))
    other = weights(torch.Generator().manual_seed(5), 1, 1, fp8=False)[1].to(DEV)
    x, logits, g = torch.empty(T, H, dtype=F16, device=DEV), torch.empty(T, E, device=DEV), torch.empty_like(grid)

    def fill(seed):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(T, H, generator=gen))
        if seed == 3:
            x[T - 1, 77] = math.inf
        logits.copy_(torch.randn(T, E, generator=gen))
        g.copy_(other if seed == 4 else grid)

    def step():
        return layer(x, logits, up, down, dense, back, g, H, N)[-1]

    capi.check("dmm_init", capi.lib().dmm_init(-1))
    fill(0)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2, 3, 4, 5):
        fill(seed)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int16), want.view(torch.int16)), seed
        assert torch.isfinite(want).all() == (seed != 3)


@pytest.mark.parametrize("M,N,K,gated", [(1, 5376, 4096, True), (2, 22000, 4096, False), (1, 40000, 4096, False)])
def test_two_streams_at_once(M, N, K, gated):
    x, codes, grid, b, r = dev(*fused_inputs(M, N, K, gated, F16, F16, seed=3))

    def call():
        return dmm.decode_matmul_fused(x, codes, grid, 0.02, bias=b, activation="silu", gated=gated, residual=r)

    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ----------------------------------------------------------------- long K
# the batch-1 body past the longest x of the plain product's batch-1 kernels, the jobs' kernel, and the last K of both
@pytest.mark.parametrize("M,N,gated", [(1, 8190, False), (1, 4100, True), (2, 12300, False)])
@pytest.mark.parametrize("K,first", [(40960, 5088), (65536, 0), (65536, 4000), (65536, 8160)])
def test_long_k_sees_every_term(M, N, gated, K, first):
    check_terms(M, N, K, gated, first, 32)


@pytest.mark.parametrize("kernel", [-1, 1, 2, 3, 4, 5], ids=["auto", "rows", "gemm", "split", "rows8", "mid"])
@pytest.mark.parametrize("K", [1 << 23, (1 << 23) + 64, (1 << 23) + 16])
@pytest.mark.parametrize("M", [1, 2, 3, 17])
def test_k_at_and_past_the_longest_of_the_row_kernels(M, K, kernel):
    """x is zero but for 256 k near the end of K; both sides of the limit."""
    capi.lib().dmm_set_ops_kernel(kernel)
    first = K // 8 - 40
    c = Case(M, 20, K, 5, first, 32)
    b, left = cancelling(c)
    y = dmm.decode_matmul_fused(*dev(c.x, c.codes, c.grid), 1.0, bias=b.to(DEV))
    check_cancelled(y, left.expand(M, 20), c.tol())


# ----------------------------------------------------------------- x of 2 GiB and more
def test_x_past_2_gib():
    """Rows on both sides of 2^31 bytes, dense and by expert, in their order and (the catch-all) through a list; blocks that begin
    anywhere, a last one that is cut."""
    T, N, K = 139269, 80, 8192                     # row 131072 begins at 2^31
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(T, K, dtype=F16, device=DEV)
    for i in range(0, T, 8192):
        x[i:i + 8192] = torch.randn(min(8192, T - i), K, generator=gen, device=DEV)
    pick = torch.tensor([0, 1, 127, 128, 65535, 65536, 131071, 131072, 131073, 131200, 139264, T - 1])
    xs = x[pick.to(DEV)].cpu().double()
    s = 1 / math.sqrt(K)
    for gated in (False, True):
        _, codes, grid, b, _ = fused_inputs(1, N, K, gated, F32, None, 4)
        r = torch.randn(T, N, generator=gen, device=DEV).half()
        y = dmm.decode_matmul_fused(x, *dev(codes, grid), s, bias=b.to(DEV), activation="silu", gated=gated, residual=r)
        assert_within(y[pick.to(DEV)], *product64(xs, decode64(codes, grid), (s, s), b, gated, "silu", r[pick.to(DEV)].cpu(), F16))
    ends = (0, 100, 131071, 131071, T - 3)         # the last three rows belong to no expert
    _, codes, grid, _, _, b = grouped_inputs((1, 1, 1, 1), 1, N, K, True, F16, False, 5)
    out = torch.full((T, N), 7.0, dtype=F16, device=DEV)
    dmm.decode_matmul_grouped(x, *dev(codes, grid), s, torch.tensor(ends, dtype=torch.int32, device=DEV), bias=b.to(DEV), activation="gelu", gated=True, out=out)
    for p, xp in zip(pick.tolist(), xs):
        if p >= ends[-1]:
            assert torch.all(out[p] == 7.0)
            continue
        e = max(i for i in range(4) if ends[i] <= p < ends[i + 1])
        assert_within(out[p:p + 1], *product64(xp[None], decode64(codes[e], grid), (s, s), b[e], True, "gelu", None, F16), "row %d" % p)
    rows = pick.int().flip(0).contiguous()
    y = dmm.decode_matmul_grouped(x, *dev(codes, grid), s, torch.tensor([0, 5, 5, 12, 12], dtype=torch.int32, device=DEV), rows=rows.to(DEV),
                                  bias=b.to(DEV), gated=True)
    for lo, hi, e in ((0, 5, 0), (5, 12, 2)):
        assert_within(y[lo:hi], *product64(xs.flip(0)[lo:hi], decode64(codes[e], grid), (s, s), b[e], True, "none", None, F16))


# ----------------------------------------------------------------- corners of the ranges
@pytest.fixture(params=[-1, 0, 1, 2, 3, 4, 5], ids=["auto", "generic", "rows", "gemm", "split", "rows8", "mid"])
def kernel(request):
    capi.lib().dmm_set_ops_kernel(request.param)
    return request.param


@pytest.mark.parametrize("K", [16, 32, 48, 80, 112, 144])
@pytest.mark.parametrize("N,gated", [(1, False), (2, True), (3, False), (15, True), (18, False)])
def test_short_k_and_few_columns(N, K, gated, kernel):
    for M in (1, 2, 3, 9, 33, 70, 140):
        x, codes, grid, b, r = fused_inputs(M, N, K, gated, F32, F16, M + N + K, coarse=True)
        y = dmm.decode_matmul_fused(*dev(x, codes, grid), 0.1, bias=b.to(DEV), activation="gelu", gated=gated, residual=r.to(DEV))
        assert_within(y, *product64(x.double(), decode64(codes, grid), (0.1, 0.1), b, gated, "gelu", r, F16), "M=%d" % M)


@pytest.mark.parametrize("gated", [False, True])
def test_thousands_of_experts(gated, kernel):
    """5000 experts, most without a row, of 16 columns and K = 48."""
    E, N, K = 5000, 16, 48
    counts = [0] * E
    for e, n in ((0, 3), (63, 1), (64, 2), (1999, 40), (2047, 1), (3333, 130), (E - 1, 2)):
        counts[e] = n
    x, codes, grid, offsets, rows, b = grouped_inputs(tuple(counts), 9, N, K, gated, F16, True, 3, behind=4, coarse=True)
    out = torch.full((rows.shape[0], N), 5.0, dtype=F16, device=DEV)
    dmm.decode_matmul_grouped(*dev(x, codes, grid), 0.1, offsets.to(DEV), rows=rows.to(DEV), bias=b.to(DEV), gated=gated, out=out)
    want, tol = grouped64(x, codes, grid, 0.1, offsets, rows, b, gated, "none", F16, N)
    assert torch.all(out[-4:] == 5.0)
    assert_within(out[:-4], want[:-4], tol[:-4])


@pytest.mark.parametrize("gated", [False, True])
def test_jobs_behind_the_numbered_ones_are_done_again(gated):
    """Forced onto 8-bit operands, 78 jobs per workgroup: infinities early and late, the rows beside them unharmed."""
    M, N, K = 40000, 16, 256
    x, codes, grid, b, r = fused_inputs(M, N, K, gated, F16, F16, 3, coarse=True)
    bad = [M - 1, M // 2, 140, 3]
    x[bad, 100] = math.inf
    capi.lib().dmm_set_ops_kernel(4)
    y = dmm.decode_matmul_fused(*dev(x, codes, grid), 0.05, bias=b.to(DEV), gated=gated, residual=r.to(DEV)).cpu()
    want, tol = product64(x.double(), decode64(codes, grid), (0.05, 0.05), b, gated, "none", r, F16)
    keep = torch.ones(M, dtype=torch.bool)
    keep[bad] = False
    assert_within(y[keep], want[keep], tol[keep])
    assert torch.equal(torch.isnan(y[bad]), torch.isnan(want[bad])) and not torch.isfinite(y[bad]).any()


@pytest.mark.parametrize("M,N,gated", [(1, 200003, False), (2, 131075, False), (2, 70001, True)])
def test_very_many_columns_see_every_term(M, N, gated):
    check_terms(M, N, 2304, gated, 200, 32)


@pytest.mark.parametrize("where", ["host", "gpu"])
def test_nothing_to_do(where):
    d = "cpu" if where == "host" else DEV
    x, codes, grid, _, _ = (t.to(d) if t is not None else None for t in fused_inputs(2, 8, 64, False, None, None, 1))
    assert dmm.decode_matmul_fused(x[:0], codes, grid, 1.0, residual=torch.empty(0, 8, device=d)).shape == (0, 8)
    assert dmm.decode_matmul_fused(x, codes[:0], grid, 1.0, gated=True, bias=torch.empty(0, device=d)).shape == (2, 0)
    offsets = torch.zeros(1, dtype=torch.int32, device=d)
    assert dmm.decode_matmul_grouped(x, codes[None][:0], grid, 1.0, offsets).shape == (2, 8)
    assert dmm.combine_experts(x[:, :0].contiguous(), torch.zeros(3, 2, dtype=torch.int32, device=d), torch.ones(3, 2, device=d)).shape == (3, 0)
    r = dmm.route_experts(torch.zeros(0, 3, device=d), 3)
    assert r.offsets.tolist() == [0] * 4 and r.rows.shape == (0,)


@pytest.mark.parametrize("where", ["host", "gpu"])
@pytest.mark.parametrize("E,k", [(5, 3), (300, 20)])
def test_route_logit_of_plus_infinity(E, k, where):
    """sigmoid: a weight like any other; softmax: inf - inf, NaN, as torch.softmax has it; chosen first either way."""
    z = torch.randn(3, E, generator=torch.Generator().manual_seed(1))
    z[1, 4] = math.inf
    zd = z if where == "host" else z.to(DEV)
    for normalize in (False, True):
        r = dmm.route_experts(zd, k, scoring="sigmoid", normalize=normalize)
        assert r.experts[1, 0] == 4 and torch.isfinite(r.weights).all()
        top = torch.sigmoid(torch.sort(z.double(), dim=1, descending=True).values[:, :k])
        want = top / top.sum(1, keepdim=True) if normalize else top
        assert_within(r.weights, want, (E + 40) * 2.0 ** -24 * want)
        r = dmm.route_experts(zd, k, normalize=normalize)
        assert r.experts[1, 0] == 4 and torch.isnan(r.weights[1]).all() and torch.isfinite(r.weights[[0, 2]]).all()
