"""The operators around the product in 64 bits, with the error a right kernel may have, and inputs for their tests."""
import math

import numpy as np
import torch

from oracle import dmm_oracle as orc

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
EPS32 = 2.0 ** -24     # half a step of float32, relative to the value
HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -134}   # half a step of the subnormals


def act64(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def decode64(codes, grid):
    """float64 [.., N, K] of codes [.., N, K/8]."""
    if codes.numel() == 0:
        return torch.zeros(*codes.shape[:-1], codes.shape[-1] * 8, dtype=torch.float64)
    flat = codes.reshape(-1, codes.shape[-1]).cpu().numpy().view(np.uint16)
    w = torch.from_numpy(orc.decode_f16(flat, grid.cpu().numpy()).astype(np.float64))
    return w.view(*codes.shape[:-1], codes.shape[-1] * 8)


def product64(x, w, scale, bias, gated, act, residual, out):
    """(y, tol) in float64: x [M,K] and w [N,K] float64, scale a pair of floats.

    tol.  A sum of K products in fp32, in any order, is off by at most (K + 2) EPS32 times the sum of the
    products' sizes (the products of halves are exact; + 2 for scale and bias).  An activation passes an error on
    with a slope of at most 1.13, and is off by itself: by 8 EPS32 of its argument's size (a handful of roundings; the
    result is the argument times a factor of at most 1).  A gate multiplies the errors by the other factor.  Then the residual's
    addition, and half a step of the output's type.  Twice the total, for the second-order terms."""
    K = x.shape[1]
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    n = w.shape[0] // 2 if gated else w.shape[0]
    sc = torch.full((w.shape[0],), float(scale[0]), dtype=torch.float64)
    if gated:
        sc[n:] = float(scale[1])
    z, size = z * sc, size * sc.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    err = (K + 2) * EPS32 * size
    if gated:
        a = act64(z[:, :n], act)
        ea = 1.13 * err[:, :n] + 8 * EPS32 * z[:, :n].abs()
        y = a * z[:, n:]
        ey = ea * z[:, n:].abs() + a.abs() * err[:, n:] + ea * err[:, n:] + EPS32 * y.abs()
    else:
        y = act64(z, act)
        ey = 1.13 * err + (8 * EPS32 * z.abs() if act != "none" else 0)
    if residual is not None:
        y = y + residual.double()
        ey = ey + EPS32 * y.abs()
    return y, 2 * ey + HALF_STEP[out] * (y.abs() + 2 * ey) + TINY[out]


def assert_within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    same_nan = torch.isnan(got) == torch.isnan(want)
    assert same_nan.all(), "%s: NaN in the wrong places" % what
    err = (got - want).abs()
    bad = ~((err <= tol) | torch.isnan(want) | (got == want))
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%s: %d of %d outside, first at %s: got %r want %r tol %r" %
                             (what, int(bad.sum()), bad.numel(), i, got[tuple(i)].item(), want[tuple(i)].item(), tol[tuple(i)].item()))


GRID_VALUES = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.25, 2.75])


def weights(gen, *shape, fp8=True):
    """Codes of the given shape and a grid; fp8=False: grid values that do not fit 8 bits."""
    codes = torch.randint(-32768, 32768, shape, generator=gen, dtype=torch.int32).to(torch.int16)
    if fp8:
        grid = GRID_VALUES[torch.randint(0, 6, (256, 8), generator=gen)].half()
    else:
        grid = (torch.rand(256, 8, generator=gen) * 3).half()
    return codes, grid


def rows_of_x(gen, rows, K, coarse):
    """Normal values, or (coarse) values of two significant bits: one 8-bit term each, every product and every sum of
    them exact on 8-bit operands too, so that the error bound of exact products holds there."""
    if not coarse:
        return torch.randn(rows, K, generator=gen).half()
    pick = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, -0.5, -1.0, -1.5, -2.0, -3.0])
    return pick[torch.randint(0, len(pick), (rows, K), generator=gen)].half()


def fused_inputs(M, N, K, gated, bias, residual, seed, fp8=True, coarse=False):
    gen = torch.Generator().manual_seed(seed)
    n2 = 2 * N if gated else N
    codes, grid = weights(gen, n2, K // 8, fp8=fp8)
    x = rows_of_x(gen, M, K, coarse)
    b = torch.randn(n2, generator=gen).to(bias) if bias else None
    r = torch.randn(M, N, generator=gen).to(residual) if residual else None
    return x, codes, grid, b, r


def grouped_inputs(counts, T, N, K, gated, bias, gather, seed, behind=0, coarse=False):
    """Rows of every expert from counts, `behind` rows that belong to none."""
    gen = torch.Generator().manual_seed(seed)
    E, n2 = len(counts), 2 * N if gated else N
    codes, grid = weights(gen, E, n2, K // 8)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    R = int(offsets[-1]) + behind
    rows = torch.randint(0, T, (R,), generator=gen, dtype=torch.int32) if gather else None
    x = rows_of_x(gen, T if gather else R, K, coarse)
    b = torch.randn(E, n2, generator=gen).to(bias) if bias else None
    return x, codes, grid, offsets, rows, b


def grouped64(x, codes, grid, scale, offsets, rows, bias, gated, act, out, N):
    """(y, tol) over all R rows; rows that belong to no expert are NaN.  scale: float, [E] or [E, 2]."""
    R = x.shape[0] if rows is None else rows.shape[0]
    w = decode64(codes, grid)
    y = torch.full((R, N), math.nan, dtype=torch.float64)
    tol = torch.zeros(R, N, dtype=torch.float64)
    for e in range(codes.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if lo >= hi:
            continue
        p = torch.arange(lo, hi)
        t = p if rows is None else rows[lo:hi].long()
        ok = (t >= 0) & (t < x.shape[0])
        xe = torch.where(ok.unsqueeze(1), x.double()[t.clamp(0, x.shape[0] - 1)], torch.zeros((), dtype=torch.float64))
        s = (scale, scale) if not isinstance(scale, torch.Tensor) else (scale.view(len(scale), -1)[e, 0].item(), scale.view(len(scale), -1)[e, -1].item())
        y[lo:hi], tol[lo:hi] = product64(xe, w[e], s, None if bias is None else bias[e], gated, act, None, out)
    return y, tol


def route64(logits, k, scoring, normalize):
    """Weights in float64 and the lists, token by token."""
    z = logits.double()
    T, E = z.shape
    weights = torch.zeros(T, k, dtype=torch.float64)
    experts = torch.full((T, k), -1, dtype=torch.int32)
    for t in range(T):
        v = z[t].tolist()
        order = sorted((e for e in range(E) if v[e] > -math.inf), key=lambda e: (-v[e], e))[:k]
        if not order:
            continue
        p = [1 / (1 + math.exp(-v[e])) if v[e] > 0 else math.exp(v[e]) / (1 + math.exp(v[e])) for e in order] if scoring == "sigmoid" else [math.exp(v[e] - v[order[0]]) for e in order]
        total = sum(p) if normalize else 1.0 if scoring == "sigmoid" else sum(math.exp(u - v[order[0]]) for u in v)
        for j, e in enumerate(order):
            experts[t, j] = e
            weights[t, j] = p[j] / total
    flat = [(int(e), i) for i, e in enumerate(experts.flatten().tolist()) if e >= 0]
    flat.sort()
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    for e, _ in flat:
        offsets[e + 1] += 1
    offsets = offsets.cumsum(0).to(torch.int32)
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    slots = torch.full((T * k,), -1, dtype=torch.int32)
    for s, (_, i) in enumerate(flat):
        rows[s] = i // k
        slots[i] = s
    return weights, experts, offsets, rows, slots.view(T, k)


def check_routing(r, logits, k, scoring, normalize):
    w, experts, offsets, rows, slots = route64(logits.cpu(), k, scoring, normalize)
    for name, got, want in (("experts", r.experts, experts), ("offsets", r.offsets, offsets), ("rows", r.rows, rows), ("slots", r.slots, slots)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), name
    # an exponential is off by a few steps and by the rounding of its argument (up to 2 |v|), the sum of up to E of
    # them by E steps at most, the division by one
    size = logits.float().nan_to_num(0, 0, 0).abs().max().item() if logits.numel() else 0.0
    assert_within(r.weights, w, (logits.shape[1] + 8 + 4 * size) * EPS32 * w + 2.0 ** -126, "weights")


def combine64(y, slots, weights, residual, out):
    R = y.shape[0]
    s = slots.long()
    live = ((s >= 0) & (s < R)).unsqueeze(-1)
    rows = torch.where(live, y.double()[s.clamp(0, max(R - 1, 0))] if R else torch.zeros(*s.shape, y.shape[1], dtype=torch.float64),
                       torch.zeros((), dtype=torch.float64))
    terms = torch.where(live, weights.double().unsqueeze(-1) * rows, torch.zeros((), dtype=torch.float64))
    z, size = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        z, size = z + residual.double(), size + residual.double().abs()
    err = (slots.shape[1] + 1) * EPS32 * size
    return z, err + HALF_STEP[out] * (z.abs() + err) + TINY[out]
