"""Inputs on which every part of the arithmetic on 8-bit operands shows: the four terms of x and both halves of the means.

On 8-bit operands a sum is made of x = t0 + t1 / 8 + t2 / 64 + t3 / 512 (t0: the top byte of the half, the next terms the same of
what is left, times 8) against fp8 weights +-g, and of the means of eight x, as two halves hi + lo, against the codes' shift.
On random inputs the last term and the low half stay below the rounding of a half output.  Here they do not:

* every g is 1/4, so a code is +-1/2 in all eight places ("active", three quarters of them) or 0 ("idle");
* x has the sign of its weight, so nothing cancels.  At active codes it has all eleven bits, with each term's leading bit
  set, and a mean whose low half has the same sign; at idle codes it is +-1.5, which has one term and no low half:
  terms or means that meet a neighbour's code are missed as well;
* two rows of x hold the same pieces at other active codes, so their sums are equal, and a float32 bias takes that sum
  away: what is left is the error, which the output's rounding does not hide."""
import numpy as np
import torch

EPS32 = 2.0 ** -24


def terms(x):
    """The four terms (as the values they add up from) of float16 x, exact."""
    out, rem = [], x.astype(np.float16)
    for t in range(4):
        top = (rem.view(np.uint16) & 0xFF00).view(np.float16)
        out.append(top.astype(np.float64) / 8.0 ** t)
        rem = ((rem - top) * np.float16(8)).astype(np.float16)
    return out


def means(x):
    """hi, lo of the means of eight: halves, lo of what hi leaves (times 8, exact)."""
    m = x.astype(np.float32).reshape(*x.shape[:-1], -1, 8).sum(-1, dtype=np.float32) / np.float32(8)
    hi = m.astype(np.float16)
    lo = ((m - hi.astype(np.float32)) * np.float32(8)).astype(np.float16)
    return hi.astype(np.float64), lo.astype(np.float64) / 8


def _pieces(rng, n):
    """n pieces of eight values in [1.5, 2) with all eleven bits, whose mean is at least 3 * 2^-13 above its high half."""
    got = []
    while sum(map(len, got)) < n:
        a, b, c, d = rng.integers(2, 4, (4096, 8)), rng.integers(4, 8, (4096, 8)), rng.integers(4, 8, (4096, 8)), rng.integers(1, 4, (4096, 8))
        m = (1 + a / 4 + b / 32 + c / 256 + d / 1024).astype(np.float16)
        got.append(m[means(m)[1][:, 0] >= 3 * 2.0 ** -13])
    return np.concatenate(got)[:n]


class Case:
    """x [M, K], codes [n, K/8], grid, and of every row of W the sum (float64) and size of its products.

    first, count: the codes at which x is not zero (a window of the K/8).  n rows of W, half of them (at random) negated."""

    def __init__(self, M, n, K, seed, first=0, count=None):
        rng = np.random.default_rng(seed)
        kc = K // 8
        count = kc - first if count is None else count
        sign = rng.choice([-1, 1], kc)
        active = rng.random(kc) < 0.75
        index = rng.integers(0, 256, kc)
        where = np.zeros(kc, bool)
        where[first:first + count] = True
        hot, idle = np.flatnonzero(where & active), np.flatnonzero(where & ~active)
        pieces = _pieces(rng, len(hot))
        x = np.zeros((M, kc, 8), np.float16)
        for m in range(M):
            x[m, hot] = rng.permutation(pieces) * sign[hot, None]
            x[m, idle] = np.float16(1.5) * sign[idle, None]
        self.x = torch.from_numpy(x.reshape(M, K))

        def word(s):        # sign row 0: all plus, 127: all minus; shift of the sign's sign (active) or against it (idle)
            w = index | np.where(s < 0, 127 << 8, 0) | np.where((s < 0) == active, 1 << 15, 0)
            return w.astype(np.uint16).view(np.int16)

        self.flip = rng.random(n) < 0.5
        self.codes = torch.from_numpy(np.where(self.flip[:, None], word(-sign)[None], word(sign)[None]))
        self.grid = torch.full((256, 8), 0.25, dtype=torch.float16)
        self.sign, self.shift = sign, np.where(active, sign, -sign) * 0.25
        self.K, self.used = K, 8 * count
        one = self._sums(self.x.numpy()[:1])[0]                       # equal for every row of x
        self.sum = torch.from_numpy(np.where(self.flip, -one, one))
        # the products with +-g and with the shift are added apart: |x| (|g| + 1/4)
        self.size = float(np.abs(x[0].astype(np.float64)).sum() * 0.5)

    def _sums(self, x, drop=None):
        t, (hi, lo) = terms(x), means(x)
        xs = sum(v for i, v in enumerate(t) if "t%d" % i != drop)
        mean = (0 if drop == "hi" else hi) + (0 if drop == "lo" else lo)
        w = np.repeat(self.sign * 0.25, 8)
        return xs @ w + mean @ (8 * self.shift)

    def emulate(self, drop=None):
        """[M, n] the sums as 8-bit operands form them, in float64; drop: a part that is left out ("t0" .. "t3", "hi", "lo")."""
        s = self._sums(self.x.numpy(), drop)
        return torch.from_numpy(np.where(self.flip[None], -s[:, None], s[:, None]))

    def tol(self):
        """What a right sum may be off by.  Every product is exact.  The matrix unit adds 128 products (or 32 of the means)
        and the accumulator at a time, each cut at worst at one step, 2 EPS32, of the largest of them, which is no
        larger than the size of the whole sum: (128 + 1 + (32 + 1) / 2) / 128 < 1.15 steps per k; the term columns have sizes of
        1 + 1/8 + 1/64 + 1/512 < 1.15 of the first one's.  The join of sixteen waves, scale and bias: eight more.  hi + lo
        has 22 bits.  Where x is zero nothing is added."""
        return (2 * EPS32 * (1.15 * 1.15 * self.used + 8) + 2.0 ** -22) * self.size


def cancelling(case, keep=0.0):
    """float32 bias that leaves about `keep` of every sum, and what is left exactly."""
    b = (keep - case.sum).float()
    return b, case.sum + b.double()


def grouped8(x, codes, grid, scale, offsets, rows, gated, act, out, N):
    """grouped64 without bias, with the bound of sums on 8-bit operands (Case.tol; |g| + 1/4 is at most |w| + 1/2)."""
    from ops_util import HALF_STEP, TINY, act64, decode64
    R, K = rows.shape[0], x.shape[1]
    y, tol = torch.full((R, N), float("nan"), dtype=torch.float64), torch.zeros(R, N, dtype=torch.float64)
    for e in range(codes.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if lo >= hi:
            continue
        w, xe = decode64(codes[e], grid), x[rows[lo:hi].long()].double()
        z = xe @ w.t() * scale
        err = (2 * EPS32 * (1.15 * 1.15 * K + 8) + 2.0 ** -22) * (xe.abs() @ (w.abs() + 0.5).t()) * scale
        a, ea = act64(z[:, :N], act), 1.13 * err[:, :N] + 8 * EPS32 * z[:, :N].abs()       # as product64
        if gated:
            u, eu = z[:, N:], err[:, N:]
            a, ea = a * u, ea * (u.abs() + eu) + a.abs() * eu + EPS32 * (a * u).abs()
        y[lo:hi], tol[lo:hi] = a, 2 * ea + HALF_STEP[out] * (a.abs() + 2 * ea) + TINY[out]
    return y, tol
