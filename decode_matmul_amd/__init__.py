"""decode_matmul_amd: decode-and-matmul for MI355X (gfx950).

Drop-in for the reference's Python module (`from decode_matmul_cuda import decode_matmul`,
/root/reference/test_decode_matmul.py:5, /root/reference/decode_matmul_cuda/decode_matmul_cuda.cu:237-239)
in the half-precision form of the same code format:

    from decode_matmul_amd import decode_matmul
    y = decode_matmul(x, codes, grid, scale)      # x half [M,K], codes int16/uint16 [N,K/8],
                                                  # grid half [256,8] -> y half [M,N]
    W = decode(codes, grid)                       # dense half [N,K], bit-exact decode

and around the product, for a model's MLP on such weights: `decode_matmul_fused` (bias, activation, gate,
residual in the epilogue), `decode_matmul_grouped` (the same per expert), `route_experts` and `combine_experts`.

The functions are the compiled PyTorch operator (`_C`, host C++) over the C ABI of
`libdmm.so` (hand-written HIP).  GPU tensors run the HIP kernels; `decode_matmul` and `decode` also
take tensors in host memory, which go to the library's own host route (plain C++ loops, the
counterpart of the reference's CPU path, test_decode_matmul.py:29-71).  Nothing falls back: without
the built extension every operator raises ImportError (the import itself succeeds, so that
`python -m decode_matmul_amd.build` can run on a fresh tree).
"""
import collections as _collections
import os as _os

_PKG_DIR = _os.path.dirname(_os.path.abspath(__file__))
LIB_PATH = _os.path.join(_PKG_DIR, "libdmm.so")
EXT_PATH = _os.path.join(_PKG_DIR, "_C.so")

import torch as _torch  # noqa: E402  (loads the HIP runtime the extension links against)

_C = None


def _ext():
    """The compiled operator module; loaded on first use, ImportError if it is not built."""
    global _C
    if _C is None:
        if not (_os.path.exists(LIB_PATH) and _os.path.exists(EXT_PATH)):
            raise ImportError(
                "decode_matmul_amd: native libraries are not built (%s, %s); run "
                "`python -m decode_matmul_amd.build`" % (LIB_PATH, EXT_PATH)
            )
        import importlib
        _C = importlib.import_module("._C", __name__)
    return _C


if _os.path.exists(LIB_PATH) and _os.path.exists(EXT_PATH):
    _ext()

from .capi import lib  # noqa: E402,F401
from .codebook import (  # noqa: E402,F401
    build_codebook_abs,
    grid_from_codebook,
    transpose_tile,
    untranspose_tile,
)

__all__ = [
    "decode_matmul",
    "decode_matmul_path",
    "decode_matmul_int8",
    "pack_codes",
    "decode_matmul_packed",
    "decode",
    "decode_matmul_fused",
    "decode_matmul_grouped",
    "route_experts",
    "combine_experts",
    "Routing",
    "lib",
    "build_codebook_abs",
    "grid_from_codebook",
    "transpose_tile",
    "untranspose_tile",
]


def decode_matmul(x, codes, table, scale=None):
    """The operator under the reference's name, dispatching on the dtype of x.

    Half x: `decode_matmul(x, codes, grid, scale)` -> half y[M,N] = half(scale * x @
    decode(codes, grid).T), fp32 accumulation; codes row-major [N, K/8], grid half [256,8].
    int8 x: the reference's own call `decode_matmul(x, weights_compressed, codebook_abs)`
    (decode_matmul_cuda.cu:178-181, test_decode_matmul.py:136) -> int32 [M,N], exact; codes in the
    reference's tile order (`transpose_tile`), table int64[256]; no scale.

    Runs on x's device and the current stream, asynchronously; raises RuntimeError on bad
    inputs like the reference's TORCH_CHECKs (decode_matmul_cuda.cu:182-207)."""
    if x.dtype == _torch.int8:
        if scale is not None:
            raise TypeError("decode_matmul: the integer form (int8 x) takes no scale")
        return _ext().decode_matmul_int8(x, codes, table, True)
    if scale is None:
        raise TypeError("decode_matmul: the half-precision form needs a scale")
    return _ext().decode_matmul(x, codes, table, float(scale))


def decode_matmul_path(x, codes, grid, scale, path="auto"):
    """decode_matmul through one named kernel path: "auto", "gemv", "gemm" or "generic".
    A path asked for outside its domain raises instead of falling back."""
    return _ext().decode_matmul_path(x, codes, grid, float(scale), path)


def decode_matmul_int8(x, weights_compressed, codebook_abs, tiled=True):
    """The reference's operator with its own dtypes: int8 x [M,K], int16 codes [N,K/8], int64[256]
    table -> int32 [M,N] (decode_matmul_cuda.cu:178-234).  tiled=True: codes as the reference's
    kernel reads them (`transpose_tile`, test_decode_matmul.py:101-109); False: row-major."""
    return _ext().decode_matmul_int8(x, weights_compressed, codebook_abs, bool(tiled))


def pack_codes(codes):
    """Offline repack of codes [N, K/8] (K % 256 == 0) for the batch-1 kernel: each wave's load
    becomes 1 KB of consecutive bytes.  The counterpart of the reference's `transpose_tile`
    (test_decode_matmul.py:101-109).  Returns [ceil(N/16)*16, K/8], same dtype."""
    return _ext().pack_codes(codes)


def decode_matmul_packed(x, packed, grid, scale, N):
    """`decode_matmul` on codes packed by `pack_codes`; N = rows of the original code matrix.
    Any M; bit-identical to `decode_matmul` on the row-major codes."""
    return _ext().decode_matmul_packed(x, packed, grid, float(scale), int(N))


def decode(codes, grid):
    """Dense half matrix W[N,K] from codes[N,K/8]; W[n, 8j+d] is dim d of codes[n, j]."""
    return _ext().decode(codes, grid)


def _number(scale, what):
    """A scale as a number; a tensor of one value is read (which waits for its device)."""
    if isinstance(scale, _torch.Tensor):
        _ext().check_no_grad(scale, what, "scale")
    return float(scale)


def _scale_pair(scale, gated, what):
    """The scales of the two halves of a gated call; the same number twice unless they come as a pair."""
    if not isinstance(scale, (tuple, list)):
        return (_number(scale, what),) * 2
    if not gated:
        raise RuntimeError("%s: a pair of scales is for a gated call" % what)
    if len(scale) != 2:
        raise RuntimeError("%s: a pair of scales is (gate, up), got %d values" % (what, len(scale)))
    return _number(scale[0], what), _number(scale[1], what)


def decode_matmul_fused(x, codes, grid, scale, *, bias=None, activation="none", gated=False, residual=None, out_dtype=None):
    """`decode_matmul` with an epilogue, fp32 until one rounding at the store:

        z = scale * x @ decode(codes, grid).T + bias
        y = act(z) + residual                              gated=False, codes [N, K/8]
        y = act(z[:, :N]) * z[:, N:] + residual            gated=True, codes [2 N, K/8]: gate rows, then up rows

    x half [M, K]; bias (one value per row of codes) and residual [M, N] half or float32; activation "none",
    "relu", "silu", "gelu" (erf) or "gelu_tanh"; out_dtype float16 (default) or float32.  scale: a number, or for a gated
    call a pair (gate, up).  No gradient: an input that requires one, or carries a forward-mode tangent, is refused."""
    scale, scale_up = _scale_pair(scale, gated, "decode_matmul_fused")
    return _ext().decode_matmul_fused(x, codes, grid, scale, scale_up, bias, activation, bool(gated), residual,
                                      out_dtype or _torch.float16)


def decode_matmul_grouped(x, codes, grid, scale, offsets, *, rows=None, bias=None, activation="none", gated=False,
                          out_dtype=None, out=None):
    """`decode_matmul_fused` per expert on rows grouped by expert: row p of the result, offsets[e] <= p < offsets[e + 1],
    is made with codes[e] from x[rows[p]] (rows=None: x[p]).

    codes [E, N, K/8] (gated: [E, 2 N, K/8]), bias [E, ...] one value per row of codes, scale a number, float32 [E], or
    for a gated call a pair (gate, up) or float32 [E, 2]; offsets int32 [E + 1] and rows int32 [R] live on x's device and are not read by the
    host (`route_experts` makes both).  An entry of rows outside x stands for a row of zeros.  Rows from
    offsets[E] on are not written: in `out` (optional, [R, N], no memory shared with an input) they stay as they were, in a
    result allocated here their content is undefined."""
    scales, number = (scale, (1.0, 1.0)) if isinstance(scale, _torch.Tensor) else (None, _scale_pair(scale, gated, "decode_matmul_grouped"))
    return _ext().decode_matmul_grouped(x, codes, grid, *number, scales, offsets, rows, bias, activation, bool(gated),
                                        out_dtype or (out.dtype if out is not None else _torch.float16), out)


Routing = _collections.namedtuple("Routing", "weights experts offsets rows slots")


def route_experts(logits, k, *, scoring="softmax", normalize=True):
    """The k largest logits of every row of logits [T, E] (half, bfloat16 or float32; T up to 2^24, E up to 1024, k up to
    64), equal ones by index, and the lists that `decode_matmul_grouped` and `combine_experts` read.  Returns a `Routing`:

        weights  float32 [T, k]   softmax over the row, or sigmoid, of the chosen; divided by their sum if normalize
        experts  int32 [T, k]     -1: no choice (a logit of -inf or NaN is never chosen; such a weight is 0)
        offsets  int32 [E + 1]    first row of every expert, rows sorted by expert, then by token
        rows     int32 [T * k]    the token of every sorted row; -1 from offsets[E] on
        slots    int32 [T, k]     the sorted row of every choice; -1: no choice

    The five share one allocation, which any of them keeps alive (clone one that is kept or saved by itself)."""
    return Routing(*_ext().route_experts(logits, int(k), scoring, bool(normalize)))


def combine_experts(y, slots, weights, *, residual=None, out_dtype=None):
    """out[t] = residual[t] + sum over j of weights[t, j] * y[slots[t, j]], in fp32 with one rounding; a slot outside y adds
    nothing.  y [R, N] half or float32, slots int32 [T, k], weights float32 [T, k], residual [T, N]."""
    return _ext().combine_experts(y, slots, weights, residual, out_dtype or _torch.float16)
