"""4-bit floating-point matrices (e2m1 codes with block scales): quantisation, read-back, the projection with 4-bit
weights and the gated feed-forward block built from it.

Formats (``FORMATS``); an element is its e2m1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and the negatives) times its block's scale,
times (nvfp4) its row's scale:

* ``"nvfp4"``: blocks of 16 along K with an e4m3 scale, and a power of two per row (the smallest 2^k with the row's
  largest magnitude <= 448 * 6 * 2^k, at least 2^-100); 4.5 bits per element.
* ``"mxfp4"``: blocks of 32 along K with a power-of-two scale (the smallest 2^e with the block's largest magnitude <=
  6 * 2^e, at least 2^-126, so nothing saturates); 4.25 bits per element.

Codes are rounded to nearest, ties to even.  Values are exact in bf16, so reading back loses nothing more (a magnitude
within a code's rounding of bf16's largest can round up past it, and reads back as infinity).  An infinity or NaN makes its
block (mxfp4) or row (nvfp4) read back as NaN.

A matrix is stored as the shared-memory images the kernels load (csrc/fp4.cuh), rows in blocks of 128 and columns in tiles
of 256.  The operators launch on the current stream of the tensors' device and can be captured in a CUDA graph; weights
must not be rewritten while a call that reads them runs.

Row counts and numerics of ``linear4`` / ``mlp4``:

* ``act4=False``, and up to 16 rows always: bf16 activations (W4A16).  Up to 96 rows each is expanded into 4-bit terms
  for the 4-bit tensor cores, which leaves out at most 2^-22 of the largest magnitude of its block of 16 (nvfp4) or 32
  (mxfp4) columns, in nvfp4 2^-39 of the row's where that is more, and up to 2^-124 of rows below 2^-85 (nvfp4) or blocks
  below 2^-105 (mxfp4); with more rows the weights are widened to bf16 inside the product, exactly.  A row's result thus
  does not depend on the other rows, but its last bits on their number;
* ``act4=True``, more than 16 rows: activations are quantised per row to the weights' format and multiplied on the
  block-scaled tensor cores (W4A4).

Sums are fp32 and added in a fixed order: a call repeats itself bit for bit.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _ext
from .kernels import GEMV_BF16, GEMV_F32, GEMV_F32_ACC  # noqa: F401  (the output modes of linear4 / mlp4)

FORMATS = ("nvfp4", "mxfp4")


def _nv(fmt: str) -> bool:
    if fmt not in FORMATS:
        raise ValueError(f"unknown 4-bit format {fmt!r} (one of {', '.join(FORMATS)})")
    return fmt == "nvfp4"


class Matrix4:
    """A 4-bit matrix [rows, k] on a CUDA device.  ``codes`` and ``scales`` are the tile images (uint8, flat),
    ``row_scale`` the fp32 row scales of nvfp4 (None for mxfp4)."""

    __slots__ = ("handle",)

    def __init__(self, handle):
        self.handle = handle

    @classmethod
    def from_parts(cls, codes, scales, row_scale, rows: int, k: int, fmt: str) -> "Matrix4":
        """A matrix from arrays in the layout of ``codes``, ``scales`` and ``row_scale``.  Codes and scales of the columns
        from k up to a multiple of 256 must be 0, as ``quantize4`` leaves them; every row scale a power of two."""
        return cls(_ext.require().Matrix4(codes, scales, row_scale, rows, k, _nv(fmt)))

    @property
    def codes(self) -> torch.Tensor:
        return self.handle.codes

    @property
    def scales(self) -> torch.Tensor:
        return self.handle.scales

    @property
    def row_scale(self) -> torch.Tensor | None:
        return self.handle.row_scale

    @property
    def rows(self) -> int:
        return self.handle.rows

    @property
    def k(self) -> int:
        return self.handle.k

    @property
    def fmt(self) -> str:
        return "nvfp4" if self.handle.nv else "mxfp4"

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + (4 * self.rows if self.handle.nv else 0)


def quantize4(x: torch.Tensor, fmt: str = "nvfp4") -> Matrix4:
    """Rows of ``x`` [R, K] (bf16 or f16, unit inner stride; K a multiple of 16 for nvfp4, of 32 for mxfp4) to 4 bits."""
    return Matrix4(_ext.require().fp4_quantize(x, _nv(fmt)))


def dequantize4(m: Matrix4, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of ``m`` as [rows, k] in bf16, f16 or fp32 (``out``: written there, its type)."""
    return _ext.require().fp4_dequantize(m.handle, out, dtype)


def linear4(x: torch.Tensor, w: Matrix4, y: torch.Tensor, mode: int = GEMV_BF16, act4: bool = False) -> torch.Tensor:
    """y [M, N] (mode: GEMV_BF16, GEMV_F32 or GEMV_F32_ACC) = x [M, K] bf16 @ w [N, K]^T; ``act4``: 4-bit activations
    above 16 rows."""
    _ext.require().fp4_linear(x, w.handle, y, mode, act4)
    return y


@dataclass
class MLP4:
    """A gated feed-forward block in 4 bits: ``gu`` holds per 128-row block 64 gate rows, then their 64 up rows (the
    last block padded with zero rows), ``down`` is [N, width]."""
    gu: Matrix4
    down: Matrix4
    width: int

    @property
    def nbytes(self) -> int:
        return self.gu.nbytes + self.down.nbytes


def pack_mlp4(gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, fmt: str = "nvfp4") -> MLP4:
    """Gate and up [width, K] and down [N, width] (bf16 or f16, width a multiple of 32) to an ``MLP4``."""
    W, K = gate.shape
    if up.shape != gate.shape or up.dtype != gate.dtype or up.device != gate.device:
        raise ValueError("pack_mlp4: gate and up must have one shape, type and device")
    if down.dim() != 2 or down.shape[1] != W or down.device != gate.device:
        raise ValueError(f"pack_mlp4: down must be [N, {W}] on the device of gate")
    if W % 32:
        raise ValueError(f"pack_mlp4: the width must be a multiple of 32, got {W}")
    blocks = (W + 63) // 64
    gu = torch.zeros(blocks, 2, 64, K, dtype=gate.dtype, device=gate.device)
    for half, t in enumerate((gate, up)):
        whole = W // 64
        gu[:whole, half] = t[:whole * 64].view(whole, 64, K)
        if W % 64:
            gu[whole, half, :W % 64] = t[whole * 64:]
    return MLP4(quantize4(gu.view(blocks * 128, K), fmt), quantize4(down, fmt), W)


def mlp4(x: torch.Tensor, m: MLP4, y: torch.Tensor, limit: float, mode: int = GEMV_F32,
         act4: bool = False) -> torch.Tensor:
    """y [M, N] (mode) = h @ down^T with h = silu(min(g, limit)) * clip(u, -limit, limit), [g | u] = x [gate | up]^T.

    h is held in bf16, or with ``act4`` (above 16 rows) in the weights' 4-bit format; nvfp4 then takes its row scale from
    max(limit, 0.2785) * limit (limit must be finite), which no |h| exceeds, instead of the row's maximum, so that h is
    quantised where it is computed.  A block of h then keeps its precision down to about 2^-14 of that bound and is 0 from
    about 2^-18 of it on; nvfp4 gate and up rows with magnitudes above 2^100 may then overflow on the way."""
    _ext.require().fp4_mlp(x, m.gu.handle, m.down.handle, y, limit, mode, act4)
    return y


def check_errors(device=None, wait: bool = True) -> None:
    """Raise if a bounded wait of these kernels ran out on ``device`` since the last check; what they wrote then is not to be
    used.  Waits for every stream of the device, or (``wait=False``) for the current one only.  Not inside a capture."""
    dev = torch.device("cuda" if device is None else device)
    if wait:
        torch.cuda.synchronize(dev)
    code = _ext.require().fp4_error(torch.cuda.current_device() if dev.index is None else dev.index)
    if code:
        raise RuntimeError(f"4-bit kernels: a bounded wait ran out (code {code:#x})")
