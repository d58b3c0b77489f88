"""8-bit floating point with a scale for each block of 128: quantisation, products, and a linear layer in it.

Values are e4m3 (3 bits of mantissa, largest 448).  A scale belongs to a block of 128 values of a row, or of 128 x 128 values of a
matrix; here it is a power of two, the least that leaves the block's largest value at 448 or below, so that a value is rounded
once and by nothing else.  Products take any fp32 scales.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _ext
from . import _any_transformed, _warn_torch_path
from . import reference as ref

BLOCK = 128


class Fp8Blocks(NamedTuple):
    """A matrix in 8 bits.  ``values``: ``(rows, cols)`` of ``float8_e4m3fn``.  ``scales``: fp32, one for each block of
    ``(block_rows, 128)`` values, ``(ceil(rows / block_rows), ceil(cols / 128))`` with any strides; ``block_rows`` is 1 or 128.
    ``powers``: every scale is known to be a power of two (from ``2**-126`` on), as those of :func:`quantize_fp8` are; products of
    two such matrices leave the scales to the tensor core.  Nobody looks at the scales: where it is set and they are others,
    results are wrong."""

    values: torch.Tensor
    scales: torch.Tensor
    block_rows: int = 1
    powers: bool = False

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the 8 bits stand for, in fp32 or rounded to bf16.  Under vmap the PyTorch formulation runs."""
        _check("Fp8Blocks.dequantize", self)
        if dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError(f"himuon_b200.ops.Fp8Blocks.dequantize: float32 or bfloat16 expected, got {dtype}")
        if self.values.is_cuda and _kernels("Fp8Blocks.dequantize", self.values, self.scales):
            return _ext.ext().fp8_dequantize(self.values, self.scales, self.block_rows, dtype == torch.float32)
        return ref.fp8_dequantize(self.values, self.scales, self.block_rows).to(dtype)


def _check(op: str, m: Fp8Blocks) -> None:
    if not isinstance(m, Fp8Blocks):
        raise RuntimeError(f"himuon_b200.ops.{op}: an Fp8Blocks expected")
    if m.block_rows not in (1, BLOCK) or m.values.dim() != 2 or m.values.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"himuon_b200.ops.{op}: a float8_e4m3fn matrix with blocks of 1 or {BLOCK} rows expected")
    rows, cols = m.values.shape
    blocks = (-(-rows // m.block_rows), -(-cols // BLOCK))
    if m.scales.dtype != torch.float32 or tuple(m.scales.shape) != blocks or m.scales.device != m.values.device:
        raise RuntimeError(f"himuon_b200.ops.{op}: scales must be fp32 of {blocks} on {m.values.device}, "
                           f"got {m.scales.dtype} of {tuple(m.scales.shape)}")


def _kernels(op: str, *tensors: torch.Tensor) -> bool:
    """Whether the kernels can have them: not under a transform, which gives tensors without memory."""
    if not _any_transformed(*tensors):
        return True
    _warn_torch_path(op, "under vmap or forward-mode differentiation")
    return False


def quantize_fp8(x2d: torch.Tensor, block_rows: int = 1, transpose: bool = False) -> Fp8Blocks:
    """``x2d`` (bf16 or fp32) in 8 bits, with a scale for each block of ``(block_rows, 128)``; with ``transpose`` ``x2d.T``, whose
    blocks are then meant.

    ``block_rows``: 1 for activations (a row's values depend on no other row), 128 for weights.  A value that is not finite
    becomes NaN and has no part in its block's scale; a block of zeros has scale 1; no scale is below ``2**-110``.  CUDA tensors
    run the sm_100a kernel.  Not differentiable."""
    if x2d.dim() != 2 or x2d.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError("himuon_b200.ops.quantize_fp8: a bf16 or fp32 matrix expected")
    if block_rows not in (1, BLOCK):
        raise RuntimeError(f"himuon_b200.ops.quantize_fp8: blocks of 1 or {BLOCK} rows, got {block_rows}")
    if _any_transformed(x2d):
        raise RuntimeError("himuon_b200.ops.quantize_fp8: not under vmap or forward-mode differentiation")
    if x2d.is_cuda:
        return Fp8Blocks(*_ext.ext().quantize_fp8(x2d, block_rows, bool(transpose)), block_rows, True)
    x2d = x2d.detach()
    return Fp8Blocks(*ref.quantize_fp8(x2d.t() if transpose else x2d, block_rows), block_rows, True)


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T`` of two 8-bit matrices ``(rows, inner)`` and ``(cols, inner)``, in bf16 or fp32.  ``a`` has blocks of 1 or 128
    rows, ``b`` of 128 (as a weight has).  The products of a block are summed by the tensor core, the blocks, scaled, in fp32 (by
    the product of two scales, which has to be a normal fp32 number).  Few rows (up to 16, or 32 of a small ``b``) run a kernel
    that streams ``b``.  Not differentiable: see :func:`fp8_linear`.  Under vmap the PyTorch formulation runs."""
    _check("fp8_matmul", a)
    _check("fp8_matmul", b)
    if a.values.shape[1] != b.values.shape[1] or a.values.device != b.values.device:
        raise RuntimeError("himuon_b200.ops.fp8_matmul: (rows, inner) and (cols, inner) on one device expected")
    if b.block_rows != BLOCK:
        raise RuntimeError(f"himuon_b200.ops.fp8_matmul: the second operand needs blocks of {BLOCK} rows")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"himuon_b200.ops.fp8_matmul: bfloat16 or float32 expected, got {out_dtype}")
    if a.values.is_cuda and _kernels("fp8_matmul", a.values, a.scales, b.values, b.scales):
        return _ext.ext().fp8_matmul(*a, *b, out_dtype == torch.float32)
    return (ref.fp8_dequantize(*a[:3]) @ ref.fp8_dequantize(*b[:3]).t()).to(out_dtype)


def fp8_linear(x: torch.Tensor, w) -> torch.Tensor:
    """``x @ w.T`` in 8 bits for ``(..., in)`` inputs.

    ``w``, a ``(out, in)`` tensor: inputs and weight are put into 8 bits on the way (rows of ``x`` by themselves, ``w`` in blocks
    of 128 x 128), and so are the products of the backward pass: ``dy`` by rows times ``w``, and ``dy.T`` by rows times ``x.T`` in
    blocks of 128 x 128.  The gradients are those of the product of the rounded operands.  Kept until the backward pass: one byte
    for each value of ``x`` and of ``w``.  Differentiable once.

    ``w``, an :class:`Fp8Blocks` with blocks of 128 rows: a weight kept in 8 bits, for use without gradients.

    bf16 CUDA tensors run the sm_100a kernels; under vmap and forward-mode differentiation the PyTorch formulation runs, in which
    rounding has the derivative of doing nothing and ``dy`` is not rounded."""
    kept = isinstance(w, Fp8Blocks)
    if kept:
        _check("fp8_linear", w)
        if w.block_rows != BLOCK:
            raise RuntimeError(f"himuon_b200.ops.fp8_linear: a kept weight needs blocks of {BLOCK} rows")
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("himuon_b200.ops.fp8_linear: a weight kept in 8 bits passes no gradient on; "
                               "give the weight itself, or call under no_grad()")
    shape = w.values.shape if kept else w.shape
    device = w.values.device if kept else w.device
    if (x.dim() < 1 or len(shape) != 2 or x.shape[-1] != shape[1] or device != x.device or not x.is_floating_point()
            or not (kept or w.dtype == x.dtype)):
        raise RuntimeError("himuon_b200.ops.fp8_linear: (..., in) inputs and an (out, in) weight of one floating point type "
                           "on one device expected")
    transformed = _any_transformed(x, w.values, w.scales) if kept else _any_transformed(x, w)
    kernels = x.is_cuda and x.dtype == torch.bfloat16
    if kernels and not transformed:
        return _ext.ext().fp8_linear_kept(x, *w) if kept else _ext.ext().fp8_linear(x, w)
    if kernels:
        _warn_torch_path("fp8_linear", "under vmap or forward-mode differentiation")
    x2d, out = x.reshape(math.prod(x.shape[:-1]), shape[1]), (*x.shape[:-1], shape[0])
    if kept:
        return (ref.fp8_dequantize(*ref.quantize_fp8(x2d.detach(), 1), 1) @ ref.fp8_dequantize(*w[:3]).t()).to(x.dtype).view(out)
    return (ref.fp8_linear_any if transformed else ref.fp8_linear)(x2d, w).view(out)
