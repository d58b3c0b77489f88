"""The gated feed-forward block: ``(act(x Wg^T) * (x Wu^T)) Wd^T``."""

from __future__ import annotations

import torch

from .. import _ext
from . import _any_transformed, _warn_torch_path, use_kernels
from . import reference as ref

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu") -> torch.Tensor:
    """``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T`` for ``(..., hidden)`` inputs, ``(inter, hidden)`` gate and up weights
    (which may be slices of one matrix) and a ``(hidden, inter)`` down weight.  ``activation``: ``"silu"``, ``"gelu"`` (exact),
    ``"gelu_tanh"`` or ``"relu"``.

    bf16 CUDA tensors whose sizes are multiples of 8 run the sm_100a kernels: both projections, the activation and the product are
    one of them, as are the down projection's gradient and the gates' on the way back.  The activation sees the projections before
    they are rounded, so that the result is nearer to the exact one than that of :func:`swiglu` on finished projections, and not
    its bits.  Few rows (up to 32, 64 where a weight has 2 ** 24 values or fewer, 384 where rows times those are 4e8 or less)
    run kernels that stream the weights.  Differentiable once in all four; the backward pass needs ``x``, and keeps 8 bytes for each
    row and intermediate feature until then.  The gradients of ``w_gate`` and ``w_up`` are made together, as the halves of one tensor,
    whichever of them is asked for: either keeps the memory of both.  Under vmap and forward-mode differentiation the PyTorch
    formulation runs."""
    number = ACTIVATIONS.get(activation)
    if number is None:
        raise RuntimeError(f"himuon_b200.ops.gated_mlp: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or not x.is_floating_point():
        raise RuntimeError("himuon_b200.ops.gated_mlp: (..., hidden) inputs and (inter, hidden) weights of floating point "
                           "expected")
    shape = w_gate.shape
    inter, hidden = shape
    if x.shape[-1] != hidden or w_up.shape != shape or w_down.shape != (hidden, inter) or not hidden or not inter:
        raise RuntimeError(f"himuon_b200.ops.gated_mlp: sizes disagree: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, "
                           f"w_up {tuple(w_up.shape)}, w_down {tuple(w_down.shape)}")
    dtype, device = x.dtype, x.device
    if (w_gate.dtype != dtype or w_up.dtype != dtype or w_down.dtype != dtype or w_gate.device != device
            or w_up.device != device or w_down.device != device):
        raise RuntimeError("himuon_b200.ops.gated_mlp: inputs and weights must be of one type on one device")
    transformed = _any_transformed(x, w_gate, w_up, w_down)
    if use_kernels(x) and hidden % 8 == 0 and inter % 8 == 0 and not transformed:
        return _ext.ext().gated_mlp(x, w_gate, w_up, w_down, number)
    if use_kernels(x):
        _warn_torch_path("gated_mlp", "under vmap or forward-mode differentiation" if transformed else
                         f"sizes of {hidden} and {inter} (the kernels take multiples of 8)")
    return ref.gated_mlp(x, w_gate, w_up, w_down, activation)
