"""Rotary positions: both layouts of the pairs, any part of the head, any position, frequencies scaled for long contexts.

:func:`head_norm_rope` turns whole heads by a table of the positions of one sequence, with the heads' norm on the way.
:func:`rotary` takes the positions themselves and needs no table: the angle of a position is exact wherever it lies.
"""

from __future__ import annotations

import math

import torch

from .. import _ext
from . import _any_transformed, _check_width, _warn_torch_path
from . import reference as ref

TWO_PI_E50 = 628318530717958647692528676655900576839433879875021      # 2 pi * 10^50
SCALINGS = ("linear", "ntk", "yarn", "llama3")
# What each of them is made of.  Any other key is refused: it may change the frequencies, and nothing would say so.
LENGTH = "original_max_position_embeddings"
SCALING_KEYS = {
    "default": (), "linear": ("factor",), "ntk": ("factor",),
    "yarn": ("factor", LENGTH, "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"),
    "llama3": ("factor", LENGTH, "low_freq_factor", "high_freq_factor"),
}


def _number(op: str, d: dict, key: str, default=None, least: float = 0.0) -> float:
    value = d.get(key, default)
    if value is None:
        raise RuntimeError(f"himuon_b200.ops.{op}: scaling needs {key}")
    value = float(value)
    if not (math.isfinite(value) and value > least):
        raise RuntimeError(f"himuon_b200.ops.{op}: {key} must be above {least}, got {value}")
    return value


def _form(op: str, theta: float, scaling: dict) -> tuple[str, dict]:
    """The form of a scaling and what it is made of."""
    scaling = {k: v for k, v in scaling.items() if v is not None}      # (a key without a value is not there)
    names = [scaling[k] for k in ("rope_type", "type") if k in scaling]
    if not names:
        raise RuntimeError(f"himuon_b200.ops.{op}: scaling needs rope_type, one of {SCALINGS}")
    kind = names[0]
    if names[-1] != kind or kind not in ("default", *SCALINGS):
        raise RuntimeError(f"himuon_b200.ops.{op}: rope_type must be one of {SCALINGS}, got {' and '.join(map(repr, names))}")
    if float(scaling.get("rope_theta", theta)) != theta:
        raise RuntimeError(f"himuon_b200.ops.{op}: rope_theta of the scaling is {scaling['rope_theta']}, theta is {theta}")
    # (a length may always be there: the forms that do not name it have no use for one)
    unknown = [str(k) for k in scaling if k not in (*SCALING_KEYS[kind], "rope_type", "type", "rope_theta", LENGTH)]
    if unknown:
        raise RuntimeError(f"himuon_b200.ops.{op}: a scaling of rope_type {kind} takes {SCALING_KEYS[kind]}, "
                           f"got {', '.join(unknown)}")
    return kind, scaling


def _frequencies(rotary_dim: int, theta: float, scaling: dict | None) -> tuple[list[float], float]:
    """(angle of each pair at position 1 in 64 bits, factor of cosine and sine)."""
    op, pairs, kind = "RotaryFrequencies", rotary_dim // 2, "default"
    if scaling is not None:
        kind, scaling = _form(op, theta, scaling)
    if kind == "default":
        return [theta ** (-2.0 * i / rotary_dim) for i in range(pairs)], 1.0
    factor = _number(op, scaling, "factor")
    if kind == "ntk":                    # a larger base: the last pair ends up `factor` times as long, the first as it was
        if rotary_dim > 2:
            theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
        return [theta ** (-2.0 * i / rotary_dim) for i in range(pairs)], 1.0
    inv = [theta ** (-2.0 * i / rotary_dim) for i in range(pairs)]
    if kind == "linear":
        return [f / factor for f in inv], 1.0
    length = _number(op, scaling, LENGTH)
    if kind == "yarn":
        # pairs that turn often within the original length stay, those that do not turn once are stretched, a ramp between them
        fast, slow = _number(op, scaling, "beta_fast", 32.0), _number(op, scaling, "beta_slow", 1.0)

        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        truncate = scaling.get("truncate", True)
        if not isinstance(truncate, bool):
            raise RuntimeError(f"himuon_b200.ops.{op}: truncate must be true or false, got {truncate!r}")
        lo, hi = pair_of(fast), pair_of(slow)
        if truncate:                     # the ramp starts and ends at whole pairs
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        span = float(hi - lo) if hi != lo else 0.001

        def stretch(k: float) -> float:
            return 0.1 * k * math.log(factor) + 1.0 if factor > 1.0 else 1.0

        if "attention_factor" in scaling:
            attention = _number(op, scaling, "attention_factor")
        elif "mscale" in scaling or "mscale_all_dim" in scaling:      # (both: readers differ on what one of them means)
            attention = stretch(_number(op, scaling, "mscale")) / stretch(_number(op, scaling, "mscale_all_dim"))
        else:
            attention = stretch(1.0)
        out = []
        for i, f in enumerate(inv):
            ramp = min(max((i - lo) / span, 0.0), 1.0)
            out.append(f / factor * ramp + f * (1.0 - ramp))
        return out, attention
    low, high = _number(op, scaling, "low_freq_factor"), _number(op, scaling, "high_freq_factor")
    if high <= low:
        raise RuntimeError(f"himuon_b200.ops.{op}: high_freq_factor must be above low_freq_factor")
    out = []
    for f in inv:                        # by how often a pair turns within the original length
        kept = min(max((length * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
        out.append(f / factor * (1.0 - kept) + f * kept)
    return out, 1.0


class RotaryFrequencies:
    """How fast the pairs of a head turn.  Made once for a model, outside of a graph's capture; every layer uses it.

    ``rotary_dim``: how many values of a head are turned, the first ones (even, 0 included).  Pair ``i`` turns by ``theta ** (-2 i
    / rotary_dim)`` a position.  ``scaling``: as ``rope_scaling`` in a model's configuration, with ``rope_type`` ``"linear"`` (all
    frequencies divided by ``factor``), ``"ntk"`` (a larger ``theta``, by ``factor ** (d / (d - 2))``), ``"yarn"`` (``factor``,
    ``original_max_position_embeddings``, ``beta_fast``, ``beta_slow``, ``truncate``, and ``attention_factor`` or ``mscale`` with
    ``mscale_all_dim``) or ``"llama3"`` (``factor``, ``low_freq_factor``, ``high_freq_factor``,
    ``original_max_position_embeddings``).  Keys whose value is ``None`` count as absent; other keys are refused, as is a
    ``rope_theta`` other than ``theta``.

    ``frequencies``: the angles at position 1 as floats; ``factor``: what cosine and sine are multiplied by (other than 1 with
    yarn).
    """

    def __init__(self, rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None, device="cuda"):
        if not isinstance(rotary_dim, int) or rotary_dim < 0 or rotary_dim % 2:
            raise RuntimeError("himuon_b200.ops.RotaryFrequencies: rotary_dim must be an even number of values, "
                               f"got {rotary_dim!r}")
        if not (math.isfinite(theta) and theta > 1.0):
            raise RuntimeError(f"himuon_b200.ops.RotaryFrequencies: theta must be above 1, got {theta}")
        self.rotary_dim, self.theta, self.scaling = rotary_dim, float(theta), None if scaling is None else dict(scaling)
        self.frequencies, self.factor = _frequencies(rotary_dim, self.theta, self.scaling)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("himuon_b200.ops.RotaryFrequencies: they would be copied from the host while a graph is captured; "
                               "make them before the capture")
        # whole numbers of 2^-64 turns a position: position times this, modulo 2^64, is the place within a turn
        ratios = (f.as_integer_ratio() for f in self.frequencies)
        turns = [((n * 2 ** 65 * 10 ** 50) // (d * TWO_PI_E50) + 1) // 2 % 2 ** 64 for n, d in ratios]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64).to(self.device)
        if self.device.type == "cuda":
            torch.cuda.current_stream(self.device).synchronize()       # calls on any stream find it there


def rotary(x2d, positions, freqs: RotaryFrequencies, heads: int, head_dim: int, interleaved: bool = False):
    """Turns the first ``freqs.rotary_dim`` values of every head of ``(rows, heads*head_dim)`` rows (which may be a column slice:
    queries and keys of one projection are turned by one call) by their position; the values behind them pass through.

    ``positions``: int64, one for each row (any value; ``PackedLayout.positions`` has those of a packed batch), or the length
    ``S`` of sequences that lie one after the other, whose rows have positions ``0..S-1``.  Pairs are ``(i, i + rotary_dim / 2)``,
    or ``(2 i, 2 i + 1)`` with ``interleaved``.  Returns a new contiguous tensor of the type of ``x2d``; differentiable in
    ``x2d``, any number of times.  bf16 and fp32 CUDA tensors run the sm_100a kernel, in fp32; under vmap and forward-mode
    differentiation the PyTorch formulation runs."""
    if not isinstance(freqs, RotaryFrequencies):
        raise RuntimeError("himuon_b200.ops.rotary: freqs must be a RotaryFrequencies")
    if x2d.dim() != 2 or not x2d.is_floating_point() or heads <= 0 or head_dim <= 0:
        raise RuntimeError("himuon_b200.ops.rotary: (rows, heads*head_dim) of floating point expected")
    _check_width("rotary", x2d, heads * head_dim)
    if freqs.rotary_dim > head_dim:
        raise RuntimeError(f"himuon_b200.ops.rotary: {freqs.rotary_dim} values to be turned in heads of {head_dim}")
    if freqs.device != x2d.device:
        raise RuntimeError(f"himuon_b200.ops.rotary: the frequencies are on {freqs.device}, the tensor on {x2d.device}")
    rows, seq_len = x2d.shape[0], 1
    if isinstance(positions, torch.Tensor):
        if positions.dtype != torch.int64 or positions.dim() != 1 or positions.shape[0] != rows or positions.device != x2d.device:
            raise RuntimeError(f"himuon_b200.ops.rotary: positions must be int64, one for each of the {rows} rows, "
                               f"on {x2d.device}")
        positions = positions.contiguous()
    else:
        seq_len, positions = positions, None
        if not isinstance(seq_len, int) or seq_len <= 0 or rows % seq_len:
            raise RuntimeError("himuon_b200.ops.rotary: positions must be a tensor or the length of sequences that "
                               f"{rows} rows hold, got {seq_len!r}")
    transformed = _any_transformed(x2d) if positions is None else _any_transformed(x2d, positions)
    if x2d.is_cuda and x2d.dtype in (torch.bfloat16, torch.float32) and not transformed:
        if x2d.stride(1) != 1 and x2d.shape[1] > 1:
            x2d = x2d.clone(memory_format=torch.contiguous_format)
        return _ext.ext().rotary(x2d, positions, freqs.turns, seq_len, heads, freqs.rotary_dim, bool(interleaved), freqs.factor)
    if x2d.is_cuda and transformed:
        _warn_torch_path("rotary", "under vmap or forward-mode differentiation")
    if positions is None:
        positions = torch.arange(rows, device=x2d.device) % seq_len
    inv = torch.tensor(freqs.frequencies, dtype=torch.float64, device=x2d.device)
    return ref.rotary(x2d, positions, inv, freqs.factor, heads, head_dim, bool(interleaved))
