"""Causal attention over documents of different lengths packed into one row of tokens.

A batch of ``n`` documents is one ``(rows, features)`` matrix: document after document, padding (if any) behind the last one.
:class:`PackedLayout` holds the documents' lengths and the list of 128-token tiles that the sm_100a kernels walk; it is made
once for a batch and shared by every layer.  Padding rows attend to nothing and are attended by nothing: their output and
their gradients are zero.
"""

from __future__ import annotations

import math
import operator

import numpy as np
import torch
from torch.nn.attention import SDPBackend, sdpa_kernel

from .. import _ext
from . import _any_transformed, _check_width, _count, _warn_torch_path, _with_rows_apart, use_kernels
from . import reference as ref

TILE = 128          # tokens of one document that a block of the kernels takes


def _tile_plan(lengths: np.ndarray) -> tuple[np.ndarray, int]:
    """``(2 * tiles + pairs, 4)`` int32 and the number of tiles.  Every tile as (first row of its document, length of it, number
    in the document, number in the batch): by falling work of the passes over a tile's keys, by falling work of the pass over
    its queries, and the first of two and two of a document by falling work of both."""
    first = np.cumsum(lengths) - lengths
    per_doc = (lengths + TILE - 1) // TILE
    doc = np.repeat(np.arange(lengths.size), per_doc)
    slot = np.arange(doc.size)
    index = slot - np.repeat(np.cumsum(per_doc) - per_doc, per_doc)
    tiles = np.stack([first[doc], lengths[doc], index, slot], axis=1)
    keys = np.minimum((index + 1) * TILE, lengths[doc])
    queries = lengths[doc] - index * TILE
    even = np.flatnonzero(index % 2 == 0)
    both = keys[even] + np.where((index[even] + 1) * TILE < lengths[doc[even]], np.minimum((index[even] + 2) * TILE, lengths[doc[even]]), 0)
    orders = [np.argsort(-keys, kind="stable"), np.argsort(-queries, kind="stable"), even[np.argsort(-both, kind="stable")]]
    return np.ascontiguousarray(tiles[np.concatenate(orders)], dtype=np.int32), slot.size


class PackedLayout:
    """Where the documents of a packed batch lie.

    ``lengths``: the documents' lengths in tokens, zero included (a sequence of whole numbers, or an integer tensor; one on a
    GPU is read back, which waits for it).  ``device``: where the batch lives.  The device-side tables are copied without a wait on
    the stream that is current when they are first needed; calls on other streams wait for them.  A graph may hold calls with a layout
    whose tables are there before its capture, and needs the layout for as long as it is replayed.
    """

    def __init__(self, lengths, device="cuda"):
        if isinstance(lengths, torch.Tensor):
            if lengths.dim() != 1 or lengths.is_floating_point() or lengths.dtype == torch.bool:
                raise RuntimeError("himuon_b200.ops.PackedLayout: lengths must be a 1-D integer tensor or a sequence of whole numbers")
            lengths = lengths.tolist()
        try:
            self.lengths = tuple(operator.index(n) for n in lengths)
        except TypeError as e:
            raise RuntimeError(f"himuon_b200.ops.PackedLayout: lengths must be whole numbers: {e}") from None
        if any(n < 0 for n in self.lengths):
            raise RuntimeError("himuon_b200.ops.PackedLayout: a length is negative")
        self.tokens = sum(self.lengths)
        if self.tokens >= 2 ** 30:
            raise RuntimeError(f"himuon_b200.ops.PackedLayout: {self.tokens} tokens in one batch (2**30 - 1 at most)")
        self.max_length = max(self.lengths, default=0)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        lens = np.asarray(self.lengths, dtype=np.int64)
        self._position = np.arange(self.tokens) - np.repeat(np.cumsum(lens) - lens, lens)
        self._tables: dict = {}
        plan, self.tiles = _tile_plan(lens)
        of = plan[self.tiles: 2 * self.tiles]
        self._query_steps = int(((of[:, 1] - of[:, 2] * TILE + 63) // 64).sum())   # of 64 queries, over all tiles, for one head
        self._table("plan", lambda: plan)

    def _table(self, key, make=None) -> torch.Tensor:
        """The device copy of a host table, safe to use on the current stream."""
        entry = self._tables.get(key)
        on_gpu = self.device.type == "cuda"
        if entry is None:
            if on_gpu and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("himuon_b200.ops.PackedLayout: a table would be copied from the host while a graph is captured; "
                                   "make the layout, and call what uses it once, before the capture")
            host = torch.from_numpy(make())
            if not on_gpu:
                entry = (host.to(self.device), None, None)
            else:
                stream = torch.cuda.current_stream(self.device)
                table = host.pin_memory().to(self.device, non_blocking=True)
                event = torch.cuda.Event()
                event.record(stream)
                entry = (table, stream, event)
            self._tables[key] = entry
        table, stream, event = entry
        if on_gpu and torch._C._cuda_getCurrentRawStream(self.device.index) != stream.cuda_stream and not torch.cuda.is_current_stream_capturing():
            # (a stream that captures a graph has been synchronised with what came before)
            here = torch.cuda.current_stream(self.device)
            here.wait_event(event)
            table.record_stream(here)
        return table

    @property
    def plan(self) -> torch.Tensor:
        return self._table("plan")

    def _check_rows(self, op: str, rows: int) -> None:
        if rows < self.tokens:
            raise RuntimeError(f"himuon_b200.ops.{op}: {rows} rows for a layout of {self.tokens} tokens")

    def splits_heads(self, Hq: int, Hkv: int) -> bool:
        """Whether the pass for dK and dV takes each query head by itself and sums the heads of a group afterwards.

        A block otherwise goes through all heads of a group, and in a small batch the longest one sets the time: one document of
        1024 tokens, 32 heads over 8, 61 us whole, 35 + 9 in parts; 2048 tokens, 16 over 8, 62 and 48 + 10.  A larger batch fills the
        GPU either way and pays for the parts (4096 tokens, 32 over 8, 225 and 264 + 40), a tiny one saves less than their sum
        costs (300 tokens, 16 over 8, 16.6 and 16.6 + 3)."""
        steps = -(-self.max_length // 64)                                     # of 64 queries, for one head of the longest tile
        group = Hq // Hkv
        return (group - 1) * steps >= 16 and group * steps > 2 * self._query_steps * Hq / _ext.ext().num_sms()

    def positions(self, rows: int | None = None) -> torch.Tensor:
        """Each row's position in its own document (int64), 0 for the padding of a batch of ``rows`` rows."""
        rows = self.tokens if rows is None else rows
        self._check_rows("PackedLayout.positions", rows)
        return self._table(("positions", rows), lambda: np.concatenate([self._position, np.zeros(rows - self.tokens, dtype=np.int64)]))

    def has_next(self, rows: int | None = None) -> torch.Tensor:
        """Whether a row is followed by a token of its own document."""
        rows = self.tokens if rows is None else rows
        self._check_rows("PackedLayout.has_next", rows)

        def make():
            out = np.zeros(rows, dtype=bool)
            out[: max(self.tokens - 1, 0)] = self._position[1:] > 0
            return out
        return self._table(("has_next", rows), make)

    def next_ids(self, ids: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
        """For each row of a packed ``ids`` the id that follows it in its document, ``ignore_index`` where none does."""
        flat = ids.reshape(-1)
        return torch.where(self.has_next(flat.numel()), torch.roll(flat, -1), ignore_index)

    def rope_table(self, cos_sin: torch.Tensor, rows: int | None = None) -> torch.Tensor:
        """The rows of a rotary table ``(max position, head_dim / 2, 2)`` that the batch's tokens need, one for each row: what
        :func:`head_norm_rope` takes as the table of one sequence of ``rows`` positions."""
        if cos_sin.shape[0] < self.max_length:
            raise RuntimeError(f"himuon_b200.ops.PackedLayout.rope_table: {cos_sin.shape[0]} positions, a document has {self.max_length}")
        return cos_sin.index_select(0, self.positions(rows))


def packed_attention(q2d, k2d, v2d, layout: PackedLayout, Hq: int, Hkv: int, head_dim: int, scale: float | None = None):
    """Causal GQA attention within each document of a packed batch, on ``(rows, heads*head_dim)`` views (``rows`` at least
    ``layout.tokens``; rows behind that are padding); returns ``(rows, Hq*head_dim)``.  ``scale`` defaults to
    ``1/sqrt(head_dim)`` and must be positive.  bf16 CUDA tensors with heads of a multiple of 8 up to 128 run the sm_100a kernels,
    forward and backward; under vmap and forward-mode differentiation, for which those have no rules, the PyTorch formulation runs.

    What is in other documents or in the padding has no part in a row, NaN and infinities included.  Those of a later token of the
    row's own document have weight 0, which does not take them out: as in :func:`attention`, a token that is not finite may reach
    neighbours that do not see it."""
    if not isinstance(layout, PackedLayout):
        raise RuntimeError("himuon_b200.ops.packed_attention: layout must be a PackedLayout")
    scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise RuntimeError(f"himuon_b200.ops.packed_attention: scale must be positive, got {scale}")
    if Hq <= 0 or Hkv <= 0 or Hq % Hkv:
        raise RuntimeError(f"himuon_b200.ops.packed_attention: {Hq} query heads over {Hkv}")
    rows = q2d.shape[0]
    for t, heads in ((q2d, Hq), (k2d, Hkv), (v2d, Hkv)):
        if t.dim() != 2 or t.shape[0] != rows or t.device != q2d.device or t.dtype != q2d.dtype:
            raise RuntimeError("himuon_b200.ops.packed_attention: q, k and v are (rows, heads*head_dim) of one type on one device")
        _check_width("packed_attention", t, heads * head_dim)
    layout._check_rows("packed_attention", rows)
    if layout.device != q2d.device:
        raise RuntimeError(f"himuon_b200.ops.packed_attention: the layout is on {layout.device}, the tensors on {q2d.device}")
    transformed = _any_transformed(q2d, k2d, v2d)
    if use_kernels(q2d) and head_dim <= 128 and head_dim % 8 == 0 and not transformed:
        q, k, v = _with_rows_apart(q2d), _with_rows_apart(k2d), _with_rows_apart(v2d)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _ext.ext().packed_attention(q, k, v, layout.plan, layout.tiles, layout.tokens, Hq, Hkv, scale, layout.splits_heads(Hq, Hkv))
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        if layout.tiles:
            _ext.ext().packed_attn_fwd(layout.plan, layout.tiles, layout.tokens, q, k, v, o, None, None, Hq, Hkv, scale)
            _count()
        else:
            o.zero_()
        return o
    if use_kernels(q2d):
        _warn_torch_path("packed_attention", "under vmap or forward-mode differentiation" if transformed else f"head_dim {head_dim} (the kernels take multiples of 8 up to 128)")
    if transformed:
        with sdpa_kernel(SDPBackend.MATH):               # (the fused implementations have no forward-mode rule)
            return ref.packed_attention(q2d, k2d, v2d, layout.lengths, Hq, Hkv, head_dim, scale)
    return ref.packed_attention(q2d, k2d, v2d, layout.lengths, Hq, Hkv, head_dim, scale)
