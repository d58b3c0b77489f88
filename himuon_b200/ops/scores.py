"""Log probabilities of given tokens, with the entropy of their distribution and the likeliest alternatives.

:func:`token_log_probs` takes logits, :func:`linear_token_log_probs` hidden states and the head's weight, whose logits never exist as
a whole; for a gradient it may keep two bytes for each.  Both are differentiable in the log probabilities and the entropy (policy
gradients, entropy bonuses, distillation); under vmap and forward-mode differentiation, for which the kernels have no rules, the
PyTorch formulation runs.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _ext
from . import _any_transformed, _warn_torch_path, _with_rows_apart, use_kernels
from . import reference as ref

MAX_TOP_K = 32


class TokenLogProbs(NamedTuple):
    """``log_probs`` and ``entropy``: fp32, one for each row.  ``top_log_probs`` / ``top_ids``: ``(rows, top_k)``, likeliest
    first, equal ones in the order of their ids; ``None`` without ``top_k``, and not differentiable."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor | None = None
    top_ids: torch.Tensor | None = None


def _check_ids(op: str, ids: torch.Tensor, rows: int, device) -> torch.Tensor:
    if ids.dtype != torch.int64 or ids.numel() != rows or ids.dim() != 1 or ids.device != device:
        raise RuntimeError(f"himuon_b200.ops.{op}: ids must be int64, one for each of the {rows} rows, on {device}")
    return ids.contiguous()


def token_log_probs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0, ignore_index: int = -100) -> TokenLogProbs:
    """Scores of ``ids`` under the rows of ``(rows, vocab)`` logits.

    A row whose id is ``ignore_index`` has log probability 0 and passes no gradient of it on; its entropy and alternatives
    are those of the row.  An id outside the vocabulary has log probability NaN and no gradient.  Logits of ``-inf`` are masked tokens; a row of
    nothing else has log probability ``-inf`` and entropy 0.  At most 32 alternatives.  bf16 and fp32 CUDA logits run the
    sm_100a kernels.
    """
    if logits.dim() != 2 or logits.shape[1] == 0 or not logits.is_floating_point():
        raise RuntimeError("himuon_b200.ops.token_log_probs: logits must be a (rows, vocab) matrix of floating point")
    rows, vocab = logits.shape
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise RuntimeError(f"himuon_b200.ops.token_log_probs: top_k must lie in 0..{min(MAX_TOP_K, vocab)}, got {top_k}")
    ids = _check_ids("token_log_probs", ids, rows, logits.device)
    transformed = _any_transformed(logits, ids)
    if logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float32) and not transformed:
        ld, inner = logits.stride()
        if inner != 1 or (rows > 1 and ld < vocab):
            logits = logits.clone(memory_format=torch.contiguous_format)      # (one column is contiguous at any stride)
        return TokenLogProbs(*_ext.ext().token_scores(logits, ids, int(top_k), int(ignore_index)))
    if logits.is_cuda and transformed:
        _warn_torch_path("token_log_probs", "under vmap or forward-mode differentiation")
    return TokenLogProbs(*ref.token_log_probs(logits, ids, top_k, ignore_index))


LAUNCH_ROWS = 8192               # of one launch: their hidden states stay in the L2 while the weight streams by
GRADIENT_VALUES = 2 ** 31        # most values of the logits' gradient alive at once (4 GiB)


def linear_token_log_probs(h2d: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, ignore_index: int = -100) -> TokenLogProbs:
    """:func:`token_log_probs` of ``h2d @ w.T`` (logits in fp32) for ``(rows, hidden)`` hidden states and a ``(vocab,
    hidden)`` head, without alternatives.  bf16 CUDA tensors whose hidden size is a multiple of 8 run the sm_100a kernels.

    Where a gradient is asked for, more than 64 rows keep two bytes for each logit until the backward pass, which needs them for the
    logits' gradient anyway, as long as that is no more than 4 GiB; a checkpoint around the call drops them.  Beyond, the backward pass makes the logits again, some thousand rows at a time.  A backward pass that
    a graph captures leaves what was kept as it is and takes as much again, because it may be replayed more than once."""
    if h2d.dim() != 2 or w.dim() != 2 or h2d.shape[1] != w.shape[1] or w.shape[0] == 0 or h2d.dtype != w.dtype or h2d.device != w.device:
        raise RuntimeError("himuon_b200.ops.linear_token_log_probs: (rows, hidden) and (vocab, hidden) of one type on one device expected")
    ids = _check_ids("linear_token_log_probs", ids, h2d.shape[0], h2d.device)
    transformed = _any_transformed(h2d, w, ids)
    if use_kernels(h2d) and h2d.shape[1] % 8 == 0 and h2d.shape[1] > 0 and not transformed:
        h2d, w = _with_rows_apart(h2d), _with_rows_apart(w)
        return TokenLogProbs(*_ext.ext().linear_scores(h2d, w, ids, int(ignore_index), LAUNCH_ROWS, GRADIENT_VALUES))
    if use_kernels(h2d):
        _warn_torch_path("linear_token_log_probs", "under vmap or forward-mode differentiation" if transformed else
                         f"hidden size {h2d.shape[1]} (the kernels take multiples of 8)")
    logits = h2d @ w.t() if h2d.dtype in (torch.float32, torch.float64) else h2d.float() @ w.float().t()
    return TokenLogProbs(*ref.token_log_probs(logits, ids, 0, ignore_index))
