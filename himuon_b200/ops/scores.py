"""Log probabilities of given tokens, with the entropy of their distribution and the likeliest alternatives.

:func:`token_log_probs` takes logits, :func:`linear_token_log_probs` hidden states and the head's weight, whose logits it never
keeps.  Both are differentiable in the log probabilities and the entropy (policy gradients, entropy bonuses, distillation).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _ext
from . import _count, _once, _with_kernel_rows, gemm, use_kernels
from . import reference as ref

MAX_TOP_K = 32


class TokenLogProbs(NamedTuple):
    """``log_probs`` and ``entropy``: fp32, one for each row.  ``top_log_probs`` / ``top_ids``: ``(rows, top_k)``, likeliest
    first, equal ones in the order of their ids; ``None`` without ``top_k``, and not differentiable."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_log_probs: torch.Tensor | None = None
    top_ids: torch.Tensor | None = None


def _incoming(g: torch.Tensor | None):
    return None if g is None else g.to(torch.float32).contiguous()


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
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[1]):
        raise RuntimeError(f"himuon_b200.ops.token_log_probs: top_k must lie in 0..{min(MAX_TOP_K, logits.shape[1])}, got {top_k}")
    ids = _check_ids("token_log_probs", ids, logits.shape[0], logits.device)
    if logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float32):
        if logits.stride(1) != 1 or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]):
            logits = logits.contiguous()
        return TokenLogProbs(*_ext.ext().token_scores(logits, ids, int(top_k), int(ignore_index)))
    return TokenLogProbs(*ref.token_log_probs(logits, ids, top_k, ignore_index))


def _long_product(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor) -> None:
    """``out = a @ b`` for a long inner dimension and few output tiles: cut along it into batches whose fp32 results are added up.

    A GEMM's time goes by its rounds of tiles over the SMs, and the cut fills them: 777 x 128256 x 640, 12 tiles of 256 x 256
    on 74 CTA pairs, 130 us in 6 cuts against 567 whole; the fp32 results are what a cut costs."""
    (rows, inner), cols = a.shape, b.shape[1]
    pairs = rows > 128 and cols > 192
    sms = _ext.ext().num_sms()
    slots, tile = (sms // 2, 256) if pairs else (sms, 128)
    tiles = -(-rows // tile) * -(-cols // 256)
    if tiles >= 4 * slots or inner < 8192:
        gemm(a, b, out=out)
        return
    unit = tile * 256 * 2 * inner / (1.4e15 / slots)           # seconds of one tile, whole
    best, cuts = None, 1
    for s in range(1, min(16, inner // 4096) + 1):
        rounds = -(-tiles * s // slots) / s
        if s == 1 and pairs and tiles > slots // 2 and 0 < tiles % slots <= slots // 2:
            rounds = tiles / slots                             # (the GEMM cuts such a last round itself)
        cost = rounds * unit + (8.0 * s * rows * cols / 6e12 + 8e-6 if s > 1 else 0.0)
        if best is None or cost < best:
            best, cuts = cost, s
    if cuts == 1:
        gemm(a, b, out=out)
        return
    step = inner // cuts // 64 * 64
    rest = inner - cuts * step
    parts = torch.empty(cuts + (rest > 0), rows, cols, device=a.device, dtype=torch.float32)
    gemm(a.as_strided((cuts, rows, step), (step, a.stride(0), 1)), b.as_strided((cuts, step, cols), (step * b.stride(0), b.stride(0), 1)), out=parts[:cuts])
    if rest:
        gemm(a[:, cuts * step:], b[cuts * step:], out=parts[cuts])
    _ext.ext().sum_parts(parts, out)
    _count()


LAUNCH_ROWS = 8192               # of one launch: their hidden states stay in the L2 while the weight streams by
GRADIENT_VALUES = 2 ** 31        # most values of the logits' gradient alive at once (4 GiB)


def _linear_scores(h, w, ids, ignore_index, keep: bool):
    """log_probs, entropy, and with ``keep`` what the gradient needs: two numbers a row, and, where they fit, the exponentials of the
    logits in the buffer that their gradient will have, with the maxima of each 64 of them."""
    rows, vocab, e = h.shape[0], w.shape[0], _ext.ext()
    log_probs = torch.empty(rows, device=h.device, dtype=torch.float32)
    entropy = torch.empty(rows, device=h.device, dtype=torch.float32)
    stats = torch.empty(rows, 2, device=h.device, dtype=torch.float32) if keep else None
    cols = (vocab + 7) // 8 * 8
    kept = slab_max = None
    if keep and rows > 64 and rows * cols <= GRADIENT_VALUES:        # (a few rows have a kernel that keeps nothing)
        kept = torch.empty(rows, cols, device=h.device, dtype=torch.bfloat16)
        slab_max = torch.empty(rows, (vocab + 63) // 64, device=h.device, dtype=torch.float32)
    if rows:
        scratch = torch.empty(e.linear_scores_scratch(min(rows, LAUNCH_ROWS), vocab), device=h.device, dtype=torch.float32)
    for r in range(0, rows, LAUNCH_ROWS):
        if rows <= LAUNCH_ROWS:
            e.linear_scores_fwd(h, w, ids, log_probs, entropy, stats, scratch, ignore_index, kept, slab_max)
        else:
            c = slice(r, min(rows, r + LAUNCH_ROWS))
            e.linear_scores_fwd(h[c], w, ids[c], log_probs[c], entropy[c], stats[c] if keep else None, scratch, ignore_index,
                                None if kept is None else kept[c], None if kept is None else slab_max[c])
        _count(2)
    return log_probs, entropy, stats, kept, slab_max


class _LinearTokenLogProbsFn(torch.autograd.Function):
    """The backward pass multiplies the logits' gradient with both operands.  It gets it from the exponentials that the forward pass kept, in
    their place; where there are none (too many, or used up by an earlier backward pass) it makes the logits again."""

    @staticmethod
    def forward(ctx, h, w, ids, ignore_index):
        ctx.set_materialize_grads(False)
        log_probs, entropy, stats, *ctx.kept = _linear_scores(h, w, ids, ignore_index, True)
        ctx.save_for_backward(h, w, ids, entropy, stats)
        ctx.ignore_index = ignore_index
        return log_probs, entropy

    @staticmethod
    def backward(ctx, g_log_probs, g_entropy):
        _once("linear_token_log_probs")
        if g_log_probs is None and g_entropy is None:
            return None, None, None, None
        h, w, ids, entropy, stats = ctx.saved_tensors
        rows, vocab = h.shape[0], w.shape[0]
        g, ge = _incoming(g_log_probs), _incoming(g_entropy)
        (buf, slab_max), ctx.kept = ctx.kept, (None, None)
        cols = (vocab + 7) // 8 * 8
        step = rows
        if buf is None:
            step = max(256, min(LAUNCH_ROWS, GRADIENT_VALUES // cols // 256 * 256))
            buf = torch.empty(min(rows, step), cols, device=h.device, dtype=torch.bfloat16)
        dh = torch.empty(h.shape, device=h.device, dtype=h.dtype) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            # a sum over several chunks is held in fp32
            dw = (torch.zeros if rows == 0 else torch.empty)(w.shape, device=w.device, dtype=torch.bfloat16 if rows <= step else torch.float32)
        for r in range(0, rows, step):
            part, dx, to = (h, ids, entropy, stats, g, ge), buf, dh
            if rows > step:
                c = slice(r, min(rows, r + step))
                part, dx = tuple(None if t is None else t[c] for t in part), buf[: c.stop - r]
                to = None if dh is None else dh[c]
            hc, idc, ec, sc, gc, gec = part
            _ext.ext().linear_scores_dlogits(hc, w, idc, ec, sc, gc, gec, dx, slab_max, ctx.ignore_index)
            _count()
            if cols != vocab:
                dx = dx[:, :vocab]
            if to is not None:
                _long_product(dx, w, to)
            if dw is not None:
                gemm(dx, hc, trans_a=True, out=dw, aux=dw if r else None, beta=1.0 if r else 0.0)
        return dh, dw if dw is None or dw.dtype == w.dtype else dw.to(w.dtype), None, None


def linear_token_log_probs(h2d: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, ignore_index: int = -100) -> TokenLogProbs:
    """:func:`token_log_probs` of ``h2d @ w.T`` (logits in fp32) for ``(rows, hidden)`` hidden states and a ``(vocab,
    hidden)`` head, without alternatives.  bf16 CUDA tensors whose hidden size is a multiple of 8 run the sm_100a kernels.

    Where a gradient is asked for, more than 64 rows keep two bytes for each logit until the backward pass, which needs them for the
    logits' gradient anyway, as long as that is no more than 4 GiB; beyond, it makes the logits again, some thousand rows at a time."""
    if h2d.dim() != 2 or w.dim() != 2 or h2d.shape[1] != w.shape[1] or w.shape[0] == 0 or h2d.dtype != w.dtype or h2d.device != w.device:
        raise RuntimeError("himuon_b200.ops.linear_token_log_probs: (rows, hidden) and (vocab, hidden) of one type on one device expected")
    ids = _check_ids("linear_token_log_probs", ids, h2d.shape[0], h2d.device)
    if use_kernels(h2d) and h2d.shape[1] % 8 == 0 and h2d.shape[1] > 0:
        h2d, w = _with_kernel_rows(h2d), _with_kernel_rows(w)
        if torch.is_grad_enabled() and (h2d.requires_grad or w.requires_grad):
            return TokenLogProbs(*_LinearTokenLogProbsFn.apply(h2d, w, ids, int(ignore_index)))
        return TokenLogProbs(*_linear_scores(h2d, w, ids, int(ignore_index), False)[:2])
    logits = h2d @ w.t() if h2d.dtype in (torch.float32, torch.float64) else h2d.float() @ w.float().t()
    return TokenLogProbs(*ref.token_log_probs(logits, ids, 0, ignore_index))
