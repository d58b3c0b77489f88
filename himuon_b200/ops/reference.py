"""Plain PyTorch implementations of every op in :mod:`himuon_b200.ops`.

They are the numerical oracle for the CUDA kernels and the execution path on CPU
(unit-test tier, fp32 regression run).  Rounding points of the Newton-Schulz iteration
follow the reference's fused kernel (``src/himuon/triton_kernels/ns5_smem.py:84-101``):
fp32 Frobenius norm, then every product is rounded to the compute dtype.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

NS_COEFFS = (3.4445, -4.7750, 2.0315)


def newton_schulz(G: torch.Tensor, steps: int = 5, compute_dtype: torch.dtype = torch.bfloat16,
                  eps: float = 1e-7) -> torch.Tensor:
    """Quintic Newton-Schulz orthogonalisation of the last two dims of ``G``.

    Transposes tall matrices, normalises by the Frobenius norm (+eps), runs ``steps``
    iterations of ``X <- aX + (bA + cA^2)X`` with ``A = X X^T`` and returns the result in
    ``G``'s dtype (``src/himuon/optimizers/himuon.py:232-284``).
    """
    assert G.ndim >= 2
    a, b, c = NS_COEFFS
    wide = compute_dtype in (torch.float32, torch.float64)

    def mm(x, y):  # product with fp32 accumulation, rounded to the compute dtype
        return x @ y if wide else (x.float() @ y.float()).to(compute_dtype)

    X = G.to(compute_dtype)
    tall = G.size(-2) > G.size(-1)
    if tall:
        X = X.transpose(-2, -1)
    acc = torch.float64 if compute_dtype == torch.float64 else torch.float32
    norm = X.to(acc).norm(dim=(-2, -1), keepdim=True)
    X = (X.to(acc) / (norm + eps)).to(compute_dtype)
    for _ in range(steps):
        A = mm(X, X.transpose(-2, -1))
        Bm = (c * (A.to(acc) @ A.to(acc)) + b * A.to(acc)).to(compute_dtype)
        X = (mm(Bm, X).to(acc) + a * X.to(acc)).to(compute_dtype)
    if tall:
        X = X.transpose(-2, -1)
    return X.to(G.dtype)


def tile(t: torch.Tensor, tile_size) -> tuple[torch.Tensor, tuple[int, int, int, int]]:
    """``(H, W) -> (R, C, Th, Tw)`` with zero padding at the bottom/right (``himuon.py:289-300``)."""
    th, tw = tile_size
    h, w = t.shape
    pad_h = (th - h % th) % th
    pad_w = (tw - w % tw) % tw
    if pad_h or pad_w:
        t = F.pad(t, (0, pad_w, 0, pad_h))
    R, C = t.shape[0] // th, t.shape[1] // tw
    return t.view(R, th, C, tw).permute(0, 2, 1, 3).contiguous(), (h, w, pad_h, pad_w)


def untile(tiled: torch.Tensor, info) -> torch.Tensor:
    """Inverse of :func:`tile` including the crop (``himuon.py:303-311``)."""
    h, w, pad_h, pad_w = info
    R, C, th, tw = tiled.shape
    out = tiled.permute(0, 2, 1, 3).contiguous().view(R * th, C * tw)
    return out[:h, :w] if (pad_h or pad_w) else out


def rmsnorm(x, w, eps):
    xf = x.float()
    y = (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype)
    return y * w


def rope_tables(seq_len: int, head_dim: int, theta: float, device=None) -> torch.Tensor:
    """``(seq_len, head_dim/2, 2)`` fp32 table of (cos, sin)."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    ang = torch.arange(seq_len, dtype=torch.float32, device=device)[:, None] * inv[None, :]
    return torch.stack([ang.cos(), ang.sin()], dim=-1).contiguous()


def apply_rope(x: torch.Tensor, cos_sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE on ``(B, S, H, D)`` with positions ``0..S-1``."""
    D = x.size(-1)
    S = x.size(1)
    cos = torch.cat([cos_sin[:S, :, 0], cos_sin[:S, :, 0]], -1)[None, :, None, :]
    sin = torch.cat([cos_sin[:S, :, 1], cos_sin[:S, :, 1]], -1)[None, :, None, :]
    xf = x.float()
    rot = torch.cat([-xf[..., D // 2:], xf[..., : D // 2]], -1)
    return (xf * cos + rot * sin).to(x.dtype)


def attention(q, k, v, scale=None):
    """Causal grouped-query attention on ``(B, S, H, D)`` tensors."""
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qh = q.transpose(1, 2)
    kh = k.transpose(1, 2).repeat_interleave(Hq // Hkv, dim=1)
    vh = v.transpose(1, 2).repeat_interleave(Hq // Hkv, dim=1)
    out = F.scaled_dot_product_attention(qh, kh, vh, is_causal=True, scale=scale)
    return out.transpose(1, 2).contiguous()


def swiglu(gate, up):
    return F.silu(gate) * up


def linear_cross_entropy(h, w, labels, ignore_index=-100):
    """Mean token cross-entropy of ``h @ w.T`` in fp32 (HF ``ForCausalLMLoss`` after the shift)."""
    logits = (h @ w.t()).float()
    return F.cross_entropy(logits, labels, ignore_index=ignore_index, reduction="mean")


def packed_attention(q2d, k2d, v2d, lengths, Hq: int, Hkv: int, head_dim: int, scale=None):
    """Causal attention within each of the documents of ``lengths`` that lie one after the other in ``(rows, heads*head_dim)``
    views; rows behind the last one are padding, whose output is zero."""
    parts, first = [], 0
    for n in lengths:
        if n:
            q, k, v = (t[first: first + n].reshape(1, n, -1, head_dim) for t in (q2d, k2d, v2d))
            parts.append(attention(q, k, v, scale).reshape(n, Hq * head_dim))
        first += n
    pad = q2d.shape[0] - first
    if pad or not parts:
        # (through empty slices, so that an empty batch has gradients as well)
        rest = F.pad(q2d[first:first], (0, 0, 0, pad))
        parts.append(rest if parts else rest + (k2d[first:first].sum() + v2d[first:first].sum()))
    return torch.cat(parts)


def token_log_probs(logits, ids, top_k: int = 0, ignore_index: int = -100):
    """``(log_probs, entropy, top_log_probs, top_ids)`` in fp32 (fp64 for fp64 logits): see ``ops.token_log_probs``."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    m = x.detach().amax(-1, keepdim=True)
    empty = torch.isneginf(m)
    d = x - torch.where(empty, torch.zeros_like(m), m)
    e = d.exp()
    s = torch.where(empty, torch.ones_like(m), e.sum(-1, keepdim=True))
    t = (e * torch.where(e == 0, torch.zeros_like(d), d)).sum(-1, keepdim=True)
    lp = d - s.log()
    entropy = (s.log() - t / s)[:, 0]
    counted, inside = ids != ignore_index, (ids >= 0) & (ids < x.shape[1])
    picked = lp.gather(1, torch.where(inside, ids, torch.zeros_like(ids))[:, None])
    picked = torch.where(empty, picked.detach(), picked)[:, 0]
    picked = picked.masked_fill(~inside, float("nan"))
    log_probs = torch.where(counted, picked, torch.zeros_like(picked))
    if not top_k:
        return log_probs, entropy, None, None
    top_ids = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :top_k].contiguous()
    return log_probs, entropy, lp.detach().gather(1, top_ids), top_ids


def rotary(x2d, positions, inv, factor: float, heads: int, head_dim: int, interleaved: bool):
    """Turns the first ``2 * len(inv)`` values of every head by ``positions * inv`` (angles in fp64), products in fp32 (fp64 for fp64)."""
    acc = torch.float64 if x2d.dtype == torch.float64 else torch.float32
    angles = positions.to(torch.float64)[:, None] * inv
    cos, sin = ((f(angles) * factor).to(acc)[:, None, :] for f in (torch.cos, torch.sin))
    x = x2d.to(acc).reshape(x2d.shape[0], heads, head_dim)
    r = 2 * inv.numel()
    head, rest = x[..., :r], x[..., r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : r // 2], head[..., r // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((head, rest), -1).reshape(x2d.shape).to(x2d.dtype)


def gated_mlp(x, w_gate, w_up, w_down, activation: str = "silu"):
    act = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda g: F.gelu(g, approximate="tanh"), "relu": F.relu}[activation]
    if x.dtype in (torch.float32, torch.float64):
        return (act(x @ w_gate.t()) * (x @ w_up.t())) @ w_down.t()
    x, dtype = x.float(), x.dtype
    h = act(x @ w_gate.float().t()) * (x @ w_up.float().t())
    return (h.to(dtype).float() @ w_down.float().t()).to(dtype)


def quantize_fp8(x, block_rows: int):
    """``(values, scales)``: e4m3 and a power of two for each block of ``(block_rows, 128)``: see ``ops.quantize_fp8``."""
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // 128)
    padded = F.pad(x.float(), (0, nc * 128 - cols, 0, nr * block_rows - rows)).view(nr, block_rows, nc, 128)
    size = torch.where(padded.isfinite(), padded.abs(), torch.zeros_like(padded))
    mantissa, exponent = torch.frexp(size.amax((1, 3)) if size.numel() else size.new_zeros(nr, nc))
    exponent = torch.where(mantissa == 0, torch.zeros_like(exponent), exponent - 9 + (mantissa > 0.875).int()).clamp(min=-110)
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    q = padded / scales[:, None, :, None]
    q = torch.where(q.isfinite(), q, torch.full_like(q, float("nan"))).to(torch.float8_e4m3fn)
    return q.view(nr * block_rows, nc * 128)[:rows, :cols].contiguous(), scales


def fp8_dequantize(values, scales, block_rows: int):
    rows, cols = values.shape
    return values.float() * scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return (_in_fp8(x, 1) @ _in_fp8(w, 128).t()).to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dx = (_in_fp8(dy, 1) @ _in_fp8(w, 128)).to(x.dtype) if ctx.needs_input_grad[0] else None
        dw = (_in_fp8(dy.t(), 1) @ _in_fp8(x.t(), 128).t()).to(w.dtype) if ctx.needs_input_grad[1] else None
        return dx, dw


def _in_fp8(x, block_rows):
    return fp8_dequantize(*quantize_fp8(x, block_rows), block_rows)


def fp8_linear(x2d, w):
    """``x2d @ w.T`` with operands rounded to 8 bits, and so the gradients' products: see ``ops.fp8_linear``."""
    return _Fp8LinearFn.apply(x2d, w)


def fp8_linear_any(x2d, w):
    """The same for any transform: rounding has the derivative of doing nothing, and the gradients' products round ``w`` and ``x`` alone."""
    def rounded(t, block_rows):
        t = t.float()
        return t + (_in_fp8(t.detach(), block_rows) - t.detach())

    return (rounded(x2d, 1) @ rounded(w, 128).t()).to(x2d.dtype)
