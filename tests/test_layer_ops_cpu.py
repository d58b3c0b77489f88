"""Rotary positions, the gated feed-forward block and 8-bit blocks off-GPU: the plain implementations against independent ones in 64 bits,
their gradients against differences, and what the operators refuse."""

import math
from fractions import Fraction

import pytest
import torch

from himuon_b200 import ops
from himuon_b200.ops import reference as ref

SCALINGS = [None, {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "ntk", "factor": 8.0},
            {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
            {"rope_type": "llama3", "factor": 32.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}]


def _freqs(rotary_dim, theta=10000.0, scaling=None):
    return ops.RotaryFrequencies(rotary_dim, theta, scaling, device="cpu")


# ------------------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("scaling", SCALINGS[:2])
def test_frequencies_are_those_of_the_rotary_table(scaling):
    f = _freqs(64, 500000.0, scaling)
    table = ref.rope_tables(2, 64, 500000.0)
    assert f.factor == 1.0
    assert torch.allclose(torch.tensor(f.frequencies).cos().float(), table[1, :, 0], atol=1e-6)
    assert torch.allclose(torch.tensor(f.frequencies).sin().float(), table[1, :, 1], atol=1e-6)


def test_scaled_frequencies():
    plain = _freqs(128, 500000.0).frequencies
    assert _freqs(128, 500000.0, SCALINGS[2]).frequencies == [f / 4 for f in plain]
    ntk = _freqs(128, 500000.0, SCALINGS[3]).frequencies
    assert ntk[0] == plain[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12)
    # llama3: more than 4 turns in the original length stay, less than one turn is divided, between them in order
    llama = _freqs(128, 500000.0, SCALINGS[5]).frequencies
    for f, g in zip(plain, llama):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            assert g == f
        elif turns <= 1:
            assert math.isclose(g, f / 32, rel_tol=1e-12)
        else:
            assert f / 32 < g < f
    # yarn: 32 turns and more stay, less than one is divided
    f = _freqs(128, 500000.0, SCALINGS[4])
    assert math.isclose(f.factor, 0.1 * math.log(4.0) + 1.0)
    for i, (a, b) in enumerate(zip(plain, f.frequencies)):
        turns = 4096 * a / (2 * math.pi)
        assert b <= a and b >= a / 4 * (1 - 1e-12)
        if turns > 34 or turns < 0.8:                              # (the ramp starts and ends at whole pairs)
            assert math.isclose(b, a if turns > 34 else a / 4, rel_tol=1e-12), i
    assert _freqs(128, 500000.0, {**SCALINGS[4], "attention_factor": 1.25}).factor == 1.25


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary_dim", [8, 4, 0])
def test_plain_rotary_against_complex_products(interleaved, rotary_dim):
    torch.manual_seed(1)
    rows, heads, hd = 6, 3, 8
    f = _freqs(rotary_dim, 10000.0, SCALINGS[4])
    x, positions = torch.randn(rows, heads * hd, dtype=torch.float64, requires_grad=True), torch.tensor([0, 5, 5, -3, 131071, 2 ** 20])
    y = ops.rotary(x, positions, f, heads, hd, interleaved=interleaved)
    want = x.detach().view(rows, heads, hd).clone()
    for i, w in enumerate(f.frequencies):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
        z = torch.complex(want[..., a].clone(), want[..., b].clone()) * torch.polar(torch.full((rows, 1), f.factor, dtype=torch.float64), positions.double()[:, None] * w)
        want[..., a], want[..., b] = z.real, z.imag
    assert torch.allclose(y, want.view(rows, -1), atol=1e-9)
    assert torch.autograd.gradcheck(lambda t: ops.rotary(t, positions, f, heads, hd, interleaved=interleaved), x)


def test_rotary_takes_a_sequence_length_and_matches_head_norm_rope():
    torch.manual_seed(2)
    B, S, heads, hd = 2, 5, 3, 16
    x = torch.randn(B * S, heads * hd)
    f = _freqs(hd)
    y = ops.rotary(x, S, f, heads, hd)
    assert torch.equal(y, ops.rotary(x, torch.arange(S).repeat(B), f, heads, hd))
    assert torch.allclose(y, ops.head_norm_rope(x, None, ref.rope_tables(S, hd, 10000.0), heads, S, hd, 1e-6), atol=1e-5)


def test_whole_turns_of_a_frequency():
    """What the kernel multiplies positions by is the frequency in 2^-64 turns, to half a unit."""
    f = _freqs(64, 10000.0, SCALINGS[2])
    two_pi = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    for w, t in zip(f.frequencies, f.turns.tolist()):
        assert abs(Fraction(w) / two_pi * 2 ** 64 - t % 2 ** 64) <= Fraction(1, 2)


def test_rotary_refusals():
    f, x = _freqs(8), torch.randn(4, 16)
    for args in ((x, torch.zeros(3, dtype=torch.int64), f, 2, 8), (x, torch.zeros(4, dtype=torch.int32), f, 2, 8), (x, torch.zeros(4, 1, dtype=torch.int64), f, 2, 8),
                 (x, 3, f, 2, 8), (x, 0, f, 2, 8), (x, 2.0, f, 2, 8), (x, 2, f, 2, 7), (x, 2, f, 4, 4), (x, 2, f, 0, 8), (x[None], 2, f, 2, 8), (x.long(), 2, f, 2, 8),
                 (x, 2, f.frequencies, 2, 8)):
        with pytest.raises(RuntimeError, match="rotary"):
            ops.rotary(*args)
    for args in ((7,), (-2,), (8.0,), (8, 1.0), (8, math.inf), (8, 1e4, {}), (8, 1e4, {"rope_type": "dynamic", "factor": 2}), (8, 1e4, {"rope_type": "linear"}),
                 (8, 1e4, {"rope_type": "linear", "factor": 0}), (8, 1e4, {"rope_type": "yarn", "factor": 2}),
                 (8, 1e4, {"rope_type": "llama3", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4, "original_max_position_embeddings": 100})):
        with pytest.raises(RuntimeError, match="RotaryFrequencies"):
            ops.RotaryFrequencies(*args, device="cpu")


# ------------------------------------------------------------------------------------------- gated feed-forward block
def _activation(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    if name == "gelu":
        return 0.5 * g * torch.erfc(-g / math.sqrt(2))
    if name == "gelu_tanh":
        return g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    return g.clamp(min=0)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_plain_gated_mlp(activation):
    torch.manual_seed(3)
    x, wg, wu, wd = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((2, 3, 5), (7, 5), (7, 5), (5, 7)))
    y = ops.gated_mlp(x, wg, wu, wd, activation=activation)
    assert torch.allclose(y, (_activation(activation, x @ wg.t()) * (x @ wu.t())) @ wd.t(), atol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: ops.gated_mlp(*a, activation=activation), (x, wg, wu, wd))
    low = [t.detach().bfloat16() for t in (x, wg, wu, wd)]
    full = ops.gated_mlp(*(t.double() for t in low), activation=activation)
    # h and y rounded to bf16: 2^-8 of each
    h = _activation(activation, low[0].double() @ low[1].double().t()) * (low[0].double() @ low[2].double().t())
    bound = 2.0 ** -8 * (full.abs() + 1.01 * h.abs() @ low[3].double().abs().t()) + 1e-4
    assert ((ops.gated_mlp(*low, activation=activation).double() - full).abs() <= bound).all()


def test_gated_mlp_of_nothing_and_refusals():
    wg, wu, wd = torch.randn(6, 4), torch.randn(6, 4), torch.randn(4, 6)
    assert ops.gated_mlp(torch.randn(0, 4), wg, wu, wd).shape == (0, 4)
    x = torch.randn(2, 4)
    for args in ((x[:, :3], wg, wu, wd), (x, wg, wu[:5], wd), (x, wg, wu, wd.t()), (x, wg[0], wu, wd), (x, wg.double(), wu, wd), (x.long(), wg, wu, wd), (x, wg, wu, wd, "swish"),
                 (x[:, :0], wg[:, :0], wu[:, :0], wd[:0])):
        with pytest.raises(RuntimeError, match="gated_mlp"):
            ops.gated_mlp(*args)


# ------------------------------------------------------------------------------------------- 8 bits
def _e4m3(v: Fraction) -> Fraction:
    """The e4m3 value nearest to v, ties to the one with an even last bit; |v| is at most 448."""
    if v == 0:
        return Fraction(0)
    e = -6
    while abs(v) >= Fraction(2) ** (e + 1):
        e += 1
    step = Fraction(2) ** (e - 3)
    return round(v / step) * step              # (round() of a Fraction takes ties to the even whole number)


def _blocks(x: torch.Tensor, block_rows: int):
    """Values that 8 bits stand for and scales, in fractions."""
    rows, cols = x.shape
    out, scales = torch.empty(rows, cols, dtype=torch.float64), torch.empty(-(-rows // block_rows), -(-cols // 128), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = x[i * block_rows: (i + 1) * block_rows, j * 128: (j + 1) * 128]
            values = [[Fraction(v) if math.isfinite(v) else None for v in r] for r in part.double().tolist()]
            top, k = max((abs(v) for r in values for v in r if v is not None), default=0), 0
            if top:
                k = -110
                while top > 448 * Fraction(2) ** k:
                    k += 1
            scales[i, j] = 2.0 ** k
            got = [[math.nan if v is None else float(_e4m3(v / Fraction(2) ** k) * Fraction(2) ** k) for v in r] for r in values]
            out[i * block_rows: i * block_rows + part.shape[0], j * 128: j * 128 + part.shape[1]] = torch.tensor(got, dtype=torch.float64)
    return out, scales


def special_values(dtype):
    """Rows that go wrong easily: zeros, a largest value at and next to 448 * 2^k, ties, tiny and huge ones, values that are not finite."""
    torch.manual_seed(5)
    x = torch.randn(150, 200) * torch.exp2(torch.randint(-20, 20, (150, 1)).float())
    x[0], x[1, 3:] = 0, 0
    x[2], x[2, 7] = torch.randint(-16, 17, (200,)) / 16.0, 448.0                  # ties of 4 bits; the largest value is 448 itself
    x[3], x[3, 9] = x[2], -448.0 * (1 + 2.0 ** -7)                                # the next value of bf16 above
    x[4] = torch.arange(200) * 2.0 ** -10                                         # around the least e4m3 steps beside 448
    x[4, 0] = 448.0
    x[5], x[6] = x[5] * 2.0 ** -120, torch.full((200,), 2.0 ** -130)              # scales at their least; subnormal values
    x[7, :] = torch.finfo(torch.bfloat16).max
    x[8, 5], x[9, 5], x[10] = math.inf, math.nan, -math.inf
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_plain_quantisation_against_fractions(dtype, block_rows):
    x = special_values(dtype)
    q = ops.quantize_fp8(x, block_rows=block_rows)
    want, scales = _blocks(x, block_rows)
    assert q.block_rows == block_rows and q.values.dtype == torch.float8_e4m3fn and torch.equal(q.scales.double(), scales)
    # (the largest numbers are rounded up to 2^128, which fp32 has only as infinity)
    assert torch.equal(q.dequantize().nan_to_num(7e37), want.float().nan_to_num(7e37))
    t = ops.quantize_fp8(x.t(), block_rows=block_rows, transpose=True)
    assert torch.equal(t.scales, q.scales) and torch.equal(t.values.view(torch.uint8), q.values.view(torch.uint8))
    assert q.dequantize(torch.bfloat16).dtype == torch.bfloat16


def test_quantisation_of_nothing():
    for shape in ((0, 5), (5, 0), (0, 0)):
        q = ops.quantize_fp8(torch.zeros(*shape), 128)
        assert q.values.shape == shape and q.scales.shape == (-(-shape[0] // 128), -(-shape[1] // 128)) and q.dequantize().shape == shape


def test_plain_products_in_8_bits():
    torch.manual_seed(7)
    x, w, dy = torch.randn(2, 9, 200), torch.randn(140, 200), torch.randn(2, 9, 140)
    x.requires_grad_(), w.requires_grad_()
    q = {n: ops.quantize_fp8(t.detach().reshape(-1, t.shape[-1]), b, transpose=tr).dequantize().double()
         for n, t, b, tr in (("x", x, 1, False), ("w", w, 128, False), ("dy", dy, 1, False), ("dyt", dy, 1, True), ("xt", x, 128, True))}
    y = ops.fp8_linear(x, w)
    y.backward(dy)
    for got, want in ((y.detach().view(18, -1), q["x"] @ q["w"].t()), (x.grad.view(18, -1), q["dy"] @ q["w"]), (w.grad, q["dyt"] @ q["xt"].t())):
        assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-4)
    a, b = ops.quantize_fp8(x.detach()[0]), ops.quantize_fp8(w.detach(), 128)
    assert torch.allclose(ops.fp8_matmul(a, b, out_dtype=torch.float32), y.detach()[0], atol=1e-4)
    assert torch.allclose(ops.fp8_linear(x.detach(), b), y.detach(), atol=1e-4)
    # under transforms rounding has the derivative of doing nothing
    got, tangent = torch.func.jvp(lambda t: ops.fp8_linear(t, w.detach()), (x.detach()[0],), (x.detach()[1],))
    assert torch.allclose(got, y.detach()[0], atol=1e-4) and torch.allclose(tangent.double(), x.detach()[1].double() @ q["w"].t(), rtol=1e-4, atol=1e-4)


def test_8_bit_refusals():
    x, w = torch.randn(4, 256), torch.randn(130, 256)
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w, 128)
    for args in ((x[0],), (x.double(),), (x.long(),), (x, 64)):
        with pytest.raises(RuntimeError, match="quantize_fp8"):
            ops.quantize_fp8(*args)
    for args in ((a, a), (a, ops.quantize_fp8(w[:, :128], 128)), (a, w), (a, ops.Fp8Blocks(b.values, b.scales[:1], 128)), (a, ops.Fp8Blocks(b.values, b.scales.double(), 128)),
                 (a, ops.Fp8Blocks(w, b.scales, 128)), (a, ops.Fp8Blocks(b.values, b.scales, 64)), (a, b, torch.float16)):
        with pytest.raises(RuntimeError, match="fp8_matmul"):
            ops.fp8_matmul(*args)
    for args in ((x, a), (x[:, :128], b), (x[:, :128], w), (x.double(), w), (x.long(), b), (x, w[0])):
        with pytest.raises(RuntimeError, match="fp8_linear"):
            ops.fp8_linear(*args)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.fp8_linear(x.clone().requires_grad_(), b)
    with torch.no_grad():
        ops.fp8_linear(x.clone().requires_grad_(), b)
    with pytest.raises(RuntimeError, match="dequantize"):
        b.dequantize(torch.float16)
    leaf = x.clone().requires_grad_()
    g = torch.autograd.grad(ops.fp8_linear(leaf, w).square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
