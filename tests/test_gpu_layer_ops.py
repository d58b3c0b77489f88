"""Rotary positions, the gated feed-forward block and 8-bit products on the GPU against 64-bit formulas (GPU tier).

The bounds are element by element and follow from the kernels' roundings: u = 2^-8 is what rounding to bf16 changes a value by at most
(relative), and each product of rounded factors passes that on through the absolute values of the terms of its sum.
"""

import math
from fractions import Fraction

import pytest
import torch

from test_layer_ops_cpu import SCALINGS, special_values

pytestmark = pytest.mark.gpu

U = 2.0 ** -8          # bf16
TURN = 2.0 ** -20      # fp32 sines and two products: 1.5 units of 2^-23 of a sine, pi * 2^-24 of an angle, three roundings of 2^-24


def _sums(n):
    """fp32 sums of n products, cut off 16 at a time, relative to the terms' absolute values; and what is done to them in fp32."""
    return 2.0 ** -23 * (n / 16 + 16)


def _ops():
    from himuon_b200 import ops

    return ops


def _clean():
    from himuon_b200._ext import ext

    torch.cuda.synchronize()
    assert ext().status(True) == 0, "a bounded device wait ran out (status word set)"


def _within(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: {(over > 0).sum().item()} of {over.numel()} outside, worst by {over.max().item():.3g}"


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------------- rotary positions
def _rotary64(x, cos, sin, heads, r, interleaved):
    """The rotation by given cosines and sines, and the absolute values of each result's terms."""
    x = x.detach().double().view(x.shape[0], heads, -1)
    out, size = x.clone(), torch.zeros_like(x)
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        c, s = cos[:, None, i], sin[:, None, i]
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return out.flatten(1), size.flatten(1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,hd,r", [(3, 128, 128), (1, 64, 32), (5, 64, 16), (2, 48, 24), (7, 80, 80), (4, 36, 20), (1, 2, 2), (2, 24, 0), (3, 9, 4), (9, 256, 192)])
def test_rotary(heads, hd, r, interleaved, dtype):
    ops = _ops()
    torch.manual_seed(hd + r)
    for rows, scaling in ((1, SCALINGS[0]), (37, SCALINGS[4]), (300, SCALINGS[5])):
        f = ops.RotaryFrequencies(r, 500000.0, scaling)
        x, dy = (torch.randn(rows, heads * hd, device="cuda").to(dtype) for _ in range(2))
        x.requires_grad_()
        positions = torch.randint(0, 131072, (rows,), device="cuda")
        positions[0] = 0
        before = ops.launch_count()
        y = ops.rotary(x, positions, f, heads, hd, interleaved=interleaved)
        dx, = torch.autograd.grad(y, x, dy)
        assert ops.launch_count() == before + 2 and y.dtype == dtype
        angles = positions.double()[:, None] * torch.tensor(f.frequencies, dtype=torch.float64, device="cuda")
        cos, sin = angles.cos() * f.factor, angles.sin() * f.factor
        for got, t, sign, what in ((y, x, 1.0, "y"), (dx, dy, -1.0, "dx")):
            want, size = _rotary64(t, cos, sign * sin, heads, r, interleaved)
            rounding = (U if dtype == torch.bfloat16 else 2.0 ** -24) * want.abs()
            _within(got, want, torch.where(size > 0, rounding + f.factor * TURN * (1 + U) * size, 0.0), what)
    _clean()


def test_rotary_of_far_positions():
    """Positions whose angles fp32, and fp64 as well, would have lost: against fractions of a turn."""
    ops = _ops()
    f = ops.RotaryFrequencies(16, 10000.0)
    positions = [0, -1, 131071, 2 ** 31 + 5, -(2 ** 33) - 7, 2 ** 40 + 1, 2 ** 44 + 3]
    two_pi = 2 * Fraction(314159265358979323846264338327950288419716939937510, 10 ** 50)
    angles = [[2 * math.pi * float(p * Fraction(w) / two_pi % 1) for w in f.frequencies] for p in positions]
    angles = torch.tensor(angles, dtype=torch.float64, device="cuda")
    x = torch.randn(len(positions), 16, device="cuda")
    y = ops.rotary(x, torch.tensor(positions, device="cuda"), f, 1, 16)
    want, size = _rotary64(x, angles.cos(), angles.sin(), 1, 16, False)
    # a frequency is off by 2^-65 of a turn a position: 2^44 * 2^-65 * 2 pi = 1.5 * 2^-19
    _within(y, want, (TURN + 2.0 ** -18) * size, "y")


def test_rotary_forms_of_positions_and_rows():
    """A sequence length is its positions; column slices, rows off the 16-byte grid, expanded and transposed ones are what their copies are."""
    ops = _ops()
    torch.manual_seed(3)
    f, heads, hd, S = ops.RotaryFrequencies(64, 10000.0), 3, 64, 50
    x = torch.randn(4 * S, heads * hd + 3, device="cuda").bfloat16()
    at = torch.arange(S, device="cuda").repeat(4)
    for t in (x[:, :-3], x[:, 3:], x[:, 1:-2], x[:1, 3:].expand(4 * S, heads * hd), x[:, 3:].contiguous().t().contiguous().t()):
        whole = t.contiguous()
        want = ops.rotary(whole, at, f, heads, hd)
        assert torch.equal(ops.rotary(t, S, f, heads, hd), want)
        assert torch.equal(ops.rotary(t, torch.stack([at, at + 1], 1)[:, 0], f, heads, hd), want)
        a, b = t.detach().requires_grad_(), whole.detach().requires_grad_()
        g = torch.randn(heads * hd, device="cuda").bfloat16().expand(4 * S, heads * hd)
        assert torch.equal(torch.autograd.grad(ops.rotary(a, S, f, heads, hd), a, g)[0], torch.autograd.grad(ops.rotary(b, S, f, heads, hd), b, g.contiguous())[0])
    table = _table(S, hd)
    near = ops.head_norm_rope(x[:, 3:].contiguous(), None, table, heads, S, hd, 1e-6)
    assert (near.float() - ops.rotary(x[:, 3:].contiguous(), S, f, heads, hd).float()).abs().max() <= 2 * U * 2 * x.float().abs().max()
    assert ops.rotary(x[:0, 3:], S, f, heads, hd).shape == (0, heads * hd)
    _clean()


def _table(S, hd):
    from himuon_b200.ops import reference as ref

    return ref.rope_tables(S, hd, 10000.0, device="cuda")


def test_rotary_keeps_pairs_apart_and_passes_bits_through():
    ops = _ops()
    torch.manual_seed(5)
    f = ops.RotaryFrequencies(32, 10000.0)
    x = torch.randn(9, 2 * 64, device="cuda").bfloat16()
    bad = x.clone()
    bad[4, 3], bad[5, 40], bad[6, 64 + 20] = math.nan, math.inf, -math.inf
    for interleaved in (False, True):
        a, b = (ops.rotary(t, 9, f, 2, 64, interleaved=interleaved) for t in (x, bad))
        assert torch.equal(a.view(9, 2, 64)[..., 32:], x.view(9, 2, 64)[..., 32:]) and b[5, 40] == math.inf
        touched = (a != b).nonzero().tolist()
        pairs = {(4, 2 if interleaved else 3), (4, 3 if interleaved else 19), (5, 40), (6, 64 + (20 if interleaved else 4)), (6, 64 + (21 if interleaved else 20))}
        assert {tuple(t) for t in touched} == pairs
    _clean()


def test_rotary_is_differentiable_again():
    ops = _ops()
    f = ops.RotaryFrequencies(8, 10000.0)
    x = torch.randn(3, 8, device="cuda", requires_grad=True)
    y = ops.rotary(x, 3, f, 1, 8)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    assert torch.allclose(g, 2 * x, atol=1e-4) and torch.allclose(h, torch.full_like(h, 2.0), atol=1e-4)
    _clean()


# ------------------------------------------------------------------------------------------- gated feed-forward block
def _activation64(name, g):
    """The activation and its derivative."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (g + 0.044715 * g ** 3))
        return g * s, s + g * s * (1 - s) * 2 * c * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).double()


def _gated64(x, wg, wu, wd, activation, dy=None):
    """Results and bounds.  |act'| is at most 1.13 and |act''| at most 1.1; fp32 exponentials and quotients are good to 2^-19."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    T, H, I = x.shape[0], x.shape[1], wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (_sums(H) * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a, d = _activation64(activation, g)
    h = a * u
    ea = 1.13 * eg + 2.0 ** -19 * (a.abs() + 1e-3)
    eh = a.abs() * eu + ea * u.abs() + ea * eu
    eh = eh + U * (h.abs() + eh)
    y = h @ wd.t()
    ey = eh @ wd.abs().t() + _sums(I) * (h.abs() + eh) @ wd.abs().t()
    out = {"y": (y, ey + U * (y.abs() + ey))}
    if dy is None:
        return out
    dy = dy.detach().double()
    dh = dy @ wd
    edh = _sums(H) * (dy.abs() @ wd.abs())
    # kept g and u: 2^-15 of each
    eg, eu = eg + 2.0 ** -15 * (g.abs() + eg), eu + 2.0 ** -15 * (u.abs() + eu)
    ea, ed = 1.13 * eg + 2.0 ** -19 * (a.abs() + 1e-3), 1.1 * eg + 2.0 ** -19 * (d.abs() + 1e-3)
    if activation == "relu":
        ed = torch.where(g.abs() <= eg, 1.0, 0.0)                      # (0 or 1, by the sign)
    dg, du = dh * u * d, dh * a

    def product(*terms):                                               # of (value, error) factors
        value = math.prod(v.abs() for v, _ in terms[1:]) * terms[0][0].abs()
        return math.prod(v.abs() + e for v, e in terms[1:]) * (terms[0][0].abs() + terms[0][1]) - value

    edg, edu = product((dh, edh), (u, eu), (d, ed)), product((dh, edh), (a, ea))
    edg, edu = edg + U * (dg.abs() + edg), edu + U * (du.abs() + edu)

    def put(name, value, error, size, n):
        error = error + _sums(n) * size
        out[name] = (value, error + U * (value.abs() + error))

    put("dx", dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs(), (dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs(), 2 * I)
    put("dwg", dg.t() @ x, edg.t() @ x.abs(), (dg.abs() + edg).t() @ x.abs(), T)
    put("dwu", du.t() @ x, edu.t() @ x.abs(), (du.abs() + edu).t() @ x.abs(), T)
    put("dwd", dy.t() @ h, dy.abs().t() @ eh, dy.abs().t() @ (h.abs() + eh), T)
    return out


def _block(T, H, I, seed=0, spread=1.5):
    torch.manual_seed(1000 * T + H + I + seed)
    x, dy = (torch.randn(T, H, device="cuda").bfloat16() for _ in range(2))
    wg, wu = ((torch.randn(I, H, device="cuda") * spread / math.sqrt(H)).bfloat16() for _ in range(2))
    return x, wg, wu, (torch.randn(H, I, device="cuda") / math.sqrt(I)).bfloat16(), dy


GATED = ("y", "dx", "dwg", "dwu", "dwd")


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("T,H,I", [(1, 8, 8), (3, 40, 24), (8, 128, 352), (17, 200, 136), (33, 64, 1000), (64, 640, 264), (65, 640, 264), (129, 72, 128), (300, 264, 520), (777, 640, 1728),
                                   (5, 264, 4104), (24, 320, 2056), (40, 72, 4096), (64, 2048, 8), (200, 264, 5648), (384, 8, 264),
                                   (385, 264, 520), (390, 8, 8), (400, 72, 128), (513, 640, 264), (65, 4096, 2056), (129, 2048, 2056), (200, 520, 5648),
                                   (100, 4104, 1000), (256, 1000, 2000), (70, 320, 19008), (48, 2056, 8200)])
def test_gated_mlp(T, H, I, activation):
    ops = _ops()
    x, wg, wu, wd, dy = _block(T, H, I)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    before = ops.launch_count()
    y = ops.gated_mlp(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, dy)
    assert ops.launch_count() >= before + 6
    _clean()
    want = _gated64(*leaves, activation, dy)
    for name, got in zip(GATED, (y, *grads)):
        _within(got, *want[name], name)
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(*leaves, activation=activation), y)           # (whether a gradient is asked for or not)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gated_mlp_of_large_gates(activation):
    """Gates of hundreds, where sigmoids are 0 and 1 and exponentials would run over, and of 1e12, where their cubes would."""
    ops = _ops()
    for T, spread in ((20, 120.0), (400, 120.0), (20, 1e12), (400, 1e12)):
        x, wg, wu, wd, dy = _block(T, 256, 384, spread=120.0)
        wg = (wg.float() * (spread / 120.0)).bfloat16()
        leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
        y = ops.gated_mlp(*leaves, activation=activation)
        grads = torch.autograd.grad(y, leaves, dy)
        want = _gated64(*leaves, activation, dy)
        for name, got in zip(GATED, (y, *grads)):
            _within(got, *want[name], name)
    _clean()


def test_gated_mlp_gradient_against_differences():
    """The kernels' gradients along a direction against a central difference of the 64-bit formula."""
    ops = _ops()
    for T in (30, 150, 400):
        x, wg, wu, wd, dy = _block(T, 128, 352)
        leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
        grads = torch.autograd.grad(ops.gated_mlp(*leaves), leaves, dy)
        want = _gated64(*leaves, "silu", dy)
        base = [t.detach().double() for t in leaves]
        for i, name in enumerate(GATED[1:]):
            d = torch.randn_like(base[i])
            f = [(_gated64(*(b + s * 1e-4 * d if j == i else b for j, b in enumerate(base)), "silu")["y"][0] * dy.double()).sum().item() for s in (1, -1)]
            slope = (f[0] - f[1]) / 2e-4
            assert abs((grads[i].double() * d).sum().item() - slope) <= (want[name][1] * d.abs()).sum().item() + 1e-5 * abs(slope)


def test_gated_mlp_of_slices_shapes_and_some_gradients():
    """Halves of one weight, rows off the 16-byte grid, expanded gradients, leading dimensions; each gradient alone has the same bits."""
    ops = _ops()
    for T in (24, 150, 400):
        x, wg, wu, wd, dy = _block(T, 128, 200)
        leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
        y = ops.gated_mlp(*leaves)
        grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert _same(torch.autograd.grad(y, leaves, dy), grads)
        both = torch.cat([wg, wu]).detach().requires_grad_()
        odd = torch.zeros(T, 129, device="cuda").bfloat16()
        odd[:, 1:] = x.detach()
        turned = wd.detach().t().contiguous().t()
        z = ops.gated_mlp(odd[:, 1:], both[:200], both[200:], turned)
        assert torch.equal(z, y)
        assert torch.equal(torch.autograd.grad(z, both, dy)[0], torch.cat(grads[1:3]))
        assert torch.equal(ops.gated_mlp(x.view(2, T // 2, 128), wg, wu, wd), y.view(2, T // 2, 128))
        assert torch.equal(ops.gated_mlp(x[0], wg, wu, wd), ops.gated_mlp(x[:1], wg, wu, wd)[0])
        for i in range(4):
            some = [t if j == i else t.detach() for j, t in enumerate(leaves)]
            assert torch.equal(torch.autograd.grad(ops.gated_mlp(*some), leaves[i], dy)[0], grads[i])
        one = torch.ones(128, device="cuda").bfloat16().expand(T, 128)
        y = ops.gated_mlp(*leaves)
        assert _same(torch.autograd.grad(y, leaves, one, retain_graph=True), torch.autograd.grad(y, leaves, one.contiguous()))
        same = x.detach()[:1].expand(T, 128)
        assert torch.equal(ops.gated_mlp(same, wg, wu, wd), ops.gated_mlp(same.contiguous(), wg, wu, wd))
    empty = x.detach()[:0].requires_grad_()
    y = ops.gated_mlp(empty, wg, wu, wd)
    assert y.shape == (0, 128) and not any(g.any() for g in torch.autograd.grad(y.sum(), [empty, wg, wu, wd]))
    _clean()


def test_gated_mlp_rows_do_not_depend_on_one_another():
    """Up to 32 rows a row has the same bits however many come with it, so it has from 33 to 64, and by tiles; NaN stays in its row and in the weights' gradients."""
    ops = _ops()
    for rows, some, H, I in ((32, (1, 7, 8, 9, 16, 30), 640, 1728), (64, (33, 50), 640, 1728), (128, (101, 120), 1360, 3200), (256, (129, 200), 1360, 3200), (400, (385, 390), 640, 1728)):
        x, wg, wu, wd, dy = _block(rows, H, I)
        whole = ops.gated_mlp(x, wg, wu, wd)
        for n in some:
            assert torch.equal(ops.gated_mlp(x[:n], wg, wu, wd), whole[:n])
    for n in (60, 120, 200, 400):
        x, wg, wu, wd, dy = _block(n, *((640, 1728) if n in (60, 400) else (1360, 3200)))
        got = []
        for t in (x, x.clone()):
            if got:
                t[3], t[5, 7] = math.nan, math.inf
            t = t.detach().requires_grad_()
            y = ops.gated_mlp(t, wg, wu, wd)
            got.append((y.detach(), torch.autograd.grad(y, t, dy)[0]))
        others = torch.ones(n, dtype=torch.bool, device="cuda")
        others[3] = others[5] = False
        for a, b in zip(*got):
            assert torch.equal(a[others], b[others]) and b[3].isnan().all() and not b[5].isfinite().all()
    _clean()


# ------------------------------------------------------------------------------------------- 8 bits
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantisation_has_the_bits_of_the_plain_one(dtype, block_rows):
    ops = _ops()
    x = special_values(dtype)
    big = torch.randn(700, 1003) * torch.exp2(torch.randint(-30, 30, (700, 1)).float())
    for t in (x, x[:1], x[:, :1], x[:128, :128], x[3:130, 1:], big.to(dtype)):
        on = t.cuda()
        for transpose in (False, True):
            for form in (on, torch.cat([on, on], 1)[:, t.shape[1]:], on.t().contiguous().t()):
                got, want = (ops.quantize_fp8(f, block_rows=block_rows, transpose=transpose) for f in (form, t))
                assert torch.equal(got.scales.cpu(), want.scales)
                a, b = got.values.cpu(), want.values
                assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.float().nan_to_num(), b.float().nan_to_num())
        full = got.dequantize().cpu()
        assert torch.equal(full.nan_to_num(), want.dequantize().nan_to_num())
        assert torch.equal(got.dequantize(torch.bfloat16).cpu().nan_to_num(), want.dequantize(torch.bfloat16).nan_to_num())
        assert torch.equal(ops.Fp8Blocks(want.values.cuda(), want.scales.cuda(), block_rows).dequantize().cpu().nan_to_num(), full.nan_to_num())
    for shape in ((0, 5), (5, 0)):
        q = ops.quantize_fp8(torch.zeros(*shape, device="cuda"), block_rows)
        assert q.values.shape == shape and q.dequantize().shape == shape
    _clean()


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 128, 128), (5, 40, 144), (8, 352, 128), (16, 130, 512), (31, 640, 1000), (64, 200, 2560), (65, 128, 640), (3, 20, 77), (129, 8, 8),
                                   (130, 1000, 1729), (300, 257, 256), (777, 1728, 640), (513, 300, 4096),
                                   (70, 520, 9728), (6400, 700, 4096), (200, 12, 5000), (8, 200, 9000), (20, 301, 5000), (32, 4000, 8192)])
def test_fp8_matmul(M, N, K):
    """Powers of two and any other fp32 scales, different from block to block, blocks of either kind in a, every row length."""
    ops = _ops()
    torch.manual_seed(M + N + K)
    for a_block, dtype, powers in ((1, torch.float32, False), (128, torch.bfloat16, False), (1, torch.bfloat16, True), (128, torch.float32, True)):
        a = ops.quantize_fp8(torch.randn(M, K, device="cuda"), a_block)
        b = ops.quantize_fp8(torch.randn(N, K, device="cuda"), 128)
        sa, sb = (torch.exp2(torch.randint(-9, 9, s.shape, device="cuda").float()) if powers else s * (0.5 + torch.rand_like(s)) for s in (a.scales, b.scales))
        a, b = ops.Fp8Blocks(a.values, sa, a_block, powers), ops.Fp8Blocks(b.values, sb.t().contiguous().t(), 128, powers)
        before = ops.launch_count()
        c = ops.fp8_matmul(a, b, out_dtype=dtype)
        assert ops.launch_count() == before + 1 and c.dtype == dtype and c.is_contiguous()
        va, vb = (_values64(m) for m in (a, b))
        want, size = va @ vb.t(), va.abs() @ vb.abs().t()
        bound = _sums(K) * size                                        # (and two roundings of a scale)
        _within(c, want, bound + (U if dtype == torch.bfloat16 else 2.0 ** -24) * (want.abs() + bound), "c")
        again = ops.Fp8Blocks(a.values.contiguous(), a.scales.contiguous(), a_block, powers), ops.Fp8Blocks(b.values.t().contiguous().t(), b.scales.contiguous(), 128, powers)
        assert torch.equal(ops.fp8_matmul(*again, out_dtype=dtype), c)
    _clean()


def _values64(m):
    rows, cols = m.values.shape
    return m.values.double() * m.scales.double().repeat_interleave(m.block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def test_fp8_matmul_of_nothing_and_of_nan():
    ops = _ops()
    q = lambda r, c, b: ops.quantize_fp8(torch.zeros(r, c, device="cuda"), b)  # noqa: E731
    assert ops.fp8_matmul(q(0, 64, 1), q(8, 64, 128)).shape == (0, 8) and ops.fp8_matmul(q(4, 64, 1), q(0, 64, 128)).shape == (4, 0)
    assert not ops.fp8_matmul(q(4, 0, 1), q(8, 0, 128)).any()
    for rows in (9, 200):
        x, w = torch.randn(rows, 256, device="cuda"), torch.randn(300, 256, device="cuda")
        clean = ops.fp8_matmul(ops.quantize_fp8(x), ops.quantize_fp8(w, 128))
        x[2, 5], x[3, 130] = math.nan, math.inf
        got = ops.fp8_matmul(ops.quantize_fp8(x), ops.quantize_fp8(w, 128))
        others = torch.ones(rows, dtype=torch.bool, device="cuda")
        others[2] = others[3] = False
        assert got[2:4].isnan().all() and torch.equal(got[others], clean[others])
    _clean()


@pytest.mark.parametrize("T,K,N", [(1, 128, 352), (30, 640, 200), (64, 72, 136), (100, 264, 128), (333, 640, 1728), (1025, 256, 77)])
def test_fp8_linear(T, K, N):
    ops = _ops()
    torch.manual_seed(T + K + N)
    x, w, dy = torch.randn(T, K, device="cuda").bfloat16(), torch.randn(N, K, device="cuda").bfloat16(), torch.randn(T, N, device="cuda").bfloat16()
    x.requires_grad_(), w.requires_grad_()
    before = ops.launch_count()
    y = ops.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert ops.launch_count() == before + 6
    _clean()
    q = {n: _values64(ops.quantize_fp8(t.detach(), b, transpose=tr)) for n, t, b, tr in
         (("x", x, 1, False), ("w", w, 128, False), ("dy", dy, 1, False), ("dyt", dy, 1, True), ("xt", x, 128, True))}
    for what, got, a, b in (("y", y, q["x"], q["w"].t()), ("dx", dx, q["dy"], q["w"]), ("dw", dw, q["dyt"], q["xt"].t())):
        want = a @ b
        bound = _sums(a.shape[1]) * (a.abs() @ b.abs())
        _within(got, want, bound + U * (want.abs() + bound), what)
    # rounding to 8 bits: at most 2^-4 of a value or 2^-10 of its block's scale (2^-18 of its largest value, 2^-17 at most)
    for name, t in (("x", x), ("w", w), ("dy", dy)):
        assert ((q[name] - t.double()).abs() <= 2.0 ** -4 * t.double().abs() + 2.0 ** -17 * t.double().abs().max()).all()
    for leaf, want in ((x, dx), (w, dw)):
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], want)
        other = [t if t is leaf else t.detach() for t in (x, w)]
        assert torch.equal(torch.autograd.grad(ops.fp8_linear(*other), leaf, dy)[0], want)
    with torch.no_grad():
        kept = ops.quantize_fp8(w, 128)
        assert torch.equal(ops.fp8_linear(x, w), y) and torch.equal(ops.fp8_linear(x, kept), y)
        assert torch.equal(ops.fp8_linear(x.view(1, T, K), kept), y.view(1, T, N))
        assert torch.equal(ops.fp8_linear(torch.cat([x, x], 1)[:, K:], w.t().contiguous().t()), y)
        if T <= 64:
            assert torch.equal(ops.fp8_linear(x[:T // 2], kept), y[:T // 2])
    empty = torch.zeros(0, K, device="cuda").bfloat16().requires_grad_()
    g = torch.autograd.grad(ops.fp8_linear(empty, w).sum(), (empty, w))
    assert g[0].shape == (0, K) and g[1].shape == (N, K) and not g[1].any()


# ------------------------------------------------------------------------------------------- all of them
def _calls(dtype=torch.bfloat16):
    """Each operator as a function of its first operand."""
    ops = _ops()
    torch.manual_seed(57)
    w = [(torch.randn(*s, device="cuda") * 0.2).to(dtype) for s in ((40, 64), (40, 64), (64, 40))]
    f = ops.RotaryFrequencies(16, 10000.0, SCALINGS[4])
    at = torch.randint(0, 10000, (14,), device="cuda")
    fns = {"rotary": lambda t: ops.rotary(t, at, f, 2, 32, interleaved=True), "gated_mlp": lambda t: ops.gated_mlp(t, *w), "fp8_linear": lambda t: ops.fp8_linear(t, w[0])}
    return fns, torch.randn(14, 64, device="cuda").to(dtype), torch.randn(14, 64, device="cuda").to(dtype)


NAMES = ["rotary", "gated_mlp", "fp8_linear"]


@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
@pytest.mark.parametrize("name", NAMES)
def test_layer_operators_under_transforms(name):
    """vmap returns what calls one by one return, forward-mode tangents are the reverse mode's gradients."""
    fns, x, d = _calls()
    fn = fns[name]
    got = torch.vmap(fn)(torch.stack([x, d]))
    for i, a in enumerate((x, d)):
        # bf16 roundings of results and of what they are made of, values of up to 8
        assert (fn(a).double() - got[i].double()).abs().max() <= 3 * U * 8
    y, tangent = torch.func.jvp(fn, (x,), (d,))
    leaf, g = x.clone().requires_grad_(), torch.randn_like(y)
    grad, = torch.autograd.grad(fn(leaf), leaf, g)
    a, b = (tangent.double() * g.double()).sum(), (grad.double() * d.double()).sum()
    # sums over a thousand values, each off by bf16 roundings (of 8 bits in fp8_linear, whose tangent does not round g)
    assert (a - b).abs() <= (0.1 if name == "fp8_linear" else 0.02) * tangent.double().norm() * g.double().norm()
    _clean()


def test_layer_operators_on_streams_and_in_graphs():
    """Another stream, two graphs in turn, gradients captured, and new inputs at each replay."""
    torch.manual_seed(61)
    for rows in (14, 140, 400):
        fns, _, _ = _calls()
        at = torch.randint(0, 10000, (rows,), device="cuda")
        ops, f = _ops(), _ops().RotaryFrequencies(32, 10000.0)
        fns["rotary"] = lambda t: ops.rotary(t, at, f, 2, 32)
        for name, fn in fns.items():
            xs = [torch.randn(rows, 64, device="cuda").bfloat16() for _ in range(4)]

            def step(t):
                leaf = t.detach().requires_grad_()
                y = fn(leaf)
                return y.detach(), torch.autograd.grad(y, leaf, torch.ones_like(y))[0]

            want = [step(t) for t in xs]
            torch.cuda.synchronize()
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                got = [step(t) for t in xs]
            side.synchronize()
            assert all(_same(a, b) for a, b in zip(got, want)), name
            inputs, graphs, outs = [torch.zeros_like(xs[0]) for _ in range(2)], [], []
            for t in inputs:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs.append(step(t))
                graphs.append(graph)
            for i in range(0, 4, 2):
                for j in range(2):
                    inputs[j].copy_(xs[i + j])
                for j in (1, 0):
                    graphs[j].replay()
                assert all(_same(outs[j], want[i + j]) for j in range(2)), name
    _clean()


def test_layer_operators_repeat_their_bits_and_run_under_a_checkpoint():
    from torch.utils.checkpoint import checkpoint

    ops = _ops()
    x, wg, wu, wd, dy = _block(700, 512, 1400)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    f, seen = ops.RotaryFrequencies(128, 10000.0), None

    def layer(x, wg, wu, wd):
        return ops.fp8_linear(ops.gated_mlp(ops.rotary(x, 700, f, 4, 128), wg, wu, wd), wd.t())

    for i in range(4):
        y = layer(*leaves) if i % 2 else checkpoint(layer, *leaves, use_reentrant=False)
        got = (y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y)))
        assert seen is None or _same(seen, got)
        seen = got
    _clean()


def test_gradients_that_are_not_differentiable_again():
    fns, x, _ = _calls()
    for name in ("gated_mlp", "fp8_linear"):
        leaf = x.clone().requires_grad_()
        y = fns[name](leaf)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)
        torch.autograd.grad(y.sum(), leaf)


def test_layer_operators_refusals_on_the_gpu():
    from himuon_b200._ext import ext

    ops, e = _ops(), ext()
    x, wg, wu, wd, _ = _block(4, 64, 40)
    f = ops.RotaryFrequencies(8, device="cpu")
    with pytest.raises(RuntimeError, match="frequencies are on"):
        ops.rotary(x, 4, f, 2, 32)
    with pytest.raises(RuntimeError, match="positions must be int64"):
        ops.rotary(x, torch.zeros(4, dtype=torch.int64), ops.RotaryFrequencies(8), 2, 32)
    with pytest.raises(RuntimeError, match="one type on one device"):
        ops.gated_mlp(x, wg.cpu(), wu, wd)
    with pytest.raises(RuntimeError, match="w_up must be"):
        e.gated_mlp(x, wg, wu[:32], wd, 0)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        e.gated_mlp(x[:, :4], wg[:, :4], wu[:, :4], wd[:4], 0)
    q = ops.quantize_fp8(x)
    with pytest.raises(RuntimeError, match="one for each block"):
        e.fp8_matmul(q.values, q.scales[:1], 1, False, q.values, q.scales, 128, False, False)
    with pytest.raises(RuntimeError, match="scales must be"):
        ops.fp8_matmul(q, ops.Fp8Blocks(q.values, q.scales.cpu(), 128))
    with pytest.raises(RuntimeError, match="one device"):
        ops.fp8_linear(x, wg.cpu())
    ops._WARNED.discard(("gated_mlp", "sizes of 63 and 40 (the kernels take multiples of 8)"))
    with pytest.warns(UserWarning, match="gated_mlp: sizes of 63 and 40"):
        ops.gated_mlp(x[:, :63], wg[:, :63], wu[:, :63], wd[:63])
    _clean()


def test_single_rows_of_any_stride():
    """A row's stride means nothing where there is one row; tensor maps take none below a row's width."""
    ops = _ops()
    torch.manual_seed(71)
    fns, x, _ = _calls()
    f = ops.RotaryFrequencies(32, 10000.0)
    fns["rotary"] = lambda t: ops.rotary(t, 1, f, 2, 32)
    kept = ops.quantize_fp8((torch.randn(40, 64, device="cuda") * 0.2).bfloat16(), 128)
    fns["kept"] = lambda t: ops.fp8_linear(t, kept)
    row = x[:1].contiguous()
    for name, fn in fns.items():
        for stride in (0, 8, 1000):
            odd = torch.as_strided(x.clone(), (1, 64), (stride, 1))
            assert torch.equal(fn(odd), fn(row)), (name, stride)
            if name == "kept":
                continue
            grads = []
            for t in (odd, row):
                leaf = t.detach().requires_grad_()
                y = fn(leaf)
                grads.append(torch.autograd.grad(y, leaf, torch.as_strided(torch.ones(40 * 64, device="cuda", dtype=y.dtype), y.shape, (stride % 16, 1)))[0])
            assert torch.equal(*grads), (name, stride)
    a, b = ops.quantize_fp8(row), ops.quantize_fp8(row, 128)
    for stride in (0, 16):
        odd = torch.as_strided(a.values.clone(), (1, 64), (stride, 1))
        assert torch.equal(ops.fp8_matmul(a._replace(values=odd), b._replace(values=odd)), ops.fp8_matmul(a, b))
        assert torch.equal(a._replace(values=odd).dequantize(), a.dequantize())
    _clean()


def test_what_is_kept_goes_through_hooks():
    """What hooks bring back is used where it is what was kept, and refused where it lies otherwise."""
    fns, x, _ = _calls()
    for name, fn in fns.items():
        leaf = x.clone().requires_grad_()
        want, = torch.autograd.grad(fn(leaf).sum(), leaf)
        with torch.autograd.graph.save_on_cpu():
            y = fn(leaf)
        assert torch.equal(torch.autograd.grad(y.sum(), leaf)[0], want), name
        for unpack in (lambda t: t[:-1] if t.dim() else t, lambda t: t.cpu(), lambda t: t.float(), lambda t: torch.cat([t, t])):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = fn(leaf)
            with pytest.raises(RuntimeError, match="himuon"):
                torch.autograd.grad(y.sum(), leaf)
    _clean()


def test_what_changes_before_the_backward_pass_is_noticed():
    ops = _ops()
    torch.manual_seed(73)
    f, at = ops.RotaryFrequencies(32, 10000.0), torch.arange(14, device="cuda")
    w = [(torch.randn(*s, device="cuda") * 0.2).bfloat16().requires_grad_() for s in ((40, 64), (40, 64), (64, 40))]
    x = torch.randn(14, 64, device="cuda").bfloat16().requires_grad_()
    for y, changed in ((ops.rotary(x, at, f, 2, 32), at), (ops.gated_mlp(x, *w), w[2]), (ops.gated_mlp(x, *w), x)):
        with torch.no_grad():
            changed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    _clean()


def test_frequencies_are_not_made_while_a_graph_is_captured():
    ops = _ops()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    t = torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph, stream=side):
        t.add_(1)
        with pytest.raises(RuntimeError, match="before the capture"):
            ops.RotaryFrequencies(32)
    graph.replay()
    torch.cuda.synchronize()
    assert (t == 1).all()


def test_one_matrix_for_gate_and_up():
    """Gradients of a matrix that is used twice are added up, and again over two passes."""
    ops = _ops()
    torch.manual_seed(79)
    for rows in (20, 100, 400):
        x = torch.randn(rows, 64, device="cuda").bfloat16()
        w, d = ((torch.randn(*s, device="cuda") * 0.2).bfloat16() for s in ((40, 64), (64, 40)))
        v = w.clone()
        for t in (w, v, d):
            t.requires_grad_()
        apart = torch.autograd.grad(ops.gated_mlp(x, w, v, d).sum(), (w, v, d))
        ops.gated_mlp(x, w, w, d).sum().backward()
        assert torch.equal(w.grad, apart[0] + apart[1]) and torch.equal(d.grad, apart[2])
        once = w.grad.clone()
        ops.gated_mlp(x, w, w, d).sum().backward()
        assert torch.equal(w.grad, once + once)
    _clean()


def test_layer_operators_from_two_threads():
    """Two threads on streams of their own, at once."""
    import threading

    ops = _ops()
    torch.manual_seed(83)
    f = ops.RotaryFrequencies(32, 10000.0)
    jobs = []
    for rows in (24, 700):
        x = torch.randn(rows, 640, device="cuda").bfloat16()
        w = [(torch.randn(*s, device="cuda") * 0.05).bfloat16() for s in ((1728, 640), (1728, 640), (640, 1728))]

        def step(x=x, w=w):
            leaves = [t.detach().requires_grad_() for t in (x, *w)]
            y = ops.gated_mlp(ops.rotary(leaves[0], x.shape[0], f, 20, 32), *leaves[1:]) + ops.fp8_linear(ops.fp8_linear(leaves[0], leaves[1]), leaves[3])
            return torch.autograd.grad(y.sum(), leaves)

        jobs.append((step, step()))
    torch.cuda.synchronize()
    wrong = []

    def work(step, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got = [step() for _ in range(10)]
                torch.cuda.current_stream().synchronize()
            wrong.extend(1 for g in got if not _same(g, want))
        except Exception as e:                             # (a thread's own would be lost)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    _clean()


@pytest.mark.parametrize("rows", [3, 24, 300, 400])
def test_launches_over_one_another_see_what_came_before(rows):
    """Inputs and weights are overwritten just before each call, eagerly and in a graph: kernels that start early must not read them early."""
    ops = _ops()
    torch.manual_seed(rows + 101)
    xs = [torch.randn(rows, 640, device="cuda").bfloat16() for _ in range(4)]
    ws = [[(torch.randn(*s, device="cuda") * 0.05).bfloat16() for s in ((1728, 640), (1728, 640), (640, 1728))] for _ in range(4)]
    kept = [ops.quantize_fp8(w[2], 128) for w in ws]
    x, w = torch.empty_like(xs[0]), [torch.empty_like(t) for t in ws[0]]
    q = ops.Fp8Blocks(torch.empty_like(kept[0].values), torch.empty_like(kept[0].scales), 128, True)

    def step(i):
        x.copy_(xs[i])
        for a, b in zip((*w, q.values.view(torch.uint8), q.scales), (*ws[i], kept[i].values.view(torch.uint8), kept[i].scales)):
            a.copy_(b)
        h = ops.gated_mlp(x, *w)
        y = ops.fp8_linear(ops.fp8_linear(h, w[0]), q)
        return h, y, ops.fp8_matmul(ops.quantize_fp8(w[1]), q._replace(values=q.values[:, :640], scales=q.scales[:, :5]))

    want = []
    for i in range(4):
        want.append(step(i))
        torch.cuda.synchronize()
    got = [step(i % 4) for i in range(40)]
    assert all(_same(g, want[i % 4]) for i, g in enumerate(got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [step(i) for i in range(4)]
    for _ in range(3):
        graph.replay()
    assert all(_same(a, b) for a, b in zip(captured, want))
    _clean()


@pytest.mark.parametrize("rows", [8, 300])
def test_products_in_branches_of_a_graph(rows):
    """First in a graph, behind copies and fills, on a branch that joins again, behind two branches."""
    ops = _ops()
    torch.manual_seed(rows + 103)
    x = torch.randn(rows, 640, device="cuda").bfloat16()
    q = [ops.quantize_fp8((torch.randn(1728, 640, device="cuda") * 0.05).bfloat16(), 128) for _ in range(2)]
    w = [(torch.randn(*s, device="cuda") * 0.05).bfloat16() for s in ((1728, 640), (1728, 640), (640, 1728))]
    a = ops.quantize_fp8(x)
    want = [ops.fp8_matmul(a, q[0]), ops.fp8_linear(x, q[1]), ops.gated_mlp(x, *w)]
    torch.cuda.synchronize()
    values, scales, y = torch.zeros_like(a.values), torch.zeros_like(a.scales), torch.zeros_like(x)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = ops.fp8_matmul(a, q[0])
        main = torch.cuda.current_stream()
        values.view(torch.uint8).copy_(a.values.view(torch.uint8))
        scales.zero_()
        scales.copy_(a.scales)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y.copy_(x)
            other = ops.fp8_linear(y, q[1])
            block = ops.gated_mlp(y, *w)
        second = ops.fp8_matmul(a._replace(values=values, scales=scales), q[0])
        main.wait_stream(side)
        joined = ops.fp8_matmul(a._replace(values=values, scales=scales), q[0])
        last = ops.gated_mlp(y, *w)
    for _ in range(3):
        for t in (first, second, joined, other, block, last):
            t.zero_()
        graph.replay()
        assert all(torch.equal(t, want[0]) for t in (first, second, joined)) and torch.equal(other, want[1])
        assert torch.equal(block, want[2]) and torch.equal(last, want[2])
    _clean()


def test_offsets_beyond_32_bits():
    """More than 2^31 values: the last rows are those of a call with nothing else."""
    ops = _ops()
    torch.manual_seed(89)
    rows, cols, tail = 547 * 128, 258 * 128, 256
    assert rows * cols > 2 ** 31
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    x[-tail:] = torch.randn(tail, cols, device="cuda")
    for block in (1, 128):
        for turned in (False, True):
            got, want = ops.quantize_fp8(x, block, turned), ops.quantize_fp8(x[-tail:], block, turned)
            if turned:
                assert torch.equal(got.values[:, -tail:].view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(got.scales[:, -tail // 128:], want.scales)
            else:
                assert torch.equal(got.values[-tail:].view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(got.scales[-tail // block:], want.scales)
                assert torch.equal(got.dequantize(torch.bfloat16)[-tail:], want.dequantize(torch.bfloat16))
            del got, want
    f = ops.RotaryFrequencies(96, 10000.0)
    at = torch.arange(rows, device="cuda")
    assert torch.equal(ops.rotary(x, at, f, 258, 128)[-tail:], ops.rotary(x[-tail:], at[-tail:], f, 258, 128))
    odd = ops.RotaryFrequencies(20, 10000.0)
    assert torch.equal(ops.rotary(x, at, odd, 258, 128)[-tail:], ops.rotary(x[-tail:], at[-tail:], odd, 258, 128))
    del x
    a, b = ops.quantize_fp8(torch.randn(rows, 136, device="cuda")), ops.quantize_fp8(torch.randn(cols, 136, device="cuda"), 128)
    for powers in (True, False):
        got = ops.fp8_matmul(a._replace(powers=powers), b)[-tail:, -tail:]
        last = ops.Fp8Blocks(a.values[-tail:], a.scales[-tail:], 1, powers), ops.Fp8Blocks(b.values[-tail:], b.scales[-tail // 128:], 128, True)
        assert torch.equal(got, ops.fp8_matmul(*last))
    _clean()


def test_gated_mlp_offsets_beyond_32_bits():
    ops = _ops()
    torch.manual_seed(97)
    rows, hidden, inter, tail = 65536, 64, 17408, 300
    assert rows * 2 * inter > 2 ** 31
    w = [(torch.randn(*s, device="cuda") * s[1] ** -0.5).bfloat16().requires_grad_() for s in ((inter, hidden), (inter, hidden), (hidden, inter))]
    x = torch.randn(rows, hidden, device="cuda").bfloat16().requires_grad_()
    g = torch.zeros(rows, hidden, device="cuda", dtype=torch.bfloat16)
    g[-tail:] = torch.randn(tail, hidden, device="cuda")
    y = ops.gated_mlp(x, *w)
    got = [y[-tail:].detach()] + [t[-tail:] if i == 0 else t for i, t in enumerate(torch.autograd.grad(y, (x, *w), g))]
    last = x[-tail:].detach().requires_grad_()
    z = ops.gated_mlp(last, *w)
    want = [z.detach(), *torch.autograd.grad(z, (last, *w), g[-tail:])]
    for a, b in zip(got, want):
        # sums may be cut elsewhere: two results rounded to bf16, and as much again for fp32 sums in another order
        assert (a.double() - b.double()).norm() <= 4 * U * b.double().norm()
    _clean()


@pytest.mark.parametrize("rows", [20, 300, 400])
def test_a_decoder_layer_of_them(rows):
    """Queries and keys of one projection in 8 bits, turned, packed attention, and the feed-forward block: forward and backward against 64 bits."""
    ops = _ops()
    torch.manual_seed(rows)
    H, heads, kv, hd, I = 256, 4, 2, 64, 352
    lengths = [rows // 2, rows - rows // 2 - 3]
    layout, f = ops.PackedLayout(lengths), ops.RotaryFrequencies(hd, 10000.0, SCALINGS[5])
    x = torch.randn(rows, H, device="cuda").bfloat16().requires_grad_()
    w = [(torch.randn(n, m, device="cuda") / math.sqrt(m)).bfloat16().requires_grad_() for n, m in (((heads + 2 * kv) * hd, H), (H, heads * hd), (I, H), (I, H), (H, I))]
    dy = torch.randn(rows, H, device="cuda").bfloat16()

    def layer(x, w, linear, rotate, attend, feed):
        qkv = linear(x, w[0])
        qk, v = rotate(qkv[:, : (heads + kv) * hd]), qkv[:, (heads + kv) * hd:]
        a = x + linear(attend(qk[:, : heads * hd], qk[:, heads * hd:], v), w[1])
        return a + feed(a, *w[2:])

    y = layer(x, w, ops.fp8_linear, lambda t: ops.rotary(t, layout.positions(rows), f, heads + kv, hd),
              lambda q, k, v: ops.packed_attention(q, k, v, layout, heads, kv, hd), ops.gated_mlp)
    grads = torch.autograd.grad(y, (x, *w), dy)
    from himuon_b200.ops import reference as ref

    x64, w64 = x.detach().double().requires_grad_(), [t.detach().double().requires_grad_() for t in w]
    inv = torch.tensor(f.frequencies, dtype=torch.float64, device="cuda")
    z = layer(x64, w64, lambda t, m: t @ m.t(), lambda t: ref.rotary(t, layout.positions(rows), inv, f.factor, heads + kv, hd, False),
              lambda q, k, v: ref.packed_attention(q, k, v, lengths, heads, kv, hd), ref.gated_mlp)
    want = torch.autograd.grad(z, (x64, *w64), dy.double())
    # 8 bits round a value by 2^-4 of itself at most, 2^-5.8 = 0.018 on average and both operands of a product: 0.025; four such products lie one behind the
    # other on the way to a gradient, and softmax passes an error of the scores on at most twice
    for name, got, exact in zip(("y", "x", "qkv", "o", "gate", "up", "down"), (y, *grads), (z, *want)):
        assert (got.double() - exact).norm() <= 0.2 * exact.norm(), name
    _clean()
