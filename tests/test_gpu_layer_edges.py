"""The rotary positions, the gated feed-forward block and the 8-bit products on the GPU where they have been wrong: far gates, rows that come
with others, transforms of operands that are not the first, angles next to half a turn (GPU tier).

Bounds follow from the kernels' roundings and stand where they are used; U = 2^-8 is what rounding to bf16 changes a value by at most.
"""

import math

import pytest
import torch

from test_gpu_layer_ops import GATED, SCALINGS, TURN, _gated64, _rotary64, _sums, _values64, _within

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def _ops():
    from himuon_b200 import ops

    return ops


def _clean():
    from himuon_b200._ext import ext

    torch.cuda.synchronize()
    assert ext().status(True) == 0, "a bounded device wait ran out (status word set)"


# ------------------------------------------------------------------------------------------- far gates
SIDE = 1448                       # hidden and intermediate features: 20, 200 and 400 rows of them go to different kernels


def _gates_as_given(rows, gates, up):
    """Leaves whose gate projections are `gates` (one for each feature) and up projections `up`, exactly, in every row; the down projection
    passes features through."""
    x = torch.zeros(rows, SIDE, device="cuda")
    x[:, 0], x[:, 1] = 1.0, 2.0 ** (math.frexp(up)[1] // 2)
    wg, wu = (torch.zeros(SIDE, SIDE, device="cuda") for _ in range(2))
    wg[:, 0] = gates
    wu[:, 1] = up / x[0, 1]
    leaves = [t.bfloat16().requires_grad_() for t in (x, wg, wu, torch.eye(SIDE, device="cuda"))]
    assert (leaves[1][:, 0].double() == gates.double()).all() and (x[0, 1].double() * leaves[2][:, 1].double() == up).all()
    return leaves


@pytest.mark.parametrize("rows", [20, 200, 400])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_far_negative_gates_are_nothing(activation, rows):
    """Below -120 an activation is smaller than fp32's least number: results and gradients are 0, up to the least gate that bf16 has."""
    ops = _ops()
    gates = -torch.exp2(torch.linspace(7.0, 127.0, SIDE, device="cuda")).bfloat16().float()
    gates[-1] = torch.finfo(torch.bfloat16).min
    leaves = _gates_as_given(rows, gates, 3.0)
    y = ops.gated_mlp(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, torch.randn_like(y))
    for name, t in zip(("y", "dx", "dwg", "dwu", "dwd"), (y, *grads)):
        assert not t.any(), (name, t.abs().max().item())
    _clean()


@pytest.mark.parametrize("rows", [20, 200, 400])
def test_gates_where_the_sigmoid_leaves_the_range_of_numbers(rows):
    """silu of -60 to -100, seen through an up projection of 2^100.  The sigmoid is 0 below 2^-126; an exponential of 127 ln 2 is good to 2^-16 (its
    argument's rounding, 2^-18, and the constant's) as is what is made of it."""
    ops = _ops()
    gates = torch.linspace(-100.0, -60.0, SIDE, device="cuda").bfloat16().float()
    up = 2.0 ** 100
    leaves = _gates_as_given(rows, gates, up)
    y = ops.gated_mlp(*leaves)
    _, dwg, dwu, _ = torch.autograd.grad(y, leaves, torch.ones_like(y))
    g = gates.double()
    s = torch.sigmoid(g)
    a, d = g * s, s * (1.0 + g * torch.sigmoid(-g))
    near, least = 2.0 ** -16, 101.0 * 2.0 ** -126
    h, side = a * up, leaves[0][0, 1].double()
    # h, or dg and du, are rounded to bf16 and so is the result
    for name, got, want, scale in (("y", y.double(), h.expand(rows, -1), up), ("dwg", dwg[:, 0].double(), rows * up * d, rows * up), ("dwu", dwu[:, 1].double(), rows * side * a, rows * side)):
        bound = (2 * U + U * U + 2 * near) * want.abs() + 1.01 * least * scale
        over = (got - want).abs() - bound
        assert (over <= 0).all(), (name, over.max().item())
    _clean()


@pytest.mark.parametrize("rows", [20, 200, 400])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_gates_that_are_no_numbers(activation, rows):
    """-inf times a sigmoid of 0 is no number, and NaN stays."""
    ops = _ops()
    for gate in (-math.inf, math.nan):
        x = torch.zeros(rows, SIDE, device="cuda")
        wg, wu = (torch.zeros(SIDE, SIDE, device="cuda") for _ in range(2))
        x[:, 0], wg[:, 0], wu[:, 0] = 1.0, gate, 1.0
        y = ops.gated_mlp(*(t.bfloat16() for t in (x, wg, wu, torch.ones(SIDE, SIDE, device="cuda"))), activation=activation)
        assert y.isnan().all()
    _clean()


# ------------------------------------------------------------------------------------------- sines and cosines
@pytest.mark.parametrize("heads,hd,interleaved", [(1, 128, False), (3, 128, True), (1, 130, False)])
def test_sines_of_every_place_in_a_turn(heads, hd, interleaved):
    """Pairs (1, 0) come out as cosine and sine.  A place in the turn has 32 bits, so an angle is off by pi * 2^-32; a sine or cosine is good to a unit of its last
    place, 2^-23 of it, and half of one for what the angle's low bits add.  So results near 0 are as good as near 1."""
    ops = _ops()
    torch.manual_seed(17)
    f = ops.RotaryFrequencies(128, 10000.0)
    x = torch.zeros(20000, heads, hd, device="cuda")
    x[..., 0:128:2] = 1.0
    if not interleaved:
        x[..., :128] = torch.cat([torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")])
    at = torch.randint(0, 131072, (20000,), device="cuda")
    y = ops.rotary(x.view(20000, -1), at, f, heads, hd, interleaved=interleaved).view(20000, heads, hd)[..., :128].double()
    cos, sin = (y[..., 0::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)
    angles = at.double()[:, None] * torch.tensor(f.frequencies, dtype=torch.float64, device="cuda")
    for got, want in ((cos, angles.cos()), (sin, angles.sin())):
        over = (got - want[:, None]).abs() - (math.pi * 2.0 ** -32 + 1e-10 + 1.5 * 2.0 ** -23 * want[:, None].abs())
        assert (over <= 0).all(), over.max().item()
    _clean()


# ------------------------------------------------------------------------------------------- rows that come with others
def _rows(m, n):
    return m._replace(values=m.values[:n], scales=m.scales[:n])


@pytest.mark.parametrize("powers", [True, False])
@pytest.mark.parametrize("outer,inner", [(2048, 2048), (200, 1000), (24, 16400)])
def test_few_8_bit_rows_do_not_depend_on_one_another(outer, inner, powers):
    """In fp32, which hides no order of sums: a row has the same bits alone and with up to 31 others."""
    ops = _ops()
    torch.manual_seed(outer + inner)
    a, b = ops.quantize_fp8(torch.randn(32, inner, device="cuda")), ops.quantize_fp8(torch.randn(outer, inner, device="cuda"), 128)
    if not powers:
        a, b = (m._replace(scales=m.scales * (0.5 + torch.rand_like(m.scales)), powers=False) for m in (a, b))
    whole = ops.fp8_matmul(a, b, out_dtype=torch.float32)
    for n in (1, 7, 8, 9, 16, 17, 31):
        assert torch.equal(ops.fp8_matmul(_rows(a, n), b, out_dtype=torch.float32), whole[:n]), n
    _clean()


def test_few_8_bit_rows_of_a_large_weight():
    """Above 2^24 values rows come in groups of up to 16 or more, each with one order of sums; the two differ by fp32 roundings of the terms: 2^-23 of
    their absolute values for each sum of 16 products and each of what is done to them."""
    ops = _ops()
    torch.manual_seed(7)
    outer, inner = 4104, 4096
    a, b = ops.quantize_fp8(torch.randn(32, inner, device="cuda")), ops.quantize_fp8(torch.randn(outer, inner, device="cuda"), 128)
    few, many = (ops.fp8_matmul(_rows(a, n), b, out_dtype=torch.float32) for n in (16, 32))
    for n in (1, 8, 9):
        assert torch.equal(ops.fp8_matmul(_rows(a, n), b, out_dtype=torch.float32), few[:n]), n
    for n in (17, 31):
        assert torch.equal(ops.fp8_matmul(_rows(a, n), b, out_dtype=torch.float32), many[:n]), n
    va, vb = (m.dequantize().double() for m in (a, b))
    want, bound = va @ vb.t(), 2.0 ** -23 * (inner / 16 + 17) * (va.abs() @ vb.abs().t())
    assert ((many.double() - want).abs() <= bound).all() and ((few.double() - want[:16]).abs() <= bound[:16]).all()
    _clean()


# ------------------------------------------------------------------------------------------- transforms of any operand
@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
def test_vmap_over_positions():
    """Rows that stay and positions that do not: what calls one by one return, but for two roundings to bf16."""
    ops = _ops()
    torch.manual_seed(11)
    f, x, at = ops.RotaryFrequencies(16), torch.randn(6, 64, device="cuda").bfloat16(), torch.randint(0, 10000, (3, 6), device="cuda")
    got = torch.vmap(lambda p: ops.rotary(x, p, f, 2, 32))(at)
    for i in range(3):
        want = ops.rotary(x, at[i], f, 2, 32).double()
        assert (got[i].double() - want).abs().max() <= 2.01 * U * want.abs().max()
    y = torch.vmap(lambda t, p: ops.rotary(t, p, f, 2, 32))(torch.stack([x] * 3), at)
    assert torch.equal(y, got)
    _clean()


@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
@pytest.mark.parametrize("over", ["values", "scales", "both"])
def test_vmap_over_8_bit_operands(over):
    """Values, scales or both of either operand, of a kept weight, and of what is put back to fp32."""
    ops = _ops()
    torch.manual_seed(13)
    x = torch.randn(5, 200, device="cuda").bfloat16()
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(torch.randn(140, 200, device="cuda"), 128)

    def forms(m):
        values = torch.stack([m.values.view(torch.uint8), m.values.flip(0).contiguous().view(torch.uint8)]).view(torch.float8_e4m3fn)
        scales = torch.stack([m.scales, m.scales * 4])
        return (values if over != "scales" else m.values.expand(2, -1, -1), scales if over != "values" else m.scales.expand(2, -1, -1))

    def each(m, fn):
        values, scales = forms(m)
        mapped = (values if over != "scales" else values[0], scales if over != "values" else scales[0])
        dims = (0 if over != "scales" else None, 0 if over != "values" else None)
        got = torch.vmap(lambda v, s: fn(m._replace(values=v, scales=s)), in_dims=dims)(*mapped)
        return [(got[i], m._replace(values=values[i].contiguous(), scales=scales[i].contiguous())) for i in range(2)]

    def size(p, q):
        return p.dequantize().double().abs() @ q.dequantize().double().abs().t()

    sums = 2 * 2.0 ** -23 * (200 / 16 + 17)                # two fp32 sums of the terms
    for got, m in each(b, lambda m: m.dequantize()):
        assert torch.equal(got, m.dequantize())
    for got, m in each(b, lambda m: ops.fp8_matmul(a, m, out_dtype=torch.float32)):
        assert ((got - ops.fp8_matmul(a, m, out_dtype=torch.float32)).abs() <= sums * size(a, m)).all()
    for got, m in each(a, lambda m: ops.fp8_matmul(m, b, out_dtype=torch.float32)):
        assert ((got - ops.fp8_matmul(m, b, out_dtype=torch.float32)).abs() <= sums * size(m, b)).all()
    for got, m in each(b, lambda m: ops.fp8_linear(x, m)):
        want = ops.fp8_linear(x, m).double()
        assert ((got.double() - want).abs() <= sums * size(a, m) + 2.01 * U * (want.abs() + sums * size(a, m))).all()
    _clean()


# ------------------------------------------------------------------------------------------- one behind the other
@pytest.mark.parametrize("rows", [20, 300])
def test_a_layer_operator_by_operator(rows):
    """Each operator of a decoder layer against 64 bits on what it was really given, forward and backward, under its own bound: column slices of one projection as
    operands, gradients that come as slices, sums of branches, 8-bit copies of what another kernel has just written."""
    ops = _ops()
    torch.manual_seed(rows + 19)
    H, heads, kv, hd, I = 256, 4, 2, 64, 352
    layout, f = ops.PackedLayout([rows // 2, rows - rows // 2 - 3]), ops.RotaryFrequencies(hd, 10000.0, SCALINGS[5])
    at = layout.positions(rows)
    x = torch.randn(rows, H, device="cuda").bfloat16().requires_grad_()
    w = [(torch.randn(n, m, device="cuda") / math.sqrt(m)).bfloat16().requires_grad_() for n, m in (((heads + 2 * kv) * hd, H), (H, heads * hd), (I, H), (I, H), (H, I))]
    calls = []

    def call(fn, t, *weights):
        given = t.view_as(t)                               # its gradient is this operator's alone
        out = fn(given, *weights)
        for s in (given, out):
            s.retain_grad()
        calls.append((given, out, weights))
        return out

    qkv = call(ops.fp8_linear, x, w[0])
    qk = call(lambda t: ops.rotary(t, at, f, heads + kv, hd), qkv[:, : (heads + kv) * hd])
    o = ops.packed_attention(qk[:, : heads * hd], qk[:, heads * hd:], qkv[:, (heads + kv) * hd:], layout, heads, kv, hd)
    a = x + call(ops.fp8_linear, o, w[1])
    y = a + call(ops.gated_mlp, a, *w[2:])
    y.backward(torch.randn_like(y))
    _clean()
    for given, out, weights in (calls[0], calls[2]):
        t, m, g = given.detach(), weights[0].detach(), out.grad
        q = {n: _values64(ops.quantize_fp8(s, b, transpose=tr)) for n, s, b, tr in
             (("x", t, 1, False), ("w", m, 128, False), ("dy", g, 1, False), ("dyt", g, 1, True), ("xt", t, 128, True))}
        for what, got, p, r in (("y", out, q["x"], q["w"].t()), ("dx", given.grad, q["dy"], q["w"]), ("dw", weights[0].grad, q["dyt"], q["xt"].t())):
            want, bound = p @ r, _sums(p.shape[1]) * (p.abs() @ r.abs())
            _within(got, want, bound + U * (want.abs() + bound), what)
    given, out, _ = calls[1]
    angles = at.double()[:, None] * torch.tensor(f.frequencies, dtype=torch.float64, device="cuda")
    for got, t, sign in ((out, given, 1.0), (given.grad, out.grad, -1.0)):
        want, size = _rotary64(t, angles.cos(), sign * angles.sin(), heads + kv, hd, False)
        _within(got, want, U * want.abs() + TURN * (1 + U) * size, "rotary")
    given, out, weights = calls[3]
    exact = _gated64(given, *weights, "silu", out.grad)
    for name, got in zip(GATED, (out, given.grad, *(m.grad for m in weights))):
        _within(got, *exact[name], name)


# ------------------------------------------------------------------------------------------- more than one device
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_products_on_a_second_device_of_the_process():
    """What a kernel is allowed, and how many of its blocks fit, is asked on each device: the same calls on the first and then on another."""
    ops = _ops()
    torch.manual_seed(5)
    for rows in (24, 100, 200, 400):
        x, wg, wu, wd = (torch.randn(*s).bfloat16() * 0.1 for s in ((rows, 640), (1728, 640), (1728, 640), (640, 1728)))
        got = []
        for device in ("cuda:0", "cuda:1"):
            leaves = [t.to(device).requires_grad_() for t in (x, wg, wu, wd)]
            y = ops.gated_mlp(*leaves) + ops.fp8_linear(ops.linear(leaves[0], leaves[1]), leaves[3])
            got.append([t.cpu() for t in (y.detach(), *torch.autograd.grad(y.sum(), leaves))])
        assert all(torch.equal(a, b) for a, b in zip(*got))
    _clean()
