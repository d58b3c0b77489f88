"""Packed attention and token scores on the GPU against 64-bit formulas (GPU tier).

The bounds are element by element and follow from the kernels' roundings: u = 2^-8 is what rounding to bf16 changes a value by
at most (relative), and each product of rounded factors passes that on through the absolute values of the terms of its sum.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8          # bf16
F = 1e-4               # fp32 sums, exponentials and differences of scores, relative to the terms' absolute values


def _ops():
    from himuon_b200 import ops

    return ops


def _clean():
    from himuon_b200._ext import ext

    torch.cuda.synchronize()
    assert ext().status(True) == 0, "a bounded device wait ran out (status word set)"


def _within(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: {(over > 0).sum().item()} of {over.numel()} outside, worst by {over.max().item():.3g}"


def _heads(t, hd):
    return t.detach().double().view(t.shape[0], -1, hd).transpose(0, 1)


def _flat(t):
    return t.transpose(0, 1).reshape(t.shape[1], -1)


def _attention64(q, k, v, lengths, Hq, Hkv, hd, scale, do=None):
    """Results and bounds in 64 bits, one document at a time; zero for padding."""
    T, G = q.shape[0], Hq // Hkv
    q, k, v = (_heads(t, hd) for t in (q, k, v))
    do = None if do is None else _heads(do, hd)
    out = {n: torch.zeros(h, T, hd, dtype=torch.float64, device=q.device) for n, h in
           (("o", Hq), ("dq", Hq), ("dk", Hkv), ("dv", Hkv), ("bo", Hq), ("bdq", Hq), ("bdk", Hkv), ("bdv", Hkv))}
    first = 0
    for n in lengths:
        c = slice(first, first + n)
        first += n
        if n == 0:
            continue
        kk, vv = (t[:, c].repeat_interleave(G, 0) for t in (k, v))
        qq = q[:, c]
        s = scale * qq @ kk.transpose(1, 2)
        p = torch.softmax(s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf), -1)
        o = p @ vv
        # P is rounded, and so is the sum of it that it is divided by; then the result
        bo = U * o.abs() + (2 * U + F) * (p @ vv.abs())
        out["o"][:, c], out["bo"][:, c] = o, bo
        if do is None:
            continue
        g = do[:, c]
        dp = g @ vv.transpose(1, 2)
        delta = (g * o).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # dS is rounded; delta has been summed from the rounded output
        bds = U * ds.abs() + p * ((g.abs() * bo).sum(-1, keepdim=True) + F * (g.abs() @ vv.abs().transpose(1, 2) + (g * o).abs().sum(-1, keepdim=True)))
        per = {"dq": (scale * ds @ kk, scale * bds @ kk.abs()),
               "dk": (scale * ds.transpose(1, 2) @ qq, scale * bds.transpose(1, 2) @ qq.abs()),
               "dv": (p.transpose(1, 2) @ g, (U + F) * p.transpose(1, 2) @ g.abs())}
        for name, (val, bound) in per.items():
            if name != "dq":
                val, bound = (t.view(Hkv, G, n, hd).sum(1) for t in (val, bound))
            out[name][:, c] = val
            out["b" + name][:, c] = bound + U * (val.abs() + bound)
    return {n: _flat(t) for n, t in out.items()}


SHAPES = [(4, 2, 32), (2, 2, 64), (8, 2, 128), (3, 1, 128), (2, 1, 72), (1, 1, 8), (6, 3, 96)]
BATCHES = [([1], 0), ([0, 0, 2], 5), ([128], 0), ([127, 1, 0, 64, 65], 7), ([129, 256, 3], 0), ([5, 1, 0, 700, 30, 513], 0), ([1100], 100), ([90] * 80, 3)]


@pytest.mark.parametrize("Hq,Hkv,hd", SHAPES)
@pytest.mark.parametrize("lengths,pad", BATCHES)
def test_packed_attention(Hq, Hkv, hd, lengths, pad):
    ops = _ops()
    torch.manual_seed(sum(lengths) + hd)
    T = sum(lengths) + pad
    q, k, v, do = (torch.randn(T, h * hd, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv, Hq))
    for t in (q, k, v):
        t.requires_grad_()
    layout = ops.PackedLayout(lengths)
    # a group's heads one by one for a long document, together in a large batch and in small ones
    assert layout.splits_heads(Hq, Hkv) == (Hq > Hkv and lengths == [1100]) or lengths[3:4] == [700]
    before = ops.launch_count()
    o = ops.packed_attention(q, k, v, layout, Hq, Hkv, hd)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    assert ops.launch_count() >= before + 3
    _clean()
    want = _attention64(q, k, v, lengths, Hq, Hkv, hd, 1 / math.sqrt(hd), do)
    for name, got in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        _within(got, want[name], want["b" + name], name)
        assert not got[sum(lengths):].any()                        # padding


def test_packed_attention_of_peaked_scores_and_another_scale():
    """Scores whose row maximum keeps growing along the document, so that the running maximum moves in every block."""
    ops = _ops()
    torch.manual_seed(3)
    lengths, Hq, Hkv, hd = [400, 37], 2, 1, 128
    T = sum(lengths)
    ramp = torch.linspace(0, 6, T, device="cuda")[:, None]
    q, k, v, do = (torch.randn(T, h * hd, device="cuda") for h in (Hq, Hkv, Hkv, Hq))
    q, k = (1 + 0.1 * q).bfloat16().requires_grad_(), (ramp + 0.1 * k).bfloat16().requires_grad_()
    v, do = v.bfloat16().requires_grad_(), do.bfloat16()
    o = ops.packed_attention(q, k, v, ops.PackedLayout(lengths), Hq, Hkv, hd, scale=0.25)
    grads = torch.autograd.grad(o, (q, k, v), do)
    _clean()
    want = _attention64(q, k, v, lengths, Hq, Hkv, hd, 0.25, do)
    # a score of up to 200 rounds to 2^-17 in fp32, and e^x passes that on
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        _within(got, want[name], want["b" + name], name)


def test_gradients_of_nearly_certain_rows():
    """One weight near 1 in a row: dP - delta is small beside both, and what delta loses by O's rounding would be a multiple of it."""
    ops = _ops()
    torch.manual_seed(47)
    H, hd, n = 3, 128, 400
    layout = ops.PackedLayout([2] * n)
    q, k, v = (torch.randn(2 * n, H * hd, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    do = torch.randn(2 * n, H * hd, device="cuda").bfloat16()
    grads = torch.autograd.grad(ops.packed_attention(q, k, v, layout, H, H, hd, scale=0.5), (q, k, v), do)
    a, b, c = (t.detach().double().view(n, 2, H, hd) for t in (q, k, v))
    g = do.double().view(n, 2, H, hd)[:, 1]
    # the second token of two: weights p and 1 - p, dS = p (1 - p) (dO v0 - dO v1) on the first and its negative on the second
    p = torch.sigmoid(0.5 * (a[:, 1] * (b[:, 0] - b[:, 1])).sum(-1))
    ds = p * (1 - p) * (g * (c[:, 0] - c[:, 1])).sum(-1)
    dq = 0.5 * ds[..., None] * (b[:, 0] - b[:, 1])
    # P and dS in bf16, O and delta to 2^-16 (and fp32 sums of 128 terms): relative to dS, and what is lost beside it, p of it on the
    # first token and 1 - p on the second
    lost = (2 * 2.0 ** -16 + 300 * 2.0 ** -24) * (g.abs() * (c[:, 0].abs() + c[:, 1].abs())).sum(-1)
    lost = lost + 2.0 ** -8 * torch.minimum(p, 1 - p) * (g * (c[:, 0] - c[:, 1])).sum(-1).abs()
    bound = 3 * 2.0 ** -8 * dq.abs() + 0.5 * (2 * 2.0 ** -8 * ds.abs() + 2 * lost)[..., None] * (b[:, 0].abs() + b[:, 1].abs()) + 1e-6
    got = grads[0].double().view(n, 2, H, hd)
    assert ((got[:, 1] - dq).abs() <= bound).all()
    certain = torch.minimum(p, 1 - p) < 1e-3
    assert certain.any()
    err = (got[:, 1] - dq)[certain].norm() / dq[certain].norm()
    assert err < 0.02, err
    _clean()


def test_packed_attention_gradient_against_differences():
    """The kernels' gradient along a direction against a central difference of the 64-bit formula."""
    ops = _ops()
    torch.manual_seed(5)
    lengths, Hq, Hkv, hd = [150, 3, 90], 4, 2, 64
    T = sum(lengths)
    q, k, v, do = (torch.randn(T, h * hd, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv, Hq))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.packed_attention(*leaves, ops.PackedLayout(lengths), Hq, Hkv, hd), leaves, do)
    want = _attention64(q, k, v, lengths, Hq, Hkv, hd, hd ** -0.5, do)
    base = [t.detach().double() for t in leaves]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like(base[i])
        at = [[b + s * 1e-4 * d if j == i else b for j, b in enumerate(base)] for s in (1, -1)]
        f = [(_attention64(*x, lengths, Hq, Hkv, hd, hd ** -0.5)["o"] * do.double()).sum().item() for x in at]
        slope = (f[0] - f[1]) / 2e-4
        got = (grads[i].double() * d).sum().item()
        assert abs(got - slope) <= (want["b" + name] * d.abs()).sum().item() + 1e-5 * abs(slope)


def test_gradients_are_not_differentiable_again():
    ops = _ops()
    q = torch.randn(20, 64, device="cuda").bfloat16().requires_grad_()
    x, ids = torch.randn(4, 64, device="cuda", requires_grad=True), torch.zeros(4, dtype=torch.int64, device="cuda")
    h, w = torch.randn(4, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(100, 64, device="cuda").bfloat16()
    for out, leaf in ((ops.packed_attention(q, q.detach(), q.detach(), ops.PackedLayout([20]), 1, 1, 64), q), (ops.token_log_probs(x, ids).entropy, x),
                      (ops.linear_token_log_probs(h, w, ids).entropy, h)):
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)
        torch.autograd.grad(out.sum(), leaf)
    _clean()


def test_packed_attention_keeps_documents_apart():
    """NaN and infinities in one document and in the padding reach no other document, forward or backward."""
    ops = _ops()
    torch.manual_seed(7)
    lengths, pad, Hq, Hkv, hd = [70, 50, 133, 9], 20, 4, 2, 128
    T = sum(lengths) + pad
    clean = [torch.randn(T, h * hd, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv, Hq)]
    bad = [t.clone() for t in clean]
    for i, t in enumerate(bad):
        t[70:120] = math.nan if i % 2 else math.inf
        t[sum(lengths):] = math.nan
    layout, got = ops.PackedLayout(lengths), []
    for q, k, v, do in (clean, bad):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.packed_attention(*leaves, layout, Hq, Hkv, hd)
        got.append((o.detach(), *torch.autograd.grad(o, leaves, do)))
    _clean()
    others = torch.ones(T, dtype=torch.bool, device="cuda")
    others[70:120] = False
    for a, b in zip(*got):
        assert torch.equal(a[others], b[others])


def test_packed_attention_takes_slices_and_odd_rows():
    """q, k, v as column slices of one projection, rows that start off the 16-byte grid, expanded gradients."""
    ops = _ops()
    torch.manual_seed(9)
    lengths, Hq, Hkv, hd = [40, 200], 4, 2, 64
    T = sum(lengths)
    packed = torch.randn(T, (Hq + 2 * Hkv) * hd + 1, device="cuda").bfloat16()
    layout = ops.PackedLayout(torch.tensor(lengths, device="cuda"))
    for base in (packed[:, :-1].contiguous(), packed[:, 1:]):
        q, k, v = base.split([Hq * hd, Hkv * hd, Hkv * hd], 1)
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = ops.packed_attention(q, k, v, layout, Hq, Hkv, hd)
        grads = torch.autograd.grad(o.sum(), (q, k, v))
        want = _attention64(q, k, v, lengths, Hq, Hkv, hd, hd ** -0.5, torch.ones(T, Hq * hd, device="cuda"))
        for name, got in zip(("o", "dq", "dk", "dv"), (o, *grads)):
            _within(got, want[name], want["b" + name], name)
    _clean()


def test_packed_attention_of_equal_documents_matches_the_unpacked_one():
    ops = _ops()
    torch.manual_seed(11)
    B, S, Hq, Hkv, hd = 3, 256, 4, 2, 128
    q, k, v = (torch.randn(B * S, h * hd, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    a = ops.packed_attention(q, k, v, ops.PackedLayout([S] * B), Hq, Hkv, hd)
    b = ops.attention(q, k, v, B, S, Hq, Hkv, hd)
    assert (a.float() - b.float()).abs().max() <= 2 * U * (1 + v.float().abs().max())
    _clean()


def test_packed_attention_on_another_stream_and_in_a_graph():
    ops = _ops()
    torch.manual_seed(13)
    lengths, H, hd = [90, 300], 2, 128
    q, k, v = (torch.randn(390, H * hd, device="cuda").bfloat16() for _ in range(3))
    layout = ops.PackedLayout(lengths)
    want = ops.packed_attention(q, k, v, layout, H, H, hd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.packed_attention(q, k, v, ops.PackedLayout(lengths), H, H, hd)
        got2 = ops.packed_attention(q, k, v, layout, H, H, hd)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got2, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.packed_attention(q, k, v, layout, H, H, hd)
    q.copy_(torch.randn_like(q))
    graph.replay()
    assert torch.equal(out, ops.packed_attention(q, k, v, layout, H, H, hd))
    _clean()


def test_layout_copies_no_table_while_a_graph_is_captured():
    ops = _ops()
    layout, graph = ops.PackedLayout([3, 5]), torch.cuda.CUDAGraph()
    layout.positions()
    with torch.cuda.graph(graph):
        there = layout.positions() + 1
        with pytest.raises(RuntimeError, match="before the capture"):
            layout.positions(10)
    graph.replay()
    assert there.tolist() == [1, 2, 3, 1, 2, 3, 4, 5]
    assert layout.positions(10).tolist() == [0, 1, 2, 0, 1, 2, 3, 4, 0, 0]


def test_packed_attention_repeats_its_bits():
    ops = _ops()
    torch.manual_seed(15)
    lengths, Hq, Hkv, hd = [1000, 24, 600, 300], 8, 2, 128
    leaves = [torch.randn(sum(lengths), h * hd, device="cuda").bfloat16().requires_grad_() for h in (Hq, Hkv, Hkv)]
    do = torch.randn(sum(lengths), Hq * hd, device="cuda").bfloat16()
    layout, seen = ops.PackedLayout(lengths), None
    for _ in range(5):
        o = ops.packed_attention(*leaves, layout, Hq, Hkv, hd)
        got = (o, *torch.autograd.grad(o, leaves, do))
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, got))
        seen = got
    _clean()


def test_packed_attention_refusals_of_the_kernel_path():
    ops = _ops()
    q = torch.randn(4, 64, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="layout is on"):
        ops.packed_attention(q, q, q, ops.PackedLayout([4], device="cpu"), 2, 2, 32)
    from himuon_b200._ext import ext
    plan, lse, low = ops.PackedLayout([4]).plan, torch.empty(256, device="cuda"), torch.empty(256 * 32, device="cuda", dtype=torch.int8)
    ok = (plan, 1, 4, q, q, q, torch.empty_like(q), lse, low, 2, 2, 0.1)
    ext().packed_attn_fwd(*ok)
    for i, bad in [(0, plan.long()), (0, plan[:, :2].contiguous()), (0, plan.cpu()), (0, plan[:1]), (1, 2), (1, -1), (2, 5), (3, q.float()), (4, q[:, :32]), (5, q[:2]),
                   (6, q.t()), (7, lse[:128]), (7, lse.double()), (7, None), (8, low[:64]), (8, low.int()), (8, low.cpu()), (9, 3), (10, 0), (3, torch.randn(5, 64, device="cuda").bfloat16().flatten()[4:260].view(4, 64))]:
        with pytest.raises(RuntimeError, match="himuon"):
            ext().packed_attn_fwd(*ok[:i], bad, *ok[i + 1:])
    _clean()


# ------------------------------------------------------------------------------------------- scores
def _log_tolerance(vocab):
    """Of a log probability: each thread adds up to vocab / 256 terms (and a row's sum at least one of 1), each exponential is
    good to 2^-21, d and the result are rounded."""
    return (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -19


def _scores64(x, ids, ignore=-100):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    counted = ids != ignore
    log_probs = lp.gather(1, torch.where(counted, ids, 0)[:, None])[:, 0].masked_fill(~counted, 0.0)
    entropy = -(lp.exp() * lp.clamp(min=-1e30)).sum(-1)
    return lp, log_probs, entropy


def _grad64(lp, entropy, ids, g, h, ignore=-100):
    counted = ids != ignore
    g = (g.double() * counted)[:, None]
    h = h.double()[:, None]
    p, l = lp.exp(), lp.clamp(min=-1e30)
    dx = -p * (g + h * torch.where(p > 0, l + entropy[:, None], 0.0))
    dx.scatter_add_(1, torch.where(counted, ids, 0)[:, None], g)
    size = p * (g.abs() + h.abs() * (torch.where(p > 0, l.abs(), 0.0) + entropy[:, None]))
    return dx, size


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 33), (5, 1000), (40, 4097), (2, 151936), (3, 32003), (700, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 3])
def test_token_log_probs(rows, vocab, dtype, offset):
    ops = _ops()
    torch.manual_seed(vocab + rows)
    wide = (torch.randn(rows, vocab + offset + (8 if offset else 0), device="cuda") * 3).to(dtype)
    x = wide[:, offset: offset + vocab].detach().requires_grad_()       # an offset: rows of a wider buffer, off the 16-byte grid
    ids = torch.randint(0, vocab, (rows,), device="cuda")
    ids[rows // 2] = -100 if rows > 2 else ids[rows // 2]
    k = min(20, vocab)
    s = ops.token_log_probs(x, ids, top_k=k)
    lp, log_probs, entropy = _scores64(x.detach(), ids)
    tol = _log_tolerance(vocab)
    _within(s.log_probs, log_probs, tol + 2.0 ** -22 * log_probs.abs(), "log_probs")
    _within(s.entropy, entropy, 2 * tol * (1 + entropy), "entropy")
    order = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(s.top_ids, order)
    _within(s.top_log_probs, lp.gather(1, order), tol + 2.0 ** -22 * lp.gather(1, order).abs(), "top")
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    for gg, hh in ((g, h), (g, None), (None, h)):
        outs = [(o, d) for o, d in ((s.log_probs, gg), (s.entropy, hh)) if d is not None]
        dx, = torch.autograd.grad([o for o, _ in outs], x, [d for _, d in outs], retain_graph=True)
        zero = torch.zeros_like(g)
        want, size = _grad64(lp, entropy, ids, zero if gg is None else gg, zero if hh is None else hh)
        u = U if dtype == torch.bfloat16 else 2.0 ** -22
        _within(dx, want, u * want.abs() + (4 * tol * (1 + entropy[:, None]) + 2.0 ** -18) * size + 1e-30, "gradient")
    again = ops.token_log_probs(x, ids)                                  # without alternatives
    assert again.top_ids is None and torch.allclose(again.log_probs, s.log_probs, rtol=0, atol=2 * tol + 2.0 ** -21 * 100)


def test_token_log_probs_gradient_against_differences():
    ops = _ops()
    torch.manual_seed(21)
    x = (2 * torch.randn(4, 500, device="cuda")).requires_grad_()
    ids = torch.tensor([0, 499, -100, 77], device="cuda")
    g, h = torch.randn(4, device="cuda"), torch.randn(4, device="cuda")

    def f(t):
        s = ops.token_log_probs(t, ids)
        return (s.log_probs * g + s.entropy * h).sum()

    dx, = torch.autograd.grad(f(x), x)
    d = torch.randn_like(x)
    slope = (f(x.detach() + 1e-2 * d).double() - f(x.detach() - 1e-2 * d).double()).item() / 2e-2
    # values of about 7 to 2^-20 over a step of 2e-2, and the third derivative times 1e-4 / 6
    assert abs((dx * d).sum().item() - slope) <= 4 * 7 * 2.0 ** -19 / 2e-2 + 1e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_log_probs_of_masks_and_extremes(dtype):
    """-inf and the type's lowest value as masks, rows with nothing left, ties, ascending rows, one token that has it all, NaN."""
    ops = _ops()
    inf, low, V = math.inf, torch.finfo(dtype).min, 5000
    torch.manual_seed(23)
    x = torch.randn(9, V, device="cuda").to(dtype)
    x[0, ::2] = -inf
    x[1] = -inf
    x[2, 10:] = low
    x[3] = low
    x[4] = 1.5
    x[5] = torch.linspace(-8, 8, V, device="cuda").to(dtype)
    x[6, 4321] = 200.0
    x[7, 4999] = math.nan
    x[8, 0], x[8, 1], x[8, 2:] = 0.0, -0.0, -1.0
    x.requires_grad_()
    ids = torch.tensor([1, 3, 12, 7, 4999, 2500, 4321, 0, 5000], device="cuda")
    s = ops.token_log_probs(x, ids, top_k=32)
    want = ops.token_log_probs(x.detach().double().cpu(), ids.cpu(), top_k=32)
    tol = _log_tolerance(V)
    assert torch.equal(s.top_ids.cpu(), want.top_ids)
    for got, w in ((s.log_probs, want.log_probs), (s.entropy, want.entropy), (s.top_log_probs, want.top_log_probs)):
        got, w = got.double().cpu(), w
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got == -inf, w == -inf)
        ok = torch.isfinite(w) & (w.abs() < 1e30)
        assert ((got - w).abs()[ok] <= 2 * tol * (1 + w.abs()[ok])).all()
        far = torch.isfinite(w) & ~ok                    # a token at the lowest value: as far down as fp32 goes
        assert ((got / w)[far] - 1).abs().max() <= 1e-6 if far.any() else True
    keep = torch.tensor([0, 1, 2, 3, 4, 5, 6, 8], device="cuda")
    g = torch.ones(9, device="cuda")
    dx, = torch.autograd.grad((s.log_probs, s.entropy), x, (g, g))
    assert torch.isfinite(dx[keep]).all() and not dx[1].any() and not dx[0, ::2].any() and dx[7].isnan().any()
    _clean()


def test_token_log_probs_refusals_of_the_kernel_path():
    from himuon_b200._ext import ext
    x = torch.randn(4, 64, device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    lp, st = torch.empty(4, device="cuda"), torch.empty(4, 2, device="cuda")
    top, tid = torch.empty(4, 5, device="cuda"), torch.empty(4, 5, device="cuda", dtype=torch.int64)
    ok = (x, ids, lp, lp.clone(), st, top, tid, -100)
    ext().token_scores_fwd(*ok)
    for i, bad in [(0, x.half()), (0, x.t()), (0, x[:1].expand(4, 64)), (1, ids.int()), (1, ids[:3]), (2, lp[:3]), (3, lp.double()), (4, lp), (5, None), (6, tid[:, :4])]:
        with pytest.raises(RuntimeError, match="himuon"):
            ext().token_scores_fwd(*ok[:i], bad, *ok[i + 1:])
    grad = torch.empty_like(x)
    ok = (x, ids, lp, st, lp, lp, grad, -100)
    ext().token_scores_bwd(*ok)
    for i, bad in [(3, lp), (4, lp[:2]), (5, lp.double()), (6, grad[:2]), (6, grad.half()), (6, grad.t())]:
        with pytest.raises(RuntimeError, match="himuon"):
            ext().token_scores_bwd(*ok[:i], bad, *ok[i + 1:])


def _logit_error(h, w):
    """Largest error of a logit: fp32 sums of hidden / 16 steps, relative to the sum of the absolute products."""
    return (h.shape[1] / 16 + 4) * 2.0 ** -22 * (h.double().abs() @ w.double().abs().t()).max().item()


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 8, 1), (1, 128, 1000), (8, 256, 5003), (3, 72, 40000), (16, 128, 151936), (17, 200, 9000), (32, 640, 128256), (33, 128, 3001), (64, 256, 5000), (65, 256, 5000), (100, 64, 264), (129, 136, 777), (300, 640, 4096), (777, 128, 2050)])
def test_linear_token_log_probs(rows, hidden, vocab):
    ops = _ops()
    torch.manual_seed(rows + vocab)
    h = torch.randn(rows, hidden, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(vocab, hidden, device="cuda") * 2 / math.sqrt(hidden)).bfloat16().requires_grad_()
    ids = torch.randint(0, vocab, (rows,), device="cuda")
    ids[rows // 2] = -100 if rows > 2 else ids[rows // 2]
    s = ops.linear_token_log_probs(h, w, ids)
    g, e = torch.randn(rows, device="cuda"), 0.3 * torch.randn(rows, device="cuda")
    dh, dw = torch.autograd.grad((s.log_probs, s.entropy), (h, w), (g, e))
    _clean()
    hd, wd = h.detach().double(), w.detach().double()
    lp, log_probs, entropy = _scores64(hd @ wd.t(), ids)
    dl = _logit_error(h.detach(), w.detach())
    tol = _log_tolerance(vocab) + 2 * dl
    _within(s.log_probs, log_probs, tol + 2.0 ** -22 * log_probs.abs(), "log_probs")
    _within(s.entropy, entropy, 2 * tol * (1 + entropy), "entropy")
    dx, size = _grad64(lp, entropy, ids, g, e)
    bx = U * dx.abs() + (4 * tol * (1 + entropy[:, None]) + 2.0 ** -18) * size
    for got, want, bound, what in ((dh, dx @ wd, bx @ wd.abs(), "dh"), (dw, dx.t() @ hd, bx.t() @ hd.abs(), "dw")):
        _within(got, want, (1 + U) * bound + U * want.abs() + F * bound + 1e-30, what)


def test_linear_token_log_probs_in_chunks(monkeypatch):
    """Nothing of a row depends on the chunk that it is in; the weight's gradient is summed over the chunks.  A gradient from kept exponentials
    (the first backward pass) has theirs and one more rounding than one from the logits again (the second)."""
    ops = _ops()
    from himuon_b200.ops import scores

    torch.manual_seed(31)
    h = torch.randn(600, 128, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(1000, 128, device="cuda") * 0.2).bfloat16().requires_grad_()
    ids = torch.randint(0, 1000, (600,), device="cuda")
    g = torch.randn(600, device="cuda")

    def both():
        s = ops.linear_token_log_probs(h, w, ids)
        passes = [torch.autograd.grad((s.log_probs, s.entropy), (h, w), (g, g), retain_graph=True) for _ in range(2)]
        return (s.log_probs, s.entropy, *passes)

    lp, entropy, kept, again = both()
    monkeypatch.setattr(scores, "GRADIENT_VALUES", 256 * 1000)
    monkeypatch.setattr(scores, "LAUNCH_ROWS", 300)
    lp2, entropy2, *parts = both()
    assert torch.equal(lp, lp2) and torch.equal(entropy, entropy2)
    for dh, dw in parts:
        assert torch.equal(dh, again[0])
        # the same fp32 terms in another order, then one rounding
        assert ((again[1].float() - dw.float()).abs() <= 2 * U * dw.float().abs() + 1e-4).all()
    x = h.detach().double() @ w.detach().double().t()
    l, _, e = _scores64(x, ids)
    dx, size = _grad64(l, e, ids, g, g)
    bound = (2 * U) * dx.abs() + 2.0 ** -10 * size       # two roundings to bf16, fp16 exponentials (also of the log in the entropy's part)
    for i, other in ((0, w), (1, h)):
        b = bound @ other.detach().double().abs() if i == 0 else bound.t() @ other.detach().double().abs()
        assert ((kept[i].double() - again[i].double()).abs() <= b + U * again[i].double().abs() * 2).all()
    _clean()


def test_operators_under_a_checkpoint():
    """Recomputed, not kept: the same bits, and no logits' worth of memory between the passes."""
    from torch.utils.checkpoint import checkpoint

    ops = _ops()
    torch.manual_seed(43)
    layout, H, hd, vocab = ops.PackedLayout([150, 3, 60]), 2, 64, 5000
    x = torch.randn(213, 3 * H * hd, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(vocab, H * hd, device="cuda") * 0.1).bfloat16().requires_grad_()
    w2 = (torch.randn(H * hd, 64, device="cuda") * 0.1).requires_grad_()
    ids = torch.randint(0, vocab, (213,), device="cuda")

    def loss(x, w, w2):
        h = ops.packed_attention(*x.split(H * hd, 1), layout, H, H, hd)
        a = ops.linear_token_log_probs(h, w, ids)
        b = ops.token_log_probs(h.float() @ w2, ids % 64)
        return (a.log_probs + 0.1 * a.entropy + b.log_probs + 0.1 * b.entropy).sum()

    want = torch.autograd.grad(loss(x, w, w2), (x, w, w2))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = checkpoint(loss, x, w, w2, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < 213 * vocab, "what the forward pass kept is still there"
    got = torch.autograd.grad(out, (x, w, w2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _clean()


def test_linear_token_log_probs_of_a_long_vocabulary():
    """Few output tiles and a long inner dimension: the hidden states' gradient is cut along the vocabulary."""
    ops = _ops()
    from himuon_b200._ext import ext

    torch.manual_seed(35)
    for rows, hidden, vocab in [(200, 256, 40000), (40, 136, 50001), (5, 128, 30001)]:
        a = torch.randn(rows, (vocab + 7) // 8 * 8, device="cuda").bfloat16()[:, :vocab]
        b = torch.randn(vocab, hidden, device="cuda").bfloat16()
        out = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16)
        before = ops.launch_count()
        ext().long_product(a, b, out)
        assert ops.launch_count() - before >= 2, "one GEMM did it all: the test covers nothing"
        want = a.double() @ b.double()
        # an fp32 sum of vocab / 16 steps, then one rounding
        _within(out, want, U * want.abs() + (vocab / 16 + 64) * 2.0 ** -24 * (a.double().abs() @ b.double().abs()), "product")
    _clean()


def test_linear_token_log_probs_slices_and_partial_gradients():
    ops = _ops()
    torch.manual_seed(33)
    buf = torch.randn(50, 200, device="cuda").bfloat16()
    h, w = buf[:, 3:131].detach().requires_grad_(), torch.randn(300, 128, device="cuda").bfloat16()
    ids = torch.randint(0, 300, (50,), device="cuda")
    s = ops.linear_token_log_probs(h, w, ids)
    dh, = torch.autograd.grad(s.log_probs.sum(), h)
    lp, log_probs, entropy = _scores64(h.detach().double() @ w.double().t(), ids)
    tol = _log_tolerance(300) + 2 * _logit_error(h.detach(), w)
    _within(s.log_probs, log_probs, tol + 2.0 ** -22 * log_probs.abs(), "log_probs")
    one, zero = torch.ones(50, device="cuda"), torch.zeros(50, device="cuda")
    dx, size = _grad64(lp, entropy, ids, one, zero)
    bound = (U * dx.abs() + (4 * tol + 2.0 ** -18) * size) @ w.double().abs()
    _within(dh, dx @ w.double(), (1 + U + F) * bound + U * (dx @ w.double()).abs() + 1e-30, "dh")
    assert ops.linear_token_log_probs(h[:0], w, ids[:0]).log_probs.shape == (0,)
    with torch.no_grad():
        assert torch.equal(ops.linear_token_log_probs(h, w, ids).log_probs, s.log_probs)
    _clean()


# ------------------------------------------------------------------------------------------- together, in a model
@pytest.mark.parametrize("model_type,head_dim", [("qwen3", 128), ("llama", 64)])
def test_model_scores_of_a_packed_batch(model_type, head_dim):
    """Packed scores and their gradients on the kernels against the fp32 model on plain operators."""
    import copy

    ops = _ops()
    from himuon_b200.models import CausalLM, DecoderConfig

    torch.manual_seed(0)
    cfg = DecoderConfig(model_type=model_type, vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                        num_attention_heads=4, num_key_value_heads=2, head_dim=head_dim, rms_norm_eps=1e-6, rope_theta=10000.0,
                        tie_word_embeddings=model_type == "qwen3", max_position_embeddings=512)
    plain = CausalLM(cfg).cuda().float()
    fast = copy.deepcopy(plain).bfloat16()
    with torch.no_grad():
        for a, b in zip(plain.parameters(), fast.parameters()):
            a.copy_(b.float())
    lengths, pad = [200, 1, 0, 77, 130], 4
    ids = torch.randint(0, 2048, (1, sum(lengths) + pad), device="cuda")
    layout = ops.PackedLayout(lengths)
    advantage = torch.randn(ids.numel(), device="cuda")
    outs = []
    for model in (plain, fast):
        s = model.score(ids, layout)
        (-(s.log_probs * advantage).sum() / ids.numel() - 0.01 * s.entropy[: sum(lengths)].mean()).backward()
        outs.append((s, model(ids, labels=ids, layout=layout).loss.item()))
    _clean()
    (a, loss_a), (b, loss_b) = outs
    # bf16 activations through two layers, as in the equal-length model's test
    assert abs(loss_a - loss_b) < 3e-2
    assert (a.log_probs - b.log_probs).abs().mean() < 3e-2 and (a.entropy - b.entropy).abs().mean() < 3e-2
    for (n, p), q in zip(plain.named_parameters(), fast.parameters()):
        x, y = p.grad.flatten(), q.grad.float().flatten()
        assert torch.dot(x, y) / (x.norm() * y.norm() + 1e-12) > 0.99, n
        assert abs(y.norm() / (x.norm() + 1e-12) - 1) < 0.05, n


def test_linear_token_log_probs_repeats_its_bits():
    """Gradients whose products leave a last wave of tiles that is cut along the sum (2048 rows by 2560 columns: 80 tiles on 74 pairs)."""
    ops = _ops()
    torch.manual_seed(51)
    h = torch.randn(2048, 2560, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(9728, 2560, device="cuda") * 0.04).bfloat16().requires_grad_()
    ids = torch.randint(0, 9728, (2048,), device="cuda")
    g, seen = torch.randn(2048, device="cuda"), None
    for _ in range(5):
        s = ops.linear_token_log_probs(h, w, ids)
        got = (s.log_probs.detach(), s.entropy.detach(), *torch.autograd.grad((s.log_probs, s.entropy), (h, w), (g, g)))
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, got))
        seen = got
    _clean()


@pytest.mark.parametrize("rows,hidden,vocab", [(6144, 2560, 2304), (24576, 640, 1024)])
def test_linear_token_log_probs_in_chunks_repeats_its_bits(monkeypatch, rows, hidden, vocab):
    """The weight's gradient summed over three chunks of rows, with tiles that do not fill their last round (9 by 10 on 74 pairs) or
    are too few for one (4 by 3)."""
    ops = _ops()
    from himuon_b200.ops import scores

    monkeypatch.setattr(scores, "GRADIENT_VALUES", rows // 3 * vocab)
    torch.manual_seed(53)
    h = torch.randn(rows, hidden, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(vocab, hidden, device="cuda") * 0.04).bfloat16().requires_grad_()
    ids, g, seen = torch.randint(0, vocab, (rows,), device="cuda"), torch.randn(rows, device="cuda"), None
    for _ in range(6):
        got = torch.autograd.grad(ops.linear_token_log_probs(h, w, ids).log_probs, (h, w), g)
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, got))
        seen = got
    _clean()


# ------------------------------------------------------------------------------------------- transforms
def _calls(dtype=torch.bfloat16):
    """Each operator as a function of its first operand, with that operand and a direction; the results are tensors."""
    ops = _ops()
    torch.manual_seed(57)
    layout = ops.PackedLayout([5, 0, 9])
    k, v = (torch.randn(14, 64, device="cuda").to(dtype) for _ in range(2))
    w, ids = (torch.randn(40, 64, device="cuda") * 0.3).to(dtype), torch.randint(0, 40, (14,), device="cuda")
    fns = {"packed_attention": lambda t: (ops.packed_attention(t, k, v, layout, 2, 2, 32),),
           "token_log_probs": lambda t: ops.token_log_probs(t, ids, top_k=3)[:2],
           "linear_token_log_probs": lambda t: ops.linear_token_log_probs(t, w, ids)[:2]}
    return fns, torch.randn(14, 64, device="cuda").to(dtype), torch.randn(14, 64, device="cuda").to(dtype)


@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
@pytest.mark.parametrize("name", ["packed_attention", "token_log_probs", "linear_token_log_probs"])
def test_forward_mode_tangents_are_not_lost(name):
    """A dual tensor asks for no gradient and still has a derivative: that of a central difference, in 32 bits."""
    from torch.autograd import forward_ad

    fns, x, d = _calls(torch.float32)
    h = 1e-2
    slopes = [((a - b) / (2 * h)) for a, b in zip(fns[name](x + h * d), fns[name](x - h * d))]
    for dtype in (torch.float32, torch.bfloat16):
        fn, a, t = _calls(dtype)[0][name], x.to(dtype), d.to(dtype)
        with forward_ad.dual_level():
            duals = [forward_ad.unpack_dual(o) for o in fn(forward_ad.make_dual(a, t))]
        for (_, tangent), slope in zip(duals, slopes):
            assert tangent is not None
            # bf16: operands and result rounded; the difference itself is good to a third derivative times h^2 / 6
            assert (tangent.double() - slope.double()).norm() <= (0.05 if dtype == torch.bfloat16 else 1e-2) * slope.double().norm()
        if dtype == torch.bfloat16:
            _, tangents = torch.func.jvp(fn, (a,), (t,))
            assert all(torch.equal(u, o.tangent) for u, o in zip(tangents, duals))
    _clean()


@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
@pytest.mark.parametrize("name", ["packed_attention", "token_log_probs", "linear_token_log_probs"])
def test_operators_under_vmap(name):
    """A batch of calls at once returns what the calls return one by one."""
    fns, x, d = _calls()
    got = torch.vmap(fns[name])(torch.stack([x, d]))
    for i, a in enumerate((x, d)):
        for one, all_of in zip(fns[name](a), got):
            # the kernels and the plain formulation: bf16 roundings of values around 1, and of fp32 log probabilities of bf16 logits
            assert (one.double() - all_of[i].double()).abs().max() <= (8 * U if name == "packed_attention" else 1e-4)
    _clean()


@pytest.mark.filterwarnings("ignore:himuon_b200.ops")
def test_scores_under_vmap_over_ids_alone():
    ops = _ops()
    torch.manual_seed(59)
    x, h, w = torch.randn(6, 40, device="cuda"), torch.randn(6, 64, device="cuda").bfloat16(), torch.randn(40, 64, device="cuda").bfloat16()
    ids = torch.randint(0, 40, (3, 6), device="cuda")
    for fn in (lambda i: ops.token_log_probs(x, i).log_probs, lambda i: ops.linear_token_log_probs(h, w, i).log_probs):
        got = torch.vmap(fn)(ids)
        assert all((fn(i) - g).abs().max() <= 1e-4 for i, g in zip(ids, got))
    _clean()


def _peaked_head(rows=128, vocab=1000):
    """Hidden states that are unit vectors, so that a row's logits stand in a column of the weight and its logits' gradient in one of dw;
    within 64 neighbours they spread over 50 nats, as beside the token of a confident row, and the neighbours' maxima over 30."""
    torch.manual_seed(61)
    top = -30 * torch.rand(rows, (vocab + 63) // 64, device="cuda")
    top[:, 3] = 0
    x = top.repeat_interleave(64, 1)[:, :vocab] - 50 * torch.rand(rows, vocab, device="cuda")
    x.scatter_(1, torch.randint(3 * 64, 4 * 64, (rows, 1), device="cuda"), 0.0)
    return torch.eye(rows, device="cuda").bfloat16().requires_grad_(), x.t().contiguous().bfloat16().requires_grad_()


@pytest.mark.parametrize("with_entropy", [False, True])
def test_head_gradient_of_peaked_rows_at_any_size(with_entropy):
    """Each entry of the logits' gradient to its own size, from kept exponentials (the first backward pass) and from the logits
    again (the second): an optimizer that normalises entries sees the error of the small ones too."""
    ops = _ops()
    h, w = _peaked_head()
    ids, rows = torch.randint(0, w.shape[0], (h.shape[0],), device="cuda"), h.shape[0]
    g, e = 0.5 + torch.rand(rows, device="cuda"), (torch.rand(rows, device="cuda") if with_entropy else torch.zeros(rows, device="cuda"))
    s = ops.linear_token_log_probs(h, w, ids)
    lp, _, entropy = _scores64(w.detach().double().t(), ids)
    dx, size = _grad64(lp, entropy, ids, g, e)
    p = lp.exp()
    part = -p * (g.double() + e.double() * entropy)[:, None] - p * e.double()[:, None] * lp          # without the own token's g
    # kept exponentials to 2^-10 (and as much of their logarithm in the entropy's part), fp32 exponents of up to 80 to 2^-17, then one
    # rounding to bf16; what is below the normal numbers may be 0
    bound = 2.0 ** -10 * (part.abs() + p * e.double()[:, None]) + 2.0 ** -13 * size
    bound = bound + 2.0 ** -8 * (dx.abs() + bound) + 1e-37
    outs = (s.log_probs, s.entropy) if with_entropy else (s.log_probs,)
    for _ in range(2):
        dw, = torch.autograd.grad(outs, w, (g, e)[: len(outs)], retain_graph=True)
        _within(dw.t(), dx, bound, "gradient of the logits")
    _clean()


def test_operands_whose_rows_share_memory():
    """Expanded and overlapping rows are results of ordinary calls: one state scored against many candidates, keys that all documents share."""
    ops = _ops()
    torch.manual_seed(63)
    h, w = torch.randn(1, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(90, 64, device="cuda").bfloat16().requires_grad_()
    flat = torch.randn(64 + 8 * 69, device="cuda").bfloat16()
    ids = torch.randint(0, 90, (70,), device="cuda")
    for rows in (h.expand(70, 64), flat.as_strided((70, 64), (8, 1)).requires_grad_()):
        got = []
        for t in (rows, rows.contiguous()):
            s = ops.linear_token_log_probs(t, w, ids)
            got.append((s.log_probs, s.entropy, *torch.autograd.grad(s.log_probs.sum(), (rows, w))))
            with torch.no_grad():
                assert (ops.linear_token_log_probs(t, w, ids).log_probs - s.log_probs).abs().max() <= 1e-4
        assert all(torch.equal(a, b) for a, b in zip(*got))
    layout = ops.PackedLayout([40, 30])
    q, k, v = (torch.randn(n, 128, device="cuda").bfloat16().requires_grad_() for n in (70, 1, 1))
    got = []
    for kk, vv in ((k.expand(70, 128), v.expand(70, 128)), (k.repeat(70, 1), v.repeat(70, 1))):
        o = ops.packed_attention(q, kk, vv, layout, 2, 2, 64)
        with torch.no_grad():
            assert torch.equal(ops.packed_attention(q, kk, vv, layout, 2, 2, 64), o)
        got.append((o, *torch.autograd.grad(o, (q, kk, vv), torch.ones_like(o))))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    got = [ops.packed_attention(t, k.expand(70, 128), v.expand(70, 128), layout, 2, 2, 64) for t in (q[:1].expand(70, 128), q[:1].repeat(70, 1))]
    assert torch.equal(*got)
    _clean()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_log_probs_of_one_token_in_a_transposed_matrix(dtype):
    ops = _ops()
    x = torch.randn(1, 6, device="cuda").to(dtype).t().requires_grad_()
    assert x.stride() == (1, 6)
    s = ops.token_log_probs(x, torch.zeros(6, dtype=torch.int64, device="cuda"), top_k=1)
    assert not s.log_probs.any() and not s.entropy.any() and not s.top_ids.any()
    assert not torch.autograd.grad((s.log_probs.sum(), s.entropy.sum()), x)[0].any()
    _clean()


def test_an_odd_hidden_size_is_said_to_run_without_the_kernels():
    ops = _ops()
    ops._WARNED.discard(("linear_token_log_probs", "hidden size 63 (the kernels take multiples of 8)"))
    h, w = torch.randn(4, 63, device="cuda").bfloat16(), torch.randn(20, 63, device="cuda").bfloat16()
    with pytest.warns(UserWarning, match="linear_token_log_probs: hidden size 63"):
        ops.linear_token_log_probs(h, w, torch.zeros(4, dtype=torch.int64, device="cuda"))


def test_scores_of_a_head_take_no_more_scratch_than_their_parts(monkeypatch):
    """Three floats for each row and 128 tokens above 64 rows, for each 64 below; a last launch of a few rows fits in as well."""
    ops = _ops()
    from himuon_b200.ops import scores

    w, ids = torch.randn(60000, 64, device="cuda").bfloat16(), torch.zeros(1024, dtype=torch.int64, device="cuda")
    h = torch.randn(1024, 64, device="cuda").bfloat16()
    with torch.no_grad():
        for rows, per in ((1024, 128), (65, 128), (64, 64), (8, 64)):
            ops.linear_token_log_probs(h[:rows], w, ids[:rows])
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            ops.linear_token_log_probs(h[:rows], w, ids[:rows])
            # (two results, roundings of a block of memory, and the scratch of two tiles that the vocabulary ends in)
            assert torch.cuda.max_memory_allocated() - before <= 12 * rows * (60000 / per + 4) + 2 ** 16
        want = ops.linear_token_log_probs(h[:129], w, ids[:129])
        monkeypatch.setattr(scores, "LAUNCH_ROWS", 65)
        got = ops.linear_token_log_probs(h[:129], w, ids[:129])
        assert (got.log_probs - want.log_probs).abs().max() <= 1e-4 and torch.equal(got.log_probs[:65], want.log_probs[:65])
    _clean()


def test_head_gradients_replayed_twice_for_one_forward_pass():
    """Captured apart, the backward pass runs as often as it is replayed: it must not use up what the forward pass kept."""
    ops = _ops()
    torch.manual_seed(67)
    h, w = torch.randn(100, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(500, 64, device="cuda").bfloat16().requires_grad_()
    ids, g = torch.randint(0, 500, (100,), device="cuda"), torch.randn(100, device="cuda")

    def scores(a, b):
        return ops.linear_token_log_probs(a, b, ids).log_probs

    want = torch.autograd.grad(scores(h, w), (h, w), g)
    graphed = torch.cuda.make_graphed_callables(scores, (h, w))
    out = graphed(h, w)
    for _ in range(3):
        got = torch.autograd.grad(out, (h, w), g, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    _clean()


def test_head_gradients_replayed_after_an_eager_pass_on_the_same_graph():
    ops = _ops()
    torch.manual_seed(69)
    h, w = torch.randn(100, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(500, 64, device="cuda").bfloat16().requires_grad_()
    ids, g = torch.randint(0, 500, (100,), device="cuda"), torch.randn(100, device="cuda")
    want = torch.autograd.grad(ops.linear_token_log_probs(h, w, ids).log_probs, (h, w), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        out = ops.linear_token_log_probs(h, w, ids).log_probs
        with torch.cuda.graph(graph, stream=side):
            captured = torch.autograd.grad(out, (h, w), g, retain_graph=True)
        eager = torch.autograd.grad(out, (h, w), g, retain_graph=True)
        graph.replay()
    side.synchronize()
    for got in (eager, captured):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    _clean()


def test_packed_attention_refuses_more_items_than_its_turns_count():
    """Blocks look up to two turns past the last (tile, head) item, whose number has to fit in 32 bits; nothing is launched."""
    from himuon_b200._ext import ext

    tiles, Hq = 1024, 2 ** 21 - 16
    assert 2 ** 31 - 2 ** 16 <= tiles * Hq < 2 ** 31
    plan = torch.zeros(2 * tiles, 4, device="cuda", dtype=torch.int32)
    q, k = torch.zeros(1, Hq * 8, device="cuda", dtype=torch.bfloat16), torch.zeros(1, 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="too many tiles"):
        ext().packed_attn_fwd(plan, tiles, 1, q, k, k, torch.empty_like(q), None, None, Hq, 1, 0.1)
    _clean()


def _certain_bounds(q, k, v, do, lengths, Hq, Hkv, hd, scale):
    """Results in 64 bits and bounds that hold for rows with one weight near 1 as well.

    With a = 2^-8 (a weight rounded to bf16), a row's weights are p_j (1 + e_j) over their sum, so that O is off by sum p_j e_j (v_j - o)
    and delta by sum p_j e_j (dP_j - delta), at most a sum |dS|.  Scores are off by the tensor core's fp32 sums, which move p alike.  Beside
    that delta has O to 2^-16, and fp32 sums of hd terms."""
    T, G, a = q.shape[0], Hq // Hkv, U
    step = (hd / 16 + 4) * 2.0 ** -22                            # of a sum of hd products, relative to their absolute values
    q, k, v, do = (_heads(t, hd) for t in (q, k, v, do))
    out = {n: torch.zeros(h, T, hd, dtype=torch.float64, device=q.device) for n, h in
           (("o", Hq), ("dq", Hq), ("dk", Hkv), ("bo", Hq), ("bdq", Hq), ("bdk", Hkv))}
    largest = torch.zeros(Hq, T, dtype=torch.float64, device=q.device)
    first = 0
    for n in lengths:
        c = slice(first, first + n)
        first += n
        if n == 0:
            continue
        kk, vv = (t[:, c].repeat_interleave(G, 0) for t in (k, v))
        qq, g = q[:, c], do[:, c]
        s = scale * qq @ kk.transpose(1, 2)
        p = torch.softmax(s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf), -1)
        o = p @ vv
        e = 2 * (step * scale * (qq.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) + 2.0 ** -22 * (2 + s.abs().amax(-1, keepdim=True)))
        dp = g @ vv.transpose(1, 2)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        size, osize = g.abs() @ vv.abs().transpose(1, 2), (g.abs() * o.abs()).sum(-1, keepdim=True)
        off = (a + e) * ds.abs().sum(-1, keepdim=True) + (2.0 ** -16 + (hd + 40) * 2.0 ** -23) * osize
        bds = (2 * a + 2 * e) * ds.abs() + p * (off + step * size)
        far = torch.stack([(p[h][..., None] * (vv[h][None] - o[h][:, None]).abs()).sum(1) for h in range(Hq)])
        bo = (a + e) * far + 2.0 ** -20 * (p @ vv.abs())
        per = {"o": (o, bo), "dq": (scale * ds @ kk, scale * bds @ kk.abs()), "dk": (scale * ds.transpose(1, 2) @ qq, scale * bds.transpose(1, 2) @ qq.abs())}
        for name, (val, bound) in per.items():
            if name == "dk":
                val, bound = (t.view(Hkv, G, n, hd).sum(1) for t in (val, bound))
            out[name][:, c] = val
            out["b" + name][:, c] = bound * (1 + 2.0 ** -8) + a * val.abs() * (1 + 2.0 ** -6) + 1e-30
        largest[:, c] = p.amax(-1)
    return {n: _flat(t) for n, t in out.items()}, largest


@pytest.mark.parametrize("Hq,Hkv,hd", SHAPES)
@pytest.mark.parametrize("lengths", [[2] * 60 + [1, 64, 65], [300, 129], [700]])
def test_gradients_of_nearly_certain_rows_of_any_head_and_length(Hq, Hkv, hd, lengths):
    """Scores that spread by 6, so that many rows have one weight near 1, of a key that the running maximum may have met late."""
    ops = _ops()
    torch.manual_seed(71 + hd)
    T, scale = sum(lengths), 6 / math.sqrt(hd)
    q, k, v = (torch.randn(T, h * hd, device="cuda").bfloat16().requires_grad_() for h in (Hq, Hkv, Hkv))
    do = torch.randn(T, Hq * hd, device="cuda").bfloat16()
    o = ops.packed_attention(q, k, v, ops.PackedLayout(lengths), Hq, Hkv, hd, scale=scale)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want, largest = _certain_bounds(q, k, v, do, lengths, Hq, Hkv, hd, scale)
    assert ((largest < 1) & (largest > 0.99)).sum() > 20
    for name, got in zip(("o", "dq", "dk"), (o, *grads)):
        _within(got, want[name], want["b" + name], name)
    with torch.no_grad():
        _within(ops.packed_attention(q, k, v, ops.PackedLayout(lengths), Hq, Hkv, hd, scale=scale), want["o"], want["bo"], "o without a graph")
    _clean()


@pytest.mark.parametrize("lengths,rows", [([], 0), ([0, 0], 0), ([], 5), ([0], 5)])
def test_a_batch_without_tokens_on_the_gpu(lengths, rows):
    ops = _ops()
    q, k, v = (torch.randn(rows, n * 64, device="cuda").bfloat16().requires_grad_() for n in (4, 2, 2))
    layout = ops.PackedLayout(lengths)
    o = ops.packed_attention(q, k, v, layout, 4, 2, 64)
    grads = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
    assert o.shape == q.shape and not o.any()
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))
    with torch.no_grad():
        assert not ops.packed_attention(q, k, v, layout, 4, 2, 64).any()
    h, w, ids = torch.randn(0, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(9, 64, device="cuda").bfloat16().requires_grad_(), torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.randn(0, 9, device="cuda", requires_grad=True)
    dh, dw = torch.autograd.grad(ops.linear_token_log_probs(h, w, ids).log_probs.sum(), (h, w))
    dx, = torch.autograd.grad(ops.token_log_probs(x, ids, top_k=2).entropy.sum(), x)
    assert dh.shape == (0, 64) and dw.shape == (9, 64) and not dw.any() and dx.shape == (0, 9)
    _clean()


def test_token_log_probs_fp32_gradient_over_several_blocks_from_strided_gradients():
    ops = _ops()
    torch.manual_seed(73)
    rows, vocab = 5, 40001
    x = (3 * torch.randn(rows, vocab + 3, device="cuda"))[:, 3:].requires_grad_()
    ids = torch.tensor([0, 40000, -100, 4096, 16383], device="cuda")
    both = torch.randn(rows, 2, device="cuda")
    s = ops.token_log_probs(x, ids)
    dx, = torch.autograd.grad((s.log_probs, s.entropy), x, (both[:, 0], both[:, 1]))
    lp, _, entropy = _scores64(x.detach(), ids)
    want, size = _grad64(lp, entropy, ids, both[:, 0], both[:, 1])
    tol = _log_tolerance(vocab)
    _within(dx, want, 2.0 ** -22 * want.abs() + (4 * tol * (1 + entropy[:, None]) + 2.0 ** -18) * size + 1e-30, "gradient")
    _clean()


def test_two_threads_on_one_retained_graph():
    """Each gets a gradient that a single caller gets: from what was kept, or from the logits again."""
    import threading

    ops = _ops()
    torch.manual_seed(75)
    h, w = torch.randn(300, 128, device="cuda").bfloat16().requires_grad_(), torch.randn(2000, 128, device="cuda").bfloat16().requires_grad_()
    ids, g = torch.randint(0, 2000, (300,), device="cuda"), torch.randn(300, device="cuda")

    def call():
        return ops.linear_token_log_probs(h, w, ids).log_probs

    out = call()
    one_by_one = [torch.autograd.grad(out, (h, w), g, retain_graph=True) for _ in range(2)]
    for _ in range(10):
        out, got = call(), []
        threads = [threading.Thread(target=lambda: got.append(torch.autograd.grad(out, (h, w), g, retain_graph=True))) for _ in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        kinds = sorted(next(i for i, want in enumerate(one_by_one) if all(torch.equal(a, b) for a, b in zip(x, want))) for x in got)
        assert kinds == [0, 1]
    _clean()


@pytest.mark.parametrize("rows", [301, 364, 365, 640, 664])
def test_a_row_of_the_head_does_not_depend_on_its_launch(monkeypatch, rows):
    """Launches of 300 rows and one, with a gradient and without: the same bits, also where a few rows are left for the last launch."""
    ops = _ops()
    from himuon_b200.ops import scores

    torch.manual_seed(77)
    h, w = torch.randn(rows, 128, device="cuda").bfloat16(), (torch.randn(3000, 128, device="cuda") * 0.2).bfloat16()
    ids = torch.randint(0, 3000, (rows,), device="cuda")
    want = ops.linear_token_log_probs(h, w, ids)
    monkeypatch.setattr(scores, "LAUNCH_ROWS", 300)
    for t in (h, h.clone().requires_grad_()):
        got = ops.linear_token_log_probs(t, w, ids)
        assert torch.equal(got.log_probs, want.log_probs) and torch.equal(got.entropy, want.entropy)
    _clean()


@pytest.mark.parametrize("rows", [40, 200])
@pytest.mark.parametrize("hidden", [640, 2560, 8192])
def test_scores_of_a_long_hidden_size_have_no_systematic_error(rows, hidden):
    """The tensor core cuts its sums off toward 0: logits of 2560 elements come out 2.3e-6 too small, all of them, which shows in the entropy.

    What is left after the common part has been put back is at most 2.5e-10 of a logit for each element (7.5e-10 is put back, 1e-9 has
    been measured); an entropy changes by the variance of the logits, 4 here, times that.  Beside it single errors of the same size for each element,
    whose mean over the distribution goes with 1 / sqrt of the number of likely tokens, and the sums' 2e-7."""
    ops = _ops()
    torch.manual_seed(79)
    h, w = torch.randn(rows, hidden, device="cuda").bfloat16(), (torch.randn(8192, hidden, device="cuda") * 2 / math.sqrt(hidden)).bfloat16()
    ids = torch.randint(0, 8192, (rows,), device="cuda")
    _, log_probs, entropy = _scores64(h.double() @ w.double().t(), ids)
    for t in (h, h.clone().requires_grad_()):
        s = ops.linear_token_log_probs(t, w, ids)
        off = (s.entropy.double() - entropy).norm() / entropy.norm()
        assert off <= 4 * 2.5e-10 * hidden / entropy.mean() + 4 * 5e-10 * hidden / 30 / entropy.mean() + 2e-7, off
        # the slope of log probabilities against the right ones, whose spread is 2: as much of a logit, and 40 rows' mean of single errors
        slope = ((s.log_probs.double() - log_probs) * (log_probs - log_probs.mean())).sum() / (log_probs - log_probs.mean()).pow(2).sum()
        assert slope.abs() <= 2.5e-10 * hidden + 3 * 6e-10 * hidden / math.sqrt(rows) + 2e-7, slope
    _clean()
