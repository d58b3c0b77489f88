"""Packed documents and token scores off-GPU: the layout's tables, the plain implementations against independent ones in 64
bits, their gradients against differences, and what the operators refuse."""

import math

import pytest
import torch

from himuon_b200 import ops
from himuon_b200.ops import reference as ref
from himuon_b200.ops.packed import TILE

LENGTHS = [[], [0], [1], [0, 0, 3], [128], [129, 0, 127], [5, 1, 0, 300, 64, 65]]


@pytest.mark.parametrize("lengths", LENGTHS)
def test_layout_lists_every_tile_once_and_heaviest_first(lengths):
    layout = ops.PackedLayout(lengths, device="cpu")
    assert layout.lengths == tuple(lengths) and layout.tokens == sum(lengths)
    plan = layout.plan
    want, first = [], 0
    for n in lengths:
        want += [(first, n, i) for i in range(-(-n // TILE))]
        first += n
    want = [(*t, slot) for slot, t in enumerate(want)]
    pairs = [t for t in want if t[2] % 2 == 0]
    assert plan.dtype == torch.int32 and layout.tiles == len(want) and plan.shape == (2 * len(want) + len(pairs), 4)
    rows = [tuple(t) for t in plan.tolist()]
    by_keys, by_queries, by_both = rows[: len(want)], rows[len(want): 2 * len(want)], rows[2 * len(want):]
    for order, all_of in ((by_keys, want), (by_queries, want), (by_both, pairs)):
        assert sorted(order, key=lambda t: t[3]) == all_of

    def keys(n, i):
        return min((i + 1) * TILE, n) if i * TILE < n else 0

    for work in ([keys(n, i) for _, n, i, _ in by_keys], [n - i * TILE for _, n, i, _ in by_queries], [keys(n, i) + keys(n, i + 1) for _, n, i, _ in by_both]):
        assert work == sorted(work, reverse=True)


def test_layout_positions_next_ids_and_rope_rows():
    layout = ops.PackedLayout(torch.tensor([3, 0, 1, 2], dtype=torch.int32), device="cpu")
    assert layout.positions(8).tolist() == [0, 1, 2, 0, 0, 1, 0, 0]
    assert layout.has_next().tolist() == [True, True, False, False, True, False]
    ids = torch.arange(10, 18)
    assert layout.next_ids(ids).tolist() == [11, 12, -100, -100, 15, -100, -100, -100]
    assert layout.next_ids(ids, ignore_index=7).tolist()[2] == 7
    table = ref.rope_tables(4, 8, 10000.0)
    rows = layout.rope_table(table, 7)
    assert torch.equal(rows, table[[0, 1, 2, 0, 0, 1, 0]])
    with pytest.raises(RuntimeError, match="positions"):
        layout.rope_table(table[:2])
    with pytest.raises(RuntimeError, match="rows"):
        layout.positions(5)


@pytest.mark.parametrize("lengths", [[-1], [1.5], ["a"], [2 ** 30], torch.ones(2), torch.ones(2, 2, dtype=torch.int64), torch.ones(2, dtype=torch.bool)])
def test_layout_refuses_lengths_that_are_none(lengths):
    with pytest.raises(RuntimeError, match="PackedLayout"):
        ops.PackedLayout(lengths, device="cpu")


def _masked_attention(q, k, v, lengths, Hq, Hkv, hd, scale):
    """One softmax over all rows, 64 bits, every other document and the future masked."""
    T, n = q.shape[0], sum(lengths)
    doc = torch.cat([torch.full((m,), i) for i, m in enumerate(lengths)] + [torch.full((T - n,), -1)])
    at = torch.arange(T)
    seen = (doc[:, None] == doc[None]) & (doc[:, None] >= 0) & (at[:, None] >= at[None])
    q, k, v = (t.view(T, -1, hd).transpose(0, 1) for t in (q, k, v))
    k, v = (t.repeat_interleave(Hq // Hkv, 0) for t in (k, v))
    e = torch.exp(scale * (q @ k.transpose(1, 2))) * seen
    return (e @ v / e.sum(-1, keepdim=True).clamp(min=1e-300)).transpose(0, 1).reshape(T, Hq * hd)


@pytest.mark.parametrize("lengths", [[1], [0, 0, 3], [5, 1, 0, 30]])
@pytest.mark.parametrize("pad", [0, 3])
def test_plain_packed_attention_is_masked_attention(lengths, pad):
    torch.manual_seed(0)
    Hq, Hkv, hd, T = 4, 2, 6, sum(lengths) + pad
    q, k, v = (torch.randn(T, h * hd, dtype=torch.float64, requires_grad=True) for h in (Hq, Hkv, Hkv))
    layout = ops.PackedLayout(lengths, device="cpu")
    o = ops.packed_attention(q, k, v, layout, Hq, Hkv, hd, scale=0.3)
    want = _masked_attention(q, k, v, lengths, Hq, Hkv, hd, 0.3)
    assert torch.allclose(o, want, rtol=1e-12, atol=1e-12) and not o[sum(lengths):].any()
    g = torch.randn_like(o)
    for a, b in zip(torch.autograd.grad(o, (q, k, v), g), torch.autograd.grad(want, (q, k, v), g)):
        assert torch.allclose(a, b, rtol=1e-10, atol=1e-12)
    if T < 12:
        assert torch.autograd.gradcheck(lambda *t: ops.packed_attention(*t, layout, Hq, Hkv, hd), (q, k, v))


def test_packed_attention_of_no_tokens():
    layout = ops.PackedLayout([0], device="cpu")
    for rows in (0, 4):
        q = torch.randn(rows, 16, requires_grad=True)
        o = ops.packed_attention(q, q.detach(), q.detach(), layout, 2, 2, 8)
        assert o.shape == (rows, 16) and not o.any()
        o.sum().backward()
        assert not q.grad.any()


def test_an_empty_batch_has_gradients():
    q, k, v = (torch.randn(3, 2 * 8, requires_grad=True) for _ in range(3))
    out = ops.packed_attention(q, k, v, ops.PackedLayout([0, 0], device="cpu"), 2, 2, 8)
    grads = torch.autograd.grad(out.sum(), (q, k, v))
    assert not out.any() and all(not g.any() for g in grads)


def test_packed_attention_refuses():
    layout = ops.PackedLayout([3], device="cpu")
    q, kv = torch.randn(3, 32), torch.randn(3, 16)
    ok = ops.packed_attention(q, kv, kv, layout, 4, 2, 8)
    assert ok.shape == q.shape
    bad = [
        ((q, kv, kv, [3], 4, 2, 8), {}),                       # no layout
        ((q, kv, kv, layout, 3, 2, 8), {}),                    # heads that do not group
        ((q, kv, kv, layout, 0, 2, 8), {}),
        ((q, kv, kv, layout, 4, 2, 16), {}),                   # widths
        ((q, kv, q, layout, 4, 2, 8), {}),
        ((q[:2], kv[:2], kv[:2], layout, 4, 2, 8), {}),        # fewer rows than tokens
        ((q, kv[:2], kv, layout, 4, 2, 8), {}),
        ((q, kv.double(), kv, layout, 4, 2, 8), {}),           # types
        ((q[0], kv, kv, layout, 4, 2, 8), {}),
        ((q, kv, kv, layout, 4, 2, 8), {"scale": 0.0}),
        ((q, kv, kv, layout, 4, 2, 8), {"scale": -1.0}),
        ((q, kv, kv, layout, 4, 2, 8), {"scale": math.nan}),
    ]
    for args, kw in bad:
        with pytest.raises(RuntimeError, match="himuon_b200"):
            ops.packed_attention(*args, **kw)


# ------------------------------------------------------------------------------------------- scores
def test_plain_token_log_probs_matches_log_softmax():
    torch.manual_seed(1)
    x = (3 * torch.randn(6, 33, dtype=torch.float64)).requires_grad_()
    ids = torch.tensor([0, 32, -100, 5, 5, 7])
    s = ops.token_log_probs(x, ids, top_k=4)
    lp = torch.log_softmax(x, -1)
    want = lp.gather(1, ids.clamp(min=0)[:, None])[:, 0] * (ids >= 0)
    assert torch.allclose(s.log_probs, want) and torch.allclose(s.entropy, -(lp.exp() * lp).sum(-1))
    top = torch.topk(lp, 4)
    assert torch.equal(s.top_ids, top.indices) and torch.allclose(s.top_log_probs, top.values) and not s.top_log_probs.requires_grad
    assert torch.autograd.gradcheck(lambda t: ops.token_log_probs(t, ids)[:2], (x,))
    h, w = torch.randn(6, 5, dtype=torch.float64, requires_grad=True), torch.randn(33, 5, dtype=torch.float64, requires_grad=True)
    a, b = ops.linear_token_log_probs(h, w, ids), ops.token_log_probs(h @ w.t(), ids)
    assert torch.allclose(a.log_probs, b.log_probs) and torch.allclose(a.entropy, b.entropy) and a.top_ids is None
    assert torch.autograd.gradcheck(lambda p, q: ops.linear_token_log_probs(p, q, ids)[:2], (h, w))


def test_plain_token_log_probs_of_masks_ties_and_bad_ids():
    inf = math.inf
    x = torch.tensor([[-inf, 1.0, 1.0, -inf], [-inf] * 4, [2.0, 2.0, 2.0, 2.0], [0.0, -0.0, 1.0, -inf]], requires_grad=True)
    s = ops.token_log_probs(x, torch.tensor([1, 2, 9, 3]), top_k=3)
    ln2 = math.log(2.0)
    assert torch.allclose(s.log_probs[:1], torch.tensor([-ln2])) and s.log_probs[1] == -inf and s.log_probs[2].isnan() and s.log_probs[3] == -inf
    assert torch.allclose(s.entropy[:3], torch.tensor([ln2, 0.0, 2 * ln2]))
    assert s.top_ids.tolist() == [[1, 2, 0], [0, 1, 2], [0, 1, 2], [2, 0, 1]]
    gx, = torch.autograd.grad(s.entropy.sum() + s.log_probs[:2].sum(), x)
    assert torch.isfinite(gx).all() and not gx[1].any() and gx[0, 0] == 0


def test_token_log_probs_refuses():
    x, ids = torch.randn(3, 40), torch.zeros(3, dtype=torch.int64)
    for args in [(x[0], ids), (x.long(), ids), (x, ids.int()), (x, ids[:2]), (x, ids[:, None]), (x, ids, 33), (x, ids, -1), (x[:, :4], ids, 5), (x[:, :0], ids)]:
        with pytest.raises(RuntimeError, match="token_log_probs"):
            ops.token_log_probs(*args)
    h, w = torch.randn(3, 8), torch.randn(40, 8)
    for args in [(h[0], w, ids), (h, w[:, :4], ids), (h, w.double(), ids), (h, w, ids[:1]), (h, w[:0], ids)]:
        with pytest.raises(RuntimeError, match="token_log_probs"):
            ops.linear_token_log_probs(*args)
    s = ops.token_log_probs(x[:0], ids[:0], top_k=2)
    assert s.log_probs.shape == (0,) and s.top_ids.shape == (0, 2)


# ------------------------------------------------------------------------------------------- a model's packed batches
def _model(model_type="qwen3"):
    from himuon_b200.models import CausalLM, DecoderConfig

    torch.manual_seed(0)
    return CausalLM(DecoderConfig(model_type=model_type, vocab_size=64, hidden_size=32, intermediate_size=64, num_hidden_layers=2,
                                  num_attention_heads=4, num_key_value_heads=2, head_dim=16, rms_norm_eps=1e-6, rope_theta=1e4,
                                  tie_word_embeddings=model_type == "qwen3", max_position_embeddings=64))


@pytest.mark.parametrize("model_type", ["qwen3", "llama"])
@pytest.mark.parametrize("checkpointing", [False, True])
def test_a_packed_batch_is_its_documents_one_by_one(model_type, checkpointing):
    model = _model(model_type).train()
    if checkpointing:
        model.gradient_checkpointing_enable()
    lengths, pad = [5, 0, 1, 9], 3
    ids = torch.randint(0, 64, (1, sum(lengths) + pad))
    layout = ops.PackedLayout(lengths, device="cpu")
    out = model(ids, labels=ids, layout=layout, return_logits=True)
    score = model.score(ids, layout)
    out.loss.backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    total, count, first = 0.0, 0, 0
    for n in lengths:
        part = ids[:, first: first + n]
        if n:
            one = model(part, labels=part, return_logits=True)
            assert torch.allclose(out.logits[:, first: first + n], one.logits, atol=1e-5)
        if n > 1:
            total, count = total + one.loss * (n - 1), count + n - 1
            lp = torch.log_softmax(one.logits[0, :-1].float(), -1)
            assert torch.allclose(score.log_probs[first: first + n - 1], lp.gather(1, part[0, 1:, None])[:, 0], atol=1e-5)
            assert torch.allclose(score.entropy[first: first + n - 1], -(lp.exp() * lp).sum(-1), atol=1e-5)
        if n:
            assert score.log_probs[first + n - 1] == 0
        first += n
    assert not score.log_probs[first:].any()
    assert torch.allclose(out.loss, total / count, atol=1e-6)
    (total / count).backward()
    for n, p in model.named_parameters():
        assert torch.allclose(grads[n], p.grad, atol=1e-6), n


def test_scores_of_a_model_train_it():
    """The gradient of the mean negative log probability is that of the loss."""
    model = _model()
    ids = torch.randint(0, 64, (1, 20))
    layout = ops.PackedLayout([12, 8], device="cpu")
    model(ids, labels=ids, layout=layout).loss.backward()
    want = [p.grad.clone() for p in model.parameters()]
    model.zero_grad()
    (-model.score(ids, layout).log_probs.sum() / 18).backward()
    for a, p in zip(want, model.parameters()):
        assert torch.allclose(a, p.grad, atol=1e-6)


def test_packed_attention_has_forward_mode_tangents_and_takes_vmap():
    torch.manual_seed(5)
    layout = ops.PackedLayout([3, 0, 6], device="cpu")
    q, k, v, d = (torch.randn(10, 16, dtype=torch.float64) for _ in range(4))

    def f(t):
        return ops.packed_attention(t, k, v, layout, 2, 2, 8)

    _, tangent = torch.func.jvp(f, (q,), (d,))
    slope = (f(q + 1e-4 * d) - f(q - 1e-4 * d)) / 2e-4
    assert torch.allclose(tangent, slope, rtol=1e-6, atol=1e-8)
    assert torch.allclose(torch.vmap(f)(torch.stack([q, d])), torch.stack([f(q), f(d)]))


def test_a_model_keeps_few_rotary_tables_for_many_longest_documents():
    model = _model()
    with torch.no_grad():
        for n in range(1, 60):
            ids = torch.randint(0, 64, (1, n + 2))
            model.score(ids, ops.PackedLayout([2, n], device="cpu"))
    assert len(model._rope_cache) <= 6                     # 2, 4, ... 64 positions
    assert sum(t.shape[0] for t in model._rope_cache.values()) <= 4 * 59
