"""Workloads of the operators for packed documents and token scores: attention over documents of different lengths packed
into one row of tokens, and the log probability of given tokens with the entropy and the likeliest alternatives, from logits
and straight from hidden states and the head's weight.

``listed()`` names the cases, ``draw(rng)`` makes one more of the same ranges, ``prepare(case, seed)`` makes what a program has
in hand before a call, ``run(state)`` is one call (with its gradients in the training cases) and ``work(case)`` the bytes and
operations that it cannot do without.  With ``own`` unset ``run`` computes the same in elementary torch operations in 32 bits;
``exact(case, seed)`` computes it in 64 bits.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
IGNORE = -100


# ------------------------------------------------------------------------------------------- cases
def _attend(name, tokens, docs, pad, heads, kv_heads, head_dim, train):
    return {"name": name, "kind": "attend", "tokens": tokens, "docs": docs, "pad": pad, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "train": train}


def _score(name, rows, vocab, dtype, top_k, masked, train):
    return {"name": name, "kind": "score", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k, "masked": masked,
            "train": train}


def _head(name, rows, hidden, vocab, train):
    return {"name": name, "kind": "head", "rows": rows, "hidden": hidden, "vocab": vocab, "train": train}


def listed():
    return [
        # a dozen short questions through a tiny model, padded to a multiple of 64 rows: what one call costs at least
        _attend("attend short questions", 300, 12, 20, 4, 2, 32, False),
        # a micro-batch of ragged documents of the 220M model, heads of 64, no grouping
        _attend("attend 220m train", 4071, 9, 25, 10, 10, 64, True),
        # a packed micro-batch of 16 heads over 8, most documents short
        _attend("attend 0.6b train", 8192, 24, 0, 16, 8, 128, True),
        # one document that fills the row, 32 heads over 8: nothing is masked but the future
        _attend("attend one document", 8192, 1, 0, 32, 8, 128, True),
        # scoring of a few long documents, forward only
        _attend("attend long scoring", 16384, 5, 0, 16, 8, 128, False),
        # the next token of four requests, vocabulary masked by a grammar, with twenty alternatives
        _score("score next token", 4, 151936, "fp32", 20, True, False),
        # an odd vocabulary: no row but the first starts on a 16-byte boundary
        _score("score odd vocabulary", 333, 32003, "bf16", 5, False, False),
        # evaluation of a batch with eight alternatives for each token
        _score("score evaluation", 1024, 128256, "bf16", 8, False, False),
        # policy gradient with an entropy bonus on logits that the program already has
        _score("score train", 2048, 151936, "bf16", 0, False, True),
        # scores of the newest token of eight sequences: the head's weight is read once
        _head("head newest tokens", 8, 1024, 151936, False),
        # a short ragged micro-batch of the 220M model
        _head("head 220m train", 777, 640, 128256, True),
        # a whole micro-batch of the 4B model
        _head("head 4b train", 8192, 2560, 151936, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _draw(rng):
    kind = rng.choice(("attend", "score", "head"))
    train = rng.random() < 0.5
    if kind == "attend":
        # (heads, kv_heads, head_dim) of the decoder configurations and of the tiny ones
        heads, kv_heads, head_dim = rng.choice(((4, 2, 32), (10, 10, 64), (16, 8, 128), (32, 8, 128), (32, 8, 64), (24, 8, 128)))
        tokens = _log_int(rng, 64, 8192)
        docs = _log_int(rng, 1, max(1, tokens // 16))
        case = _attend("", tokens, docs, rng.choice((0, 0, rng.randrange(1, 100))), heads, kv_heads, head_dim, train)
    elif kind == "score":
        vocab = rng.choice((1024, 32000, 128256, 151936, rng.randrange(1000, 152000)))
        case = _score("", _log_int(rng, 1, 2048), vocab, rng.choice(("bf16", "fp32")), 0 if train else rng.choice((0, 1, 5, 8, 20)),
                      rng.random() < 0.3, train)
    else:
        hidden = rng.choice((128, 640, 1024, 2048, 2560))
        case = _head("", _log_int(rng, 1, 8192), hidden, rng.choice((1024, 32000, 128256, 151936)), train)
    del case["name"]
    return case


def _lengths(case):
    """The documents' lengths: a few long ones, many short ones, some empty; the same for every seed."""
    rng = random.Random(1000003 * case["docs"] + case["tokens"])
    weights = [rng.random() ** 3 for _ in range(case["docs"])]
    total, at, cuts = sum(weights), 0.0, [0]
    for w in weights:
        at += w
        cuts.append(int(round(case["tokens"] * at / total)))
    cuts[-1] = case["tokens"]
    return [b - a for a, b in zip(cuts, cuts[1:])]


# ------------------------------------------------------------------------------------------- inputs
def _ids(gen, rows, vocab, masked=None):
    ids = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
    if masked is not None:                        # a grammar allows the token that was taken
        ids = ids - ids % 8
    skip = torch.rand(rows, generator=gen, device=DEVICE) < 0.1
    return torch.where(skip, torch.full_like(ids, IGNORE), ids)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "attend":
        rows = case["tokens"] + case["pad"]

        def mat(heads):
            return torch.randn(rows, heads * case["head_dim"], generator=gen, device=DEVICE).bfloat16()

        lengths = _lengths(case)
        state.update(q=mat(case["heads"]), k=mat(case["kv_heads"]), v=mat(case["kv_heads"]), lengths=lengths)
        if case["train"]:
            state["do"] = mat(case["heads"])
            for name in "qkv":
                state[name].requires_grad_()
        if own:                                   # made once for a batch; every layer of the model uses it
            from himuon_b200 import ops
            state["layout"] = ops.PackedLayout(lengths, device=DEVICE)
        else:
            doc = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
            doc = torch.cat([doc, torch.full((case["pad"],), -1)])
            state["doc"] = doc.to(DEVICE)         # the document of each row, -1 for padding
    else:
        rows, vocab = case["rows"], case["vocab"]
        if case["kind"] == "score":
            x = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2.5
            if case["masked"]:                    # a grammar that leaves one token in eight
                x = x.masked_fill(torch.arange(vocab, device=DEVICE) % 8 != 0, -math.inf)
            x = x if case["dtype"] == "fp32" else x.bfloat16()
            state["logits"] = x.requires_grad_(case["train"])
            state["ids"] = _ids(gen, rows, vocab, True if case["masked"] else None)
        else:
            hidden = case["hidden"]
            # normalised hidden states, and a head whose logits spread as a trained model's do
            state["h"] = torch.randn(rows, hidden, generator=gen, device=DEVICE).bfloat16().requires_grad_(case["train"])
            state["w"] = (torch.randn(vocab, hidden, generator=gen, device=DEVICE) * (2.0 / math.sqrt(hidden))).bfloat16()
            state["w"].requires_grad_(case["train"])
            state["ids"] = _ids(gen, rows, vocab)
        if case["train"]:
            # advantages over the number of tokens, and the weight of an entropy bonus
            state["g_log_probs"] = torch.randn(rows, generator=gen, device=DEVICE) / rows
            state["g_entropy"] = torch.full((rows,), 0.01 / rows, device=DEVICE)
    return state


# ------------------------------------------------------------------------------------------- one call
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        if case["kind"] == "attend":
            return _plain_attend(state, case)
        if case["kind"] == "score":
            return _plain_score(state, case)
        return _plain_head(state, case)


def _run_own(state, case):
    from himuon_b200 import ops

    if case["kind"] == "attend":
        o = ops.packed_attention(state["q"], state["k"], state["v"], state["layout"], case["heads"], case["kv_heads"],
                                 case["head_dim"])
        if not case["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["kind"] == "score":
        s = ops.token_log_probs(state["logits"], state["ids"], top_k=case["top_k"])
        out = {"log_probs": s.log_probs, "entropy": s.entropy}
        if case["top_k"]:
            out.update(top_log_probs=s.top_log_probs, top_ids=s.top_ids)
        if case["train"]:
            out["dlogits"] = torch.autograd.grad((s.log_probs, s.entropy), state["logits"],
                                                 (state["g_log_probs"], state["g_entropy"]))[0]
    else:
        s = ops.linear_token_log_probs(state["h"], state["w"], state["ids"])
        out = {"log_probs": s.log_probs, "entropy": s.entropy}
        if case["train"]:
            out["dh"], out["dw"] = torch.autograd.grad((s.log_probs, s.entropy), (state["h"], state["w"]),
                                                       (state["g_log_probs"], state["g_entropy"]))
    return {k: v.detach() for k, v in out.items()}


def _plain_attend(state, case):
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    G, scale, doc = H // K, 1.0 / math.sqrt(case["head_dim"]), state["doc"]
    T = doc.numel()

    def grouped(x):                               # (T, H * D) -> (K, G * T, D)
        return x.float().view(T, K, -1, D).permute(1, 2, 0, 3).reshape(K, -1, D)

    def flat(x, heads):                           # and back
        return x.reshape(heads, T, D).transpose(0, 1).reshape(T, heads * D).bfloat16()

    q, k, v = grouped(state["q"]), grouped(state["k"]), grouped(state["v"])
    at = torch.arange(T, device=doc.device)
    hidden = (doc[:, None] != doc[None, :]) | (doc[:, None] < 0) | (at[:, None] < at[None, :])
    s = (q @ k.transpose(1, 2)).mul_(scale).view(H, T, T).masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m.isinf(), torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)               # 0 for padding
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total))).view(K, G * T, T)
    o = p @ v
    out = {"o": flat(o, H)}
    if case["train"]:
        do = grouped(state["do"])
        dv = p.transpose(1, 2) @ do
        ds = (do @ v.transpose(1, 2)).sub_((o * do).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out.update(dq=flat(ds @ k, H), dk=flat(ds.transpose(1, 2) @ q, K), dv=flat(dv, K))
    return out


def _plain_log_probs(x, ids):
    """(log_probs, entropy, log of every probability) of fp32 logits."""
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    s = e.sum(-1, keepdim=True)
    t = (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(-1)
    log_s = s.log()
    counted = ids != IGNORE
    picked = d.gather(1, torch.where(counted, ids, torch.zeros_like(ids))[:, None])
    log_probs = torch.where(counted, (picked - log_s)[:, 0], torch.zeros_like(t))
    return log_probs, log_s[:, 0] - t / s[:, 0], d - log_s


def _plain_gradient(lp, entropy, ids, g_log_probs, g_entropy):
    """The gradient that reaches the logits, from the log of every probability."""
    counted = ids != IGNORE
    g = torch.where(counted, g_log_probs, torch.zeros_like(g_log_probs))
    p = lp.exp()
    dx = -p * (g[:, None] + g_entropy[:, None] * (torch.where(p > 0, lp, torch.zeros_like(lp)) + entropy[:, None]))
    return dx.scatter_add_(1, torch.where(counted, ids, torch.zeros_like(ids))[:, None], g[:, None])


def _plain_score(state, case):
    x, ids = state["logits"].float(), state["ids"]
    log_probs, entropy, lp = _plain_log_probs(x, ids)
    out = {"log_probs": log_probs, "entropy": entropy}
    if case["top_k"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]].contiguous()
        out.update(top_log_probs=lp.gather(1, order), top_ids=order)
    if case["train"]:
        out["dlogits"] = _plain_gradient(lp, entropy, ids, state["g_log_probs"], state["g_entropy"]).to(state["logits"].dtype)
    return out


def _plain_head(state, case):
    h, w, ids = state["h"].float(), state["w"].float(), state["ids"]
    log_probs, entropy, lp = _plain_log_probs(h @ w.t(), ids)
    out = {"log_probs": log_probs, "entropy": entropy}
    if case["train"]:
        dx = _plain_gradient(lp, entropy, ids, state["g_log_probs"], state["g_entropy"])
        out.update(dh=(dx @ w).bfloat16(), dw=(dx.t() @ h).bfloat16())
    return out


# ------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    train = case["train"]
    if case["kind"] == "attend":
        H, K, D, rows = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"] + case["pad"]
        pairs = sum(n * (n + 1) // 2 for n in _lengths(case))
        return {"bytes": 2 * rows * D * ((4 * H + 4 * K) if train else (2 * H + 2 * K)), "flops": (14 if train else 4) * D * H * pairs}
    rows, vocab = case["rows"], case["vocab"]
    if case["kind"] == "score":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": rows * (vocab * size * (2 if train else 1) + 16 + 12 * case["top_k"] + (8 if train else 0)), "flops": 0}
    hidden = case["hidden"]
    return {"bytes": 2 * hidden * (rows + vocab) * (2 if train else 1) + rows * (24 if train else 16),
            "flops": (6 if train else 2) * rows * hidden * vocab}


# ------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_attend(state, case) if case["kind"] == "attend" else _exact_scores(state, case)


def _exact_attend(state, case):
    """One document and one head at a time, from softmax's definition."""
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    rows, train = case["tokens"] + case["pad"], case["train"]
    q, k, v = (state[n].detach().double().view(rows, -1, D) for n in "qkv")
    o, dq, dk, dv = (torch.zeros(rows, n, D, dtype=torch.float64, device=DEVICE) for n in (H, H, K, K))
    do = state["do"].double().view(rows, H, D) if train else None
    first = 0
    for n in state["lengths"]:
        part = slice(first, first + n)
        first += n
        future = torch.ones(n, n, dtype=torch.bool, device=DEVICE).triu(1)
        for h in range(H if n else 0):
            g = h // (H // K)
            p = torch.softmax((q[part, h] @ k[part, g].T / math.sqrt(D)).masked_fill(future, -math.inf), dim=-1)
            o[part, h] = p @ v[part, g]
            if train:
                dp = do[part, h] @ v[part, g].T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[part, h] = ds @ k[part, g]
                dk[part, g] += ds.T @ q[part, h]
                dv[part, g] += p.T @ do[part, h]
    out = {"o": o.view(rows, -1)}
    if train:
        out.update(dq=dq.view(rows, -1), dk=dk.view(rows, -1), dv=dv.view(rows, -1))
    return out


def _exact_scores(state, case):
    """512 rows at a time, through the logarithm of the sum of exponentials."""
    rows, train, ids = case["rows"], case["train"], state["ids"]
    head = case["kind"] == "head"
    w = state["w"].detach().double() if head else None
    got = {n: [] for n in ("log_probs", "entropy", "top_log_probs", "dlogits", "dh")}
    dw = torch.zeros_like(w) if head and train else None
    for first in range(0, rows, 512):
        part = slice(first, first + 512)
        h = state["h"].detach()[part].double() if head else None
        x = (h @ w.T if head else state["logits"].detach()[part].double()).requires_grad_(train)
        with torch.set_grad_enabled(train):
            lp = torch.log_softmax(x, dim=-1)
            at = ids[part]
            log_probs = lp.gather(1, at.clamp(min=0)[:, None])[:, 0] * (at != IGNORE)
            entropy = -(lp.exp() * lp.clamp(min=-1e30)).sum(-1)
            if train:
                loss = (log_probs * state["g_log_probs"][part].double()).sum() + (entropy * state["g_entropy"][part].double()).sum()
        got["log_probs"].append(log_probs.detach())
        got["entropy"].append(entropy.detach())
        if case.get("top_k"):
            got["top_log_probs"].append(torch.topk(lp, case["top_k"], dim=-1).values)
        if train:
            dx = torch.autograd.grad(loss, x)[0]
            if head:
                got["dh"].append(dx @ w)
                dw += dx.T @ h
            else:
                got["dlogits"].append(dx)
    out = {n: torch.cat(t) for n, t in got.items() if t}
    if dw is not None:
        out["dw"] = dw
    if case.get("top_k"):
        out["top_ids"] = None
    return out
