"""What the block operators are measured on: windowed attention with first tokens that stay visible, the token embedding
with its scale, and the norm after a block joined with its gate, residual scale and the norm before the next block.

A case is a dict of plain values. ``run`` computes one pass of an operator, in elementary torch operations of 32 bits, or
through this framework's kernels where ``own`` is set; a training pass returns the output and every gradient.

Windowed attention: query ``i`` of ``Sq`` stands at key index ``p = i + Sk - Sq``. A document is a run of equal sequence ids
(the whole row without ids), ``s(p)`` its first index, and padding (id -1) sees and is seen by nothing. Then

    key j is visible to p  <=>  s(p) <= j <= p  and  (p - j < window  or  j - s(p) < sinks)
    out = softmax(scale * q k^T over visible keys) v          (zero where nothing is visible)

Embedding: ``out[t] = scale * weight[ids[t]]``, ``dweight[r] = scale * sum over t with ids[t] == r != padding_idx of dout[t]``.

Block norm: ``u = weight * x / rms(x)`` (``u = x`` without a weight), ``h = residual + scale * gate * u``,
``y = next_weight * h / rms(h)``, ``rms(x) = sqrt(mean(x^2) + eps)``; gate is absent, one value a channel, or one an element.
"""
import math

import torch

own = False
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def _attention(name, B, Sq, Sk, hq, hkv, D, window, sinks, docs=0, train=True, packed_qkv=False):
    case = dict(op="attention", B=B, Sq=Sq, Sk=Sk, hq=hq, hkv=hkv, D=D, window=window, sinks=sinks, docs=docs, train=train,
                packed_qkv=packed_qkv)
    return dict(case, name=name) if name else case


def _embedding(name, vocab, hidden, B, S, dtype, scale, pad, train=True):
    case = dict(op="embedding", vocab=vocab, hidden=hidden, B=B, S=S, dtype=dtype, scale=scale, pad=pad, train=train)
    return dict(case, name=name) if name else case


def _norm(name, rows, hidden, dtype, post, pre, gate, scale, train=True):
    case = dict(op="norm", rows=rows, hidden=hidden, dtype=dtype, post=post, pre=pre, gate=gate, scale=scale, train=train)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the 50 M model's layer: eight heads of 64, one row of 1024 tokens, a short window
        _attention("attention 50M layer", 1, 1024, 1024, 8, 8, 64, 256, 4),
        # the 8 B model's layer on one GPU: grouped heads, one row of 8192 tokens
        _attention("attention 8B layer", 1, 8192, 8192, 32, 8, 128, 1024, 4),
        # a tensor-parallel quarter of that layer on a row twice as long, with a wide window and more first tokens
        _attention("attention long row", 1, 16384, 16384, 8, 2, 128, 4096, 16),
        # fine-tuning: packed documents with a padded tail, an odd row length, heads of a packed projection (half of 40 heads)
        _attention("attention packed documents", 1, 4093, 4093, 20, 20, 128, 512, 4, docs=9, packed_qkv=True),
        # scoring the continuation of a long prompt: 1000 new tokens over 5000 keys, forward only
        _attention("attention continuation", 2, 1000, 5000, 32, 8, 128, 2048, 4, train=False),
        # one new token a row over long rows: the smallest call
        _attention("attention one token", 8, 1, 8191, 32, 8, 128, 2048, 4, train=False),
        # the 50 M model: a short row, the vocabulary's gradient is mostly zeros
        _embedding("embedding 50M model", 32000, 512, 1, 1024, "bf16", 22.627, False),
        # the 8 B model: the largest table, four rows of 8192 tokens
        _embedding("embedding 8B model", 128256, 4096, 4, 8192, "bf16", 64.0, False),
        # fine-tuning in 32 bits with odd rows whose padded tail is all one token
        _embedding("embedding padded rows", 100352, 768, 3, 2047, "fp32", 1.0, True),
        # a few tokens through a gated block, forward only: latency
        _norm("norm few tokens", 16, 1024, "bf16", True, True, "element", 1.0, train=False),
        # norms on both sides of a block of the 8 B model, with the residual scaled by depth
        _norm("norm both sides", 8192, 4096, "bf16", True, True, "none", 0.125),
        # a norm after the block alone, with a gate a channel, on an odd number of rows
        _norm("norm after, channel gate", 4093, 5120, "bf16", True, False, "channel", 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "embedding", "norm"])
    if op == "attention":
        hkv = rng.choice([1, 2, 4, 5, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        D = rng.choice([64, 128])
        Sk = _log(rng, 1, 16384)
        kind = rng.choice(["train", "train", "train", "chunk", "token"])
        B = _log(rng, 1, 8)
        while B * hq * Sk * Sk > 8 * 16384 * 16384:
            Sk = Sk * 2 // 3 + rng.randrange(3)
        Sq = Sk if kind == "train" else 1 if kind == "token" else _log(rng, 1, Sk)
        docs = rng.choice([0, 0, 0, 1, 3, 8]) if kind == "train" and Sk >= 64 else 0
        return _attention(None, B, Sq, Sk, hq, hkv, D, _log(rng, 1, 8192), rng.choice([0, 0, 1, 4, 4, 16, 64, 200]), docs,
                          kind == "train", kind == "train" and rng.random() < 0.3)
    if op == "embedding":
        hidden = 8 * _log(rng, 8, 640)
        vocab = _log(rng, 500, 128256)
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        while vocab * hidden * (4 if dtype == "fp32" else 2) > 128256 * 4096 * 2:
            vocab = vocab * 2 // 3
        return _embedding(None, vocab, hidden, rng.choice([1, 2, 3, 4]), _log(rng, 1, 8192), dtype,
                          rng.choice([1.0, round(math.sqrt(hidden), 3)]), rng.random() < 0.3, rng.random() < 0.8)
    hidden = 8 * _log(rng, 8, 1024)
    rows = _log(rng, 1, 16384)
    while rows * hidden > 8192 * 4096:
        rows = rows * 2 // 3
    post = rng.random() < 0.8
    return _norm(None, rows, hidden, rng.choice(["bf16", "bf16", "fp32"]), post, not post or rng.random() < 0.6,
                 rng.choice(["none", "channel", "element"]), rng.choice([1.0, 0.125, 0.7]), rng.random() < 0.8)


_DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _documents(case):
    """Lengths of the packed documents of every row; what is left of the row is padding."""
    n = case["docs"]
    room = case["Sk"] - case["Sk"] // 16
    parts = [1 + (7 * k * k + 3 * k) % 11 for k in range(n)]
    ends = [room * sum(parts[:k + 1]) // sum(parts) for k in range(n)]
    return [e - (ends[k - 1] if k else 0) for k, e in enumerate(ends)]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["op"] == "attention":
        B, Sq, Sk, hq, hkv, D = (case[k] for k in ("B", "Sq", "Sk", "hq", "hkv", "D"))
        ids = None
        first = torch.zeros(Sk, dtype=torch.bool, device="cuda")
        first[:max(1, case["sinks"])] = True
        if case["docs"]:
            ids = torch.full((B, Sk), -1, dtype=torch.int64, device="cuda")
            at = 0
            for n, length in enumerate(_documents(case)):
                ids[:, at:at + length] = n
                first[at:at + min(length, max(1, case["sinks"]))] = True
                at += length
        # queries lean towards what the first tokens of a document hold, as trained models' do
        lean = torch.nn.functional.normalize(randn(D), dim=0)
        qkv = randn(B, Sk, hq + 2 * hkv, D)
        qkv[:, :, :hq] += 3 * lean
        qkv[:, :, hq:hq + hkv] += 12 * lean * first.view(1, Sk, 1, 1)
        qkv = qkv.bfloat16()
        q, k, v = qkv[:, Sk - Sq:, :hq], qkv[:, :, hq:hq + hkv], qkv[:, :, hq + hkv:]
        if not case["packed_qkv"]:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        state = dict(case=case, ids=ids, q=q.detach(), k=k.detach(), v=v.detach())
        if case["train"]:
            state["dout"] = randn(B, Sq, hq, D).bfloat16()
            for t in "qkv":
                state[t].requires_grad_()
        return state
    dtype = _DTYPE[case["dtype"]]
    if case["op"] == "embedding":
        V, H, B, S = case["vocab"], case["hidden"], case["B"], case["S"]
        weight = (0.02 * randn(V, H)).to(dtype)
        # token frequencies fall with the rank, ranks are spread over the vocabulary; a padded tail is one token
        rank = torch.exp(torch.rand(B, S, device="cuda", generator=g) * math.log(V)).long().clamp_(1, V) - 1
        ids = rank * 40503 % V
        pad = None
        if case["pad"]:
            pad = V - 1
            for b in range(B):
                ids[b, S - (S * (b + 1)) // (B + 2):] = pad
        state = dict(case=case, ids=ids, pad=pad, weight=weight)
        if case["train"]:
            weight.requires_grad_()
            state["dout"] = (0.01 * randn(B, S, H)).to(dtype)
        return state
    rows, H = case["rows"], case["hidden"]
    state = dict(case=case, x=(3 * randn(rows, H)).to(dtype), residual=(5 * randn(rows, H)).to(dtype), weight=None, next_weight=None, gate=None)
    if case["post"]:
        state["weight"] = (1 + 0.2 * randn(H)).to(dtype)
    if case["pre"]:
        state["next_weight"] = (1 + 0.2 * randn(H)).to(dtype)
        state["dy"] = randn(rows, H).to(dtype)
    if case["gate"] != "none":
        state["gate"] = torch.sigmoid(randn(*((H,) if case["gate"] == "channel" else (rows, H)))).to(dtype)
    state["dh"] = randn(rows, H).to(dtype)
    if case["train"]:
        for t in ("x", "residual", "weight", "next_weight", "gate"):
            if state[t] is not None:
                state[t].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _starts(ids, Sk):
    """First index of every token's document, and whether the token is no padding: [B, Sk] each."""
    at = torch.arange(Sk, device=ids.device).expand(ids.shape)
    begins = torch.ones_like(ids, dtype=torch.bool)
    begins[:, 1:] = ids[:, 1:] != ids[:, :-1]
    return torch.where(begins, at, 0).cummax(dim=1).values, ids != -1


def _visible(case, ids):
    """[B or 1, Sq, Sk]"""
    Sq, Sk = case["Sq"], case["Sk"]
    j = torch.arange(Sk, device="cuda").view(1, 1, Sk)
    p = torch.arange(Sk - Sq, Sk, device="cuda").view(1, Sq, 1)
    if ids is None:
        return (j <= p) & ((p - j < case["window"]) | (j < case["sinks"]))
    start, real = _starts(ids, Sk)
    start, real = start[:, Sk - Sq:].unsqueeze(2), real[:, Sk - Sq:].unsqueeze(2)
    return real & (j >= start) & (j <= p) & ((p - j < case["window"]) | (j - start < case["sinks"]))


def _plain_attention(state):
    case = state["case"]
    B, Sq, Sk, hq, hkv, D = (case[k] for k in ("B", "Sq", "Sk", "hq", "hkv", "D"))
    group, scale = hq // hkv, 1 / math.sqrt(D)

    def heads(t):                                  # [B, S, h, D] -> [B, hkv, h / hkv, S, D]
        return t.detach().float().permute(0, 2, 1, 3).reshape(B, hkv, -1, t.shape[1], D)

    def back(t, like):                             # and back, in the inputs' type
        return t.reshape(B, -1, t.shape[3], D).permute(0, 2, 1, 3).to(like.dtype).contiguous()

    q, k, v = heads(state["q"]), heads(state["k"]), heads(state["v"])
    seen = _visible(case, state["ids"]).view(-1, 1, 1, Sq, Sk)
    p = torch.matmul(q * scale, k.transpose(-1, -2)).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0, top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    out = torch.matmul(p, v)
    if not case["train"]:
        return back(out, state["q"])
    dout = heads(state["dout"])
    dv = torch.matmul(p.transpose(-1, -2), dout).sum(2, keepdim=True)
    ds = torch.matmul(dout, v.transpose(-1, -2)).sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True)
    return {"out": back(out, state["q"]), "dq": back(dq, state["q"]), "dk": back(dk, state["k"]), "dv": back(dv, state["v"])}


def _plain_embedding(state):
    case, weight, ids = state["case"], state["weight"], state["ids"]
    out = (weight.detach()[ids].float() * case["scale"]).to(weight.dtype)
    if not case["train"]:
        return out
    rows = state["dout"].float().reshape(-1, case["hidden"]) * case["scale"]
    flat = ids.reshape(-1)
    if state["pad"] is not None:
        rows = rows * (flat != state["pad"]).unsqueeze(1)
    dweight = torch.zeros(case["vocab"], case["hidden"], device=rows.device).index_add_(0, flat, rows)
    return {"out": out, "dweight": dweight.to(weight.dtype)}


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    x, residual, weight, following, gate = (None if state[t] is None else state[t].detach().float()
                                            for t in ("x", "residual", "weight", "next_weight", "gate"))
    s = case["scale"]
    g = 1.0 if gate is None else gate
    if weight is None:
        u = x
    else:
        rx = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        xn = x * rx
        u = xn * weight
    h = residual + s * g * u
    got = {"h": h.to(dtype)}
    if following is not None:
        rh = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        hn = h * rh
        got["y"] = (hn * following).to(dtype)
    if not case["train"]:
        return got
    dh = state["dh"].float()
    if following is not None:
        dy = state["dy"].float()
        got["dnext_weight"] = (dy * hn).sum(0).to(dtype)
        dn = dy * following
        dh = dh + rh * (dn - hn * (dn * hn).mean(-1, keepdim=True))
    du = dh * (s * g)
    if gate is not None:
        dg = s * dh * u
        got["dgate"] = (dg.sum(0) if case["gate"] == "channel" else dg).to(dtype)
    if weight is not None:
        got["dweight"] = (du * xn).sum(0).to(dtype)
        dn = du * weight
        du = rx * (dn - xn * (dn * xn).mean(-1, keepdim=True))
    return dict(got, dx=du.to(dtype), dresidual=dh.to(dtype))


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_attention(state):
    from maltos_b200.ops.attention import sliding_window_attention

    case, leaves = state["case"], (state["q"], state["k"], state["v"])
    with torch.set_grad_enabled(case["train"]):
        out = sliding_window_attention(*leaves, window=case["window"], sinks=case["sinks"], sequence_ids=state["ids"])
    if not case["train"]:
        return out
    dq, dk, dv = torch.autograd.grad(out, leaves, state["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_embedding(state):
    from maltos_b200.ops.embedding import embedding

    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        out = embedding(state["ids"], state["weight"], scale=case["scale"], padding_idx=state["pad"])
    if not case["train"]:
        return out
    return {"out": out.detach(), "dweight": torch.autograd.grad(out, state["weight"], state["dout"])[0]}


def _own_norm(state):
    from maltos_b200.ops.norm import block_norm

    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        res = block_norm(state["x"], state["residual"], state["weight"], state["next_weight"], gate=state["gate"], scale=case["scale"], eps=EPS)
    y, h = res if case["pre"] else (None, res)
    got = {"h": h.detach()}
    if y is not None:
        got["y"] = y.detach()
    if not case["train"]:
        return got
    names = [t for t in ("x", "residual", "weight", "next_weight", "gate") if state[t] is not None]
    outs, grads = ((h,), (state["dh"],)) if y is None else ((y, h), (state["dy"], state["dh"]))
    for name, d in zip(names, torch.autograd.grad(outs, [state[t] for t in names], grads)):
        got["d" + name] = d
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_attention(state) if op == "attention" else _own_embedding(state) if op == "embedding" else _own_norm(state)
    return _plain_attention(state) if op == "attention" else _plain_embedding(state) if op == "embedding" else _plain_norm(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs of one head and row."""
    W, n = case["window"], case["sinks"]

    def of_document(length, first):
        total = 0
        for p in range(first, length):
            total += min(p + 1, min(W, p + 1) + min(n, max(0, p + 1 - W)))
        return total

    if case["docs"]:
        return sum(of_document(length, 0) for length in _documents(case))
    return of_document(case["Sk"], case["Sk"] - case["Sq"])


def work(case):
    if case["op"] == "attention":
        B, Sq, Sk, hq, hkv, D = (case[k] for k in ("B", "Sq", "Sk", "hq", "hkv", "D"))
        # keys that some query sees: from the first query's window on, and the first tokens
        low = max(0, Sk - Sq - case["window"] + 1)
        keys = Sk - low + min(low, case["sinks"])
        nq, nk = B * Sq * hq * D * 2, B * keys * hkv * D * 2
        pairs = _pairs(case) * B * hq
        if case["train"]:                          # q, k, v, dout in; out, dq, dk, dv out
            return {"bytes": 4 * nq + 4 * nk, "flops": 14 * pairs * D}
        return {"bytes": 2 * nq + 2 * nk, "flops": 4 * pairs * D}
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "embedding":
        tokens, H, V = case["B"] * case["S"], case["hidden"], case["vocab"]
        # distinct rows of the log-uniform draw: sum over ranks of 1 - (1 - p)^tokens, with p = log(1 + 1 / rank) / log(V)
        n, distinct, r = tokens, 0.0, 1
        while r <= V:
            upto = min(V, r + max(0, r // 64))
            p = math.log((upto + 1) / r) / math.log(V) / (upto - r + 1)
            distinct += (upto - r + 1) * (1 - math.exp(-n * p))
            r = upto + 1
        read = int(min(distinct, tokens)) * H * size + tokens * 8
        if case["train"]:
            return {"bytes": read + 2 * tokens * H * size + tokens * 8 + V * H * size, "flops": 2 * tokens * H}
        return {"bytes": read + tokens * H * size, "flops": tokens * H}
    n = case["rows"] * case["hidden"]
    gate = n if case["gate"] == "element" else 0
    forward = 3 * n + gate + (n if case["pre"] else 0)                       # x, residual, gate in; h, y out
    backward = 3 * n + 2 * gate + (2 * n if case["pre"] else 0)              # dh, x, gate, dy, h in; dx, dresidual, dgate out
    if not case["train"]:
        return {"bytes": forward * size, "flops": 10 * n}
    if not case["post"] and case["gate"] == "none":
        backward -= n                                                        # x is not needed again
    return {"bytes": (forward + backward) * size, "flops": 35 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_attention(case, state):
    B, Sq, Sk, hq, hkv, D = (case[k] for k in ("B", "Sq", "Sk", "hq", "hkv", "D"))
    names = ("out", "dq", "dk", "dv") if case["train"] else ("out",)
    got = {"out": torch.zeros(B, Sq, hq, D, dtype=torch.float64, device="cuda")}
    if case["train"]:
        got |= {"dq": torch.zeros_like(got["out"]), "dk": torch.zeros(B, Sk, hkv, D, dtype=torch.float64, device="cuda")}
        got["dv"] = torch.zeros_like(got["dk"])
    spans = [(0, Sk)]
    if case["docs"]:
        spans, at = [], 0
        for length in _documents(case):
            spans.append((at, at + length))
            at += length
    for b in range(B):
        for lo, hi in spans:                       # one document at a time, positions counted from its start
            first = max(lo, Sk - Sq)               # first query of the document
            if first >= hi:
                continue
            pos = torch.arange(first - lo, hi - lo, device="cuda").unsqueeze(1)
            key = torch.arange(hi - lo, device="cuda").unsqueeze(0)
            hidden = (key > pos) | ((key <= pos - case["window"]) & (key >= case["sinks"]))
            for h in range(hq):
                n = h * hkv // hq
                rows = slice(first - (Sk - Sq), hi - (Sk - Sq))
                q = state["q"][b, rows, h].detach().double()
                k, v = state["k"][b, lo:hi, n].detach().double(), state["v"][b, lo:hi, n].detach().double()
                if case["train"]:
                    for t in (q, k, v):
                        t.requires_grad_()
                a = (q @ k.t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                o = torch.exp(a - torch.logsumexp(a, 1, keepdim=True)) @ v
                got["out"][b, rows, h] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["dout"][b, rows, h].double())
                    got["dq"][b, rows, h] = dq
                    got["dk"][b, lo:hi, n] += dk
                    got["dv"][b, lo:hi, n] += dv
    return got if case["train"] else got[names[0]]


def _exact_embedding(case, state):
    weight, ids = state["weight"].detach(), state["ids"]
    out = weight[ids].double().mul_(case["scale"])
    if not case["train"]:
        return out
    flat, rows = ids.reshape(-1), state["dout"].reshape(-1, case["hidden"])
    order = torch.argsort(flat, stable=True)
    token, count = torch.unique_consecutive(flat[order], return_counts=True)
    ends = count.cumsum(0)
    dweight = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device="cuda")
    for c in range(0, case["hidden"], 512):        # sums of runs, a slice of columns at a time
        part = rows[order, c:c + 512].double()
        total = torch.segment_reduce(part, "sum", lengths=count, axis=0)
        dweight[token, c:c + 512] = total * case["scale"]
    if state["pad"] is not None:
        dweight[state["pad"]] = 0
    assert int(ends[-1]) == flat.numel()
    return {"out": out, "dweight": dweight}


def _exact_norm(case, state):
    leaf = {t: None if state[t] is None else state[t].detach().double().requires_grad_(case["train"])
            for t in ("x", "residual", "weight", "next_weight", "gate")}

    def rms_norm(t, w):
        return w * t / torch.sqrt((t * t).sum(-1, keepdim=True) / t.shape[-1] + EPS)

    branch = leaf["x"] if leaf["weight"] is None else rms_norm(leaf["x"], leaf["weight"])
    if leaf["gate"] is not None:
        branch = branch * leaf["gate"]
    h = leaf["residual"] + case["scale"] * branch
    outs, grads, got = [h], [state["dh"].double()], {"h": h.detach()}
    if case["pre"]:
        y = rms_norm(h, leaf["next_weight"])
        outs, grads = outs + [y], grads + [state["dy"].double()]
        got["y"] = y.detach()
    if case["train"]:
        used = [t for t in leaf if leaf[t] is not None]
        for t, d in zip(used, torch.autograd.grad(outs, [leaf[t] for t in used], grads)):
            got["d" + t] = d
    return got


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, state)
    return _exact_embedding(case, state) if case["op"] == "embedding" else _exact_norm(case, state)
