"""Operators of a training step and of scoring, each with its plain form: attention whose backward pass recomputes the
probabilities, log probabilities of given tokens (with entropy and the best alternatives), and distillation from a teacher's
top logits.

A case is one call of an operator on seeded data, and, where ``backward`` says so, the gradients of its inputs for a given
gradient of its outputs:

``attention``  queries ``[batch, heads, sq, dim]`` over keys ``[batch, kv_heads, skv, dim]`` (views of token-major activations,
               as projections give them), causal or not, with a window, with padded sequences (``pad``).
``logprobs``   ``[batch, tokens, vocab]`` logits with one target a row; ``top`` alternatives.
``distill``    the same logits against ``k`` teacher tokens a row; ``tail``: all other tokens are one more class.
"""
import math

import torch

own = False

GRAD_STD = 1.0 / 16
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # a test model's layer: the smallest call, where launches and host time count
        dict(name="attention-64-tokens", kind="attention", batch=1, heads=4, kv_heads=4, sq=64, skv=64, dim=64, causal=True,
             window=0, pad="none", dtype="bfloat16", backward=True),
        # one layer of the QLoRA benchmark: Llama-2-13B, micro-batch 4, 512 tokens
        dict(name="attention-13b", kind="attention", batch=4, heads=40, kv_heads=40, sq=512, skv=512, dim=128, causal=True,
             window=0, pad="none", dtype="bfloat16", backward=True),
        # a batch of the collator, which pads on the right, of an odd length
        dict(name="attention-7b-padded", kind="attention", batch=3, heads=32, kv_heads=32, sq=333, skv=333, dim=128,
             causal=True, window=0, pad="right", dtype="float16", backward=True),
        # long sequences on shared key heads: the tensor cores' time
        dict(name="attention-70b-4096", kind="attention", batch=1, heads=64, kv_heads=8, sq=4096, skv=4096, dim=128,
             causal=True, window=0, pad="none", dtype="bfloat16", backward=True),
        # a window and left padding (rows that see nothing), heads of 80
        dict(name="attention-window-80", kind="attention", batch=2, heads=32, kv_heads=8, sq=1031, skv=1031, dim=80,
             causal=True, window=256, pad="left", dtype="float16", backward=True),
        # an encoder's layer, evaluated: both directions, no gradient
        dict(name="attention-encoder", kind="attention", batch=2, heads=20, kv_heads=20, sq=1500, skv=1500, dim=64,
             causal=False, window=0, pad="none", dtype="float16", backward=False),
        # a served token with its log probability and five alternatives
        dict(name="logprobs-1-row", kind="logprobs", batch=1, tokens=1, vocab=32000, top=5, temperature=1.0, dtype="float16",
             backward=False),
        # the loss of the QLoRA benchmark's micro-batch with an entropy term: both gradients
        dict(name="logprobs-train", kind="logprobs", batch=4, tokens=512, vocab=32000, top=0, temperature=1.0,
             dtype="bfloat16", backward=True),
        # scoring a prompt of the 70B model's vocabulary with twenty alternatives a position
        dict(name="logprobs-score-128k", kind="logprobs", batch=1, tokens=2048, vocab=128256, top=20, temperature=0.7,
             dtype="bfloat16", backward=False),
        # a few rows of an odd vocabulary (three tokens added) in 32 bits
        dict(name="distill-37-rows", kind="distill", batch=1, tokens=37, vocab=32003, k=8, temperature=1.0, tail=False,
             dtype="float32", backward=True),
        # distillation at the QLoRA benchmark's micro-batch
        dict(name="distill-train", kind="distill", batch=4, tokens=512, vocab=32000, k=64, temperature=2.0, tail=False,
             dtype="bfloat16", backward=True),
        # the 128k vocabulary, where what the teacher did not give is a class of its own
        dict(name="distill-tail-128k", kind="distill", batch=2, tokens=1024, vocab=128256, k=100, temperature=1.0, tail=True,
             dtype="bfloat16", backward=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "logprobs", "distill"])
    if kind == "attention":
        kv = rng.choice([1, 2, 3, 4, 5, 8])
        sq = _log_int(rng, 1, 2048)
        skv = sq if rng.random() < 0.7 else sq + _log_int(rng, 1, 1024)
        causal = rng.random() < 0.75
        heads = kv * rng.choice([1, 1, 2, 4, 6])
        batch = min(rng.randint(1, 4), max(1, (1 << 29) // (heads * sq * skv)))
        return dict(kind=kind, batch=batch, heads=heads, kv_heads=kv, sq=sq, skv=skv,
                    dim=rng.choice([32, 64, 64, 72, 80, 96, 112, 128, 128, 128]), causal=causal,
                    window=_log_int(rng, 1, 1024) if causal and rng.random() < 0.3 else 0,
                    pad=rng.choice(["none", "none", "right", "left"]), dtype=rng.choice(["bfloat16", "float16"]),
                    backward=rng.random() < 0.8)
    vocab = _log_int(rng, 500, 130000)
    rows = _log_int(rng, 1, min(2048, int(1.2e8 / vocab)))
    batch = rng.choice([1, 1, 2, 3])
    case = dict(kind=kind, batch=batch, tokens=max(1, rows // batch), vocab=vocab,
                temperature=rng.choice([1.0, 1.0, 0.5, 2.0]), dtype=rng.choice(["bfloat16", "float16", "float32"]))
    if kind == "logprobs":
        return dict(case, top=rng.choice([0, 1, 5, 20, 32]), backward=rng.random() < 0.6)
    return dict(case, k=_log_int(rng, 1, 128), tail=rng.random() < 0.5, backward=rng.random() < 0.8)


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(g, shape, std):
    return torch.randn(shape, generator=g, device="cuda") * std


def _key_mask(case, g):
    """True where a key is a real token: between a half and all of every sequence, padded on one side."""
    if case["pad"] == "none":
        return None
    n = case["skv"]
    real = n - (torch.rand(case["batch"], 1, generator=g, device="cuda") * (n // 2 + 1)).long().clamp(max=n - 1)
    at = torch.arange(n, device="cuda").view(1, n)
    return at < real if case["pad"] == "right" else at >= n - real


def _prepare_attention(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    B, H, G, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]

    def heads(n, s, std):
        return _normal(g, (B, s, n, D), std).to(dt).transpose(1, 2)

    st = dict(q=heads(H, case["sq"], 1.5), k=heads(G, case["skv"], 1.0), v=heads(G, case["skv"], 1.0),
              grad=heads(H, case["sq"], GRAD_STD), mask=_key_mask(case, g))
    for name in "qkv":
        st[name].requires_grad_(case["backward"])
    return st


def _targets(case, g):
    """A token for each row; the last of a sequence has none to predict (-100)."""
    t = torch.randint(0, case["vocab"], (case["batch"], case["tokens"]), generator=g, device="cuda")
    if case["tokens"] > 1:
        t[:, -1] = -100
    return t


def _logits(case, g, targets):
    """Scores with a handful of likely tokens: what an output layer gives."""
    x = _normal(g, (case["batch"], case["tokens"], case["vocab"]), 2.5)
    lift = 4.0 + 4.0 * torch.rand(case["batch"], case["tokens"], 1, generator=g, device="cuda")
    return x.scatter_add_(2, targets.clamp(min=0).unsqueeze(2), lift)


def _prepare_logprobs(case, seed):
    g = _generator(seed)
    targets = _targets(case, g)
    logits = _logits(case, g, targets).to(DTYPES[case["dtype"]]).requires_grad_(case["backward"])
    rows = (case["batch"], case["tokens"])
    return dict(logits=logits, targets=targets, grad=_normal(g, rows, 1.0), grad_entropy=_normal(g, rows, 0.1))


def _prepare_distill(case, seed):
    g = _generator(seed)
    x = _logits(case, g, _targets(case, g))
    teacher = 1.1 * x + _normal(g, x.shape, 0.5)
    best = torch.topk(teacher, case["k"], dim=-1)
    lse = torch.logsumexp(teacher / case["temperature"], dim=-1) if case["tail"] else None
    return dict(logits=x.to(DTYPES[case["dtype"]]).requires_grad_(case["backward"]), ids=best.indices, values=best.values,
                lse=lse, grad=_normal(g, (case["batch"], case["tokens"]), 1.0))


def prepare(case, seed):
    with torch.no_grad():
        st = dict(attention=_prepare_attention, logprobs=_prepare_logprobs, distill=_prepare_distill)[case["kind"]](case, seed)
    return dict(st, case=case)


# ---- the plain forms, in 32 bits ------------------------------------------------------------------------------------------
def _visible(case, mask, b):
    """[sq, skv]: which keys a query of sequence b sees."""
    last = torch.arange(case["sq"], device="cuda").view(-1, 1) + (case["skv"] - case["sq"])
    key = torch.arange(case["skv"], device="cuda").view(1, -1)
    see = torch.ones(case["sq"], case["skv"], dtype=torch.bool, device="cuda")
    if case["causal"]:
        see = see & (key <= last)
    if case["window"]:
        see = see & (key > last - case["window"])
    return see if mask is None else see & mask[b].view(1, -1)


def _plain_attention(st):
    case = st["case"]
    q, k, v, dt = st["q"], st["k"], st["v"], st["q"].dtype
    scale = case["dim"] ** -0.5
    per = case["heads"] // case["kv_heads"]
    step = max(1, (1 << 27) // (case["sq"] * case["skv"]))      # query heads at a time: half a GB of scores
    out = torch.empty_like(q)
    grads = [torch.empty_like(q), torch.zeros_like(k, dtype=torch.float32), torch.zeros_like(v, dtype=torch.float32)]
    for b in range(case["batch"]):
        see = _visible(case, st["mask"], b)
        for h0 in range(0, case["heads"], step):
            hs = torch.arange(h0, min(h0 + step, case["heads"]), device="cuda")
            gs = hs // per
            qf, kf, vf = q[b, hs].float(), k[b, gs].float(), v[b, gs].float()
            s = (qf @ kf.transpose(1, 2) * scale).masked_fill(~see, -math.inf)
            top = s.amax(dim=-1, keepdim=True).clamp(min=-1e30)
            p = torch.exp(s - top)
            total = p.sum(dim=-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            o = p @ vf
            out[b, hs] = o.to(dt)
            if not case["backward"]:
                continue
            do = st["grad"][b, hs].float()
            ds = p * (do @ vf.transpose(1, 2) - (do * o).sum(dim=-1, keepdim=True))
            grads[0][b, hs] = (ds @ kf * scale).to(dt)
            grads[1][b].index_add_(0, gs, ds.transpose(1, 2) @ qf * scale)
            grads[2][b].index_add_(0, gs, p.transpose(1, 2) @ do)
    if not case["backward"]:
        return {"out": out}
    return {"out": out, "dq": grads[0], "dk": grads[1].to(dt), "dv": grads[2].to(dt)}


def _plain_logprobs(st):
    case, x, targets = st["case"], st["logits"].float(), st["targets"]
    y = x / case["temperature"]
    y = y - y.amax(dim=-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(dim=-1, keepdim=True)
    y = y - torch.log(total)                                        # log probabilities
    e = e / total
    real = targets != -100
    at = targets.clamp(min=0).unsqueeze(2)
    got = {"logprob": torch.where(real, y.gather(2, at).squeeze(2), 0.0),
           "entropy": torch.where(real, -(e * y).sum(dim=-1), 0.0)}
    if case["top"]:
        ids, x = [], x.clone()
        for _ in range(case["top"]):                                # the first of equal ones each time
            ids.append(x.argmax(dim=-1, keepdim=True))
            x.scatter_(2, ids[-1], -math.inf)
        got["top_ids"] = torch.cat(ids, dim=-1)
        got["top_logprobs"] = y.gather(2, got["top_ids"])
    if case["backward"]:
        g = torch.where(real, st["grad"], 0.0).unsqueeze(2)
        ge = torch.where(real, st["grad_entropy"], 0.0).unsqueeze(2)
        d = -e * (g + ge * (y + got["entropy"].unsqueeze(2)))
        d = d.scatter_add_(2, at, g) / case["temperature"]
        got["dlogits"] = d.to(st["logits"].dtype)
    return got


def _plain_distill(st):
    case, x, ids = st["case"], st["logits"].float(), st["ids"]
    T = case["temperature"]
    y = x / T
    y = y - y.amax(dim=-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(dim=-1, keepdim=True)
    t = st["values"] / T
    if case["tail"]:
        logq = t - st["lse"].unsqueeze(2)
        q = torch.exp(logq)
        rest = (1.0 - q.double().sum(dim=-1, keepdim=True)).clamp(min=0.0).float()
    else:
        top = t.amax(dim=-1, keepdim=True)
        logq = t - top - torch.log(torch.exp(t - top).sum(dim=-1, keepdim=True))
        q = torch.exp(logq)
        rest = torch.zeros_like(total)
    loss = (q * (logq - (y.gather(2, ids) - torch.log(total)))).sum(dim=-1, keepdim=True)
    if case["tail"]:
        others = e.scatter(2, ids, 0.0)
        left = others.sum(dim=-1, keepdim=True) / total
        some = (rest > 0) & (left > 0)
        loss = loss + torch.where(some, rest * (torch.log(rest) - torch.log(left)), 0.0)
    got = {"loss": (loss * (T * T)).squeeze(2)}
    if case["backward"]:
        d = e / total * (q.sum(dim=-1, keepdim=True) + rest)
        if case["tail"]:
            d = d - others / total * torch.where(some, rest / left, 0.0)
        d = d.scatter_add_(2, ids, -q) * (st["grad"].unsqueeze(2) * T)
        got["dlogits"] = d.to(st["logits"].dtype)
    return got


# ---- the framework's operators ----------------------------------------------------------------------------------------
def _own_attention(st):
    from ipex_llm_b200.ops.train_attn import attention
    case = st["case"]
    out = attention(st["q"], st["k"], st["v"], causal=case["causal"], window=case["window"], key_mask=st["mask"])
    if not case["backward"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["grad"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_logprobs(st):
    from ipex_llm_b200.ops.token_loss import token_logprobs
    case = st["case"]
    r = token_logprobs(st["logits"], st["targets"], temperature=case["temperature"], entropy=True, top=case["top"])
    got = {"logprob": r.logprob.detach(), "entropy": r.entropy.detach()}
    if case["top"]:
        got["top_ids"], got["top_logprobs"] = r.top_ids, r.top_logprobs
    if case["backward"]:
        got["dlogits"], = torch.autograd.grad((r.logprob, r.entropy), (st["logits"],), (st["grad"], st["grad_entropy"]))
    return got


def _own_distill(st):
    from ipex_llm_b200.ops.token_loss import distill_loss
    loss = distill_loss(st["logits"], st["ids"], st["values"], temperature=st["case"]["temperature"],
                        teacher_logsumexp=st["lse"])
    got = {"loss": loss.detach()}
    if st["case"]["backward"]:
        got["dlogits"], = torch.autograd.grad(loss, (st["logits"],), st["grad"])
    return got


def run(state):
    if own:
        return dict(attention=_own_attention, logprobs=_own_logprobs, distill=_own_distill)[state["case"]["kind"]](state)
    with torch.no_grad():
        return dict(attention=_plain_attention, logprobs=_plain_logprobs, distill=_plain_distill)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _pairs(case):
    """Seen pairs of one head and sequence, padding apart."""
    sq, skv, n = case["sq"], case["skv"], 0
    if not case["causal"]:
        return sq * skv
    for i in range(sq):
        end = i + skv - sq + 1
        n += end - max(0, end - case["window"] if case["window"] else 0)
    return n


def work(case):
    if case["kind"] == "attention":
        row = 2 * case["batch"] * case["dim"]
        queries, keys = row * case["heads"] * case["sq"], row * case["kv_heads"] * case["skv"]
        flops = _pairs(case) * case["batch"] * case["heads"] * case["dim"]
        if not case["backward"]:
            return {"bytes": 2 * queries + 2 * keys, "flops": 4.0 * flops}
        return {"bytes": 4 * queries + 4 * keys, "flops": 14.0 * flops}
    rows = case["batch"] * case["tokens"]
    per = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    logits = rows * case["vocab"]
    if case["kind"] == "logprobs":
        side = rows * (8 + 8 + 12 * case["top"] + (8 if case["backward"] else 0))
    else:
        side = rows * (12 * case["k"] + 4 + (4 if case["tail"] else 0) + (4 if case["backward"] else 0))
    return {"bytes": logits * per * (2 if case["backward"] else 1) + side, "flops": logits * (8.0 if case["backward"] else 4.0)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_attention(case, st):
    per = case["heads"] // case["kv_heads"]
    shape = {n: st[n].shape for n in "qkv"}
    out = torch.zeros(shape["q"], dtype=torch.float64, device="cuda")
    grads = {n: torch.zeros(shape[n], dtype=torch.float64, device="cuda") for n in "qkv"}
    for b in range(case["batch"]):
        see = _visible(case, st["mask"], b)
        some = see.any(dim=1)
        if not bool(some.any()):
            continue
        seen = see[some]
        for h in range(case["heads"]):
            q, k, v = (st[n][b, h if n == "q" else h // per].detach().double().requires_grad_() for n in "qkv")
            w = (q[some] @ k.t() / math.sqrt(case["dim"])).masked_fill(~seen, -math.inf)
            o = torch.exp(w - torch.logsumexp(w, dim=1, keepdim=True)) @ v
            out[b, h, some] = o.detach()
            if case["backward"]:
                for n, d in zip("qkv", torch.autograd.grad(o, (q, k, v), st["grad"][b, h][some].double())):
                    grads[n][b, h if n == "q" else h // per] += d
    if not case["backward"]:
        return {"out": out}
    return {"out": out, "dq": grads["q"], "dk": grads["k"], "dv": grads["v"]}


def _by_rows(case, most=1 << 27):
    n = max(1, most // case["vocab"])
    rows = case["batch"] * case["tokens"]
    return [slice(i, min(i + n, rows)) for i in range(0, rows, n)]


def _joined(case, parts):
    rows = (case["batch"], case["tokens"])
    return {n: torch.cat([p[n] for p in parts]).reshape(*rows, *parts[0][n].shape[1:]) for n in parts[0]}


def _exact_logprobs(case, st):
    rows, V = case["batch"] * case["tokens"], case["vocab"]
    flat = st["logits"].detach().reshape(rows, V)
    targets, g, ge = (st[n].reshape(rows) for n in ("targets", "grad", "grad_entropy"))
    parts = []
    for at in _by_rows(case):
        x = flat[at].double().requires_grad_(case["backward"])
        logp = x / case["temperature"]
        logp = logp - torch.logsumexp(logp, dim=1, keepdim=True)
        t = targets[at]
        ok = (t != -100).double()
        lp = logp[torch.arange(len(t), device="cuda"), t.clamp(min=0)] * ok
        h = -(torch.exp(logp) * logp).sum(dim=1) * ok
        part = {"logprob": lp.detach(), "entropy": h.detach()}
        if case["top"]:
            part["top_logprobs"] = torch.sort(logp.detach(), dim=1, descending=True).values[:, :case["top"]]
        if case["backward"]:
            part["dlogits"], = torch.autograd.grad((lp, h), (x,), (g[at].double(), ge[at].double()))
        parts.append(part)
    got = _joined(case, parts)
    return dict(got, top_ids=None) if case["top"] else got


def _exact_distill(case, st):
    rows, V, T = case["batch"] * case["tokens"], case["vocab"], case["temperature"]
    flat, ids = st["logits"].detach().reshape(rows, V), st["ids"].reshape(rows, -1)
    values, g = st["values"].reshape(rows, -1).double() / T, st["grad"].reshape(rows).double()
    parts = []
    for at in _by_rows(case):
        x = flat[at].double().requires_grad_(case["backward"])
        logp = x / T - torch.logsumexp(x / T, dim=1, keepdim=True)
        t = values[at]
        logq = t - (st["lse"].reshape(rows, 1)[at].double() if case["tail"] else torch.logsumexp(t, dim=1, keepdim=True))
        q = torch.exp(logq)
        loss = (q * (logq - logp.gather(1, ids[at]))).sum(dim=1)
        if case["tail"] and case["k"] < V:
            rest = (1.0 - q.sum(dim=1)).clamp(min=0.0)
            given = torch.zeros(x.shape, dtype=torch.bool, device="cuda").scatter_(1, ids[at], True)
            left = torch.logsumexp(logp.masked_fill(given, -math.inf), dim=1)
            loss = loss + torch.xlogy(rest, rest) - rest * left
        loss = loss * T * T
        part = {"loss": loss.detach()}
        if case["backward"]:
            part["dlogits"], = torch.autograd.grad(loss, (x,), g[at])
        parts.append(part)
    return _joined(case, parts)


def exact(case, seed):
    st = prepare(case, seed)
    return dict(attention=_exact_attention, logprobs=_exact_logprobs, distill=_exact_distill)[case["kind"]](case, st)
