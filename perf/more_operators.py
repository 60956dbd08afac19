"""Operators of preference finetuning and of the optimizer behind it, each with its plain form: the loss of preferred over rejected
sequences, the clipped policy loss with a KL term, the norm of all gradients, and an AdamW step over many tensors with states in 32
or in 8 bits.

A case is one call of an operator on seeded data and, for the losses, the gradient of the logits for a given gradient of the loss:

``preference``  logits ``[2 pairs, tokens, vocab]``, preferred sequences first; prompts and padding have no target.
``policy``      logits ``[batch, tokens, vocab]`` with the log probabilities that the tokens were drawn at, advantages, and the log
                probabilities of a reference model.
``norm``        gradients of ``repeat`` times the tensors of ``shapes``.
``adamw``       the same tensors with gradients and moments; ``bits`` of the moments, ``master``: what is kept of 16-bit parameters
                beside themselves (``rest``: the 16 bits below bf16; ``fp32``: a copy in 32 bits; ``none``).

Moments (and what is kept beside the parameters) of all tensors lie one behind the other, each tensor's at a multiple of 256.
8-bit moments are e4m3 and e5m2 numbers with a power of two for each 256, rounded up or down at random: by a hash of the element's
place, the step and a seed.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BLOCK = 256
BETAS, EPS, LR = (0.9, 0.999), 1e-8, 2e-4
CLIP = (0.2, 0.28)
LOW = 32                 # a block's power of two is held above 2^(32 - 127)

LORA_13B = "8x5120 5120x8 8x5120 5120x8 8x5120 5120x8"
LAYER_7B = "4096 4096 4096x4096 4096x4096 4096x4096 4096x4096 4096x11008 11008x4096 11008x4096"


def listed():
    return [
        # a test model's pair, 32-bit logits: the smallest call, where launches and host time count
        dict(name="preference-1-pair", kind="preference", pairs=1, tokens=24, vocab=1000, form="sigmoid", beta=0.1, smoothing=0.0,
             margin=0.0, reference=True, average=False, more=False, dtype="float32"),
        # the micro-batch of the QLoRA benchmark (4 x 512 tokens) as two pairs, with a likelihood term of the preferred sequences
        dict(name="preference-7b", kind="preference", pairs=2, tokens=512, vocab=32000, form="sigmoid", beta=0.1, smoothing=0.1,
             margin=0.0, reference=True, average=False, more=True, dtype="bfloat16"),
        # the 128k vocabulary, log probabilities averaged over the tokens, no reference model
        dict(name="preference-128k", kind="preference", pairs=1, tokens=1021, vocab=128256, form="ipo", beta=0.1, smoothing=0.0,
             margin=0.0, reference=False, average=True, more=False, dtype="bfloat16"),
        # a few tokens of an odd vocabulary (three tokens added) in fp16, one update a batch
        dict(name="policy-37-tokens", kind="policy", batch=1, tokens=37, vocab=32003, kl=0.0, drawn=False, each=False,
             temperature=1.0, dtype="float16"),
        # a micro-batch of completions with one advantage for each, near a reference model
        dict(name="policy-7b", kind="policy", batch=4, tokens=512, vocab=32000, kl=0.04, drawn=True, each=False, temperature=1.0,
             dtype="bfloat16"),
        # the 128k vocabulary, sampled at 0.7, an advantage for each token
        dict(name="policy-128k", kind="policy", batch=2, tokens=1024, vocab=128256, kl=0.1, drawn=True, each=True, temperature=0.7,
             dtype="bfloat16"),
        # adapters of a 13B model's projections: 240 tensors of 40960
        dict(name="norm-lora-13b", kind="norm", shapes=LORA_13B, repeat=40, dtype="bfloat16"),
        # a whole decoder layer of the 7B model, as layer-wise finetuning trains it
        dict(name="norm-layer-7b", kind="norm", shapes=LAYER_7B, repeat=1, dtype="bfloat16"),
        # a test model's adapters in 32 bits: the smallest step
        dict(name="adamw-8-tensors", kind="adamw", shapes="8x256 256x8 8x256 688x8", repeat=2, bits=32, master="none", clip=True,
             decay=0.0, dtype="float32"),
        dict(name="adamw-lora-13b", kind="adamw", shapes=LORA_13B, repeat=40, bits=32, master="rest", clip=True, decay=0.0,
             dtype="bfloat16"),
        # odd sizes in fp16 with 32-bit copies, 8-bit moments
        dict(name="adamw-odd-8-bit", kind="adamw", shapes="1 7 255 257 4099 333x1031 2049x515", repeat=9, bits=8, master="fp32",
             clip=False, decay=0.1, dtype="float16"),
        dict(name="adamw-layer-7b-8-bit", kind="adamw", shapes=LAYER_7B, repeat=1, bits=8, master="rest", clip=True, decay=0.01,
             dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["preference", "preference", "policy", "policy", "norm", "adamw", "adamw", "adamw"])
    if kind in ("preference", "policy"):
        vocab = _log_int(rng, 500, 130000)
        rows = _log_int(rng, 2, min(2048, int(1.2e8 / vocab)))
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        if kind == "preference":
            pairs = min(rng.choice([1, 1, 2, 3, 5]), max(1, rows // 4))
            form = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
            return dict(kind=kind, pairs=pairs, tokens=max(2, rows // (2 * pairs)), vocab=vocab, form=form,
                        beta=rng.choice([0.05, 0.1, 0.5]), smoothing=rng.choice([0.0, 0.0, 0.2]) if form == "sigmoid" else 0.0,
                        margin=rng.choice([0.0, 0.5]) if form == "sigmoid" else 0.0, reference=rng.random() < 0.7,
                        average=form == "ipo" or rng.random() < 0.3, more=rng.random() < 0.4, dtype=dtype)
        batch = rng.choice([1, 1, 2, 3])
        return dict(kind=kind, batch=batch, tokens=max(2, rows // batch), vocab=vocab, kl=rng.choice([0.0, 0.04, 0.5]),
                    drawn=rng.random() < 0.8, each=rng.random() < 0.5, temperature=rng.choice([1.0, 1.0, 0.7, 1.5]), dtype=dtype)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    most, shapes = _log_int(rng, 1000, 5e7), []
    for _ in range(rng.choice([1, 3, 8])):
        n = _log_int(rng, 1, most)
        rows = _log_int(rng, 1, min(n, 64))
        shapes.append("%dx%d" % (rows, max(1, n // rows)))
    repeat = min(rng.choice([1, 2, 30, 100]), max(1, int(6e7 / sum(_count(s) for s in shapes))))
    case = dict(kind=kind, shapes=" ".join(shapes), repeat=repeat, dtype=dtype)
    if kind == "norm":
        return case
    master = {"bfloat16": ["rest", "fp32", "none"], "float16": ["fp32", "none"], "float32": ["none"]}[dtype]
    return dict(case, bits=rng.choice([32, 8]), master=rng.choice(master), clip=rng.random() < 0.6, decay=rng.choice([0.0, 0.01, 0.1]))


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _sequences(batch, tokens, vocab, g):
    """Tokens of completions: -100 for a prompt of up to half, for padding of up to a quarter, and for the last position."""
    t = torch.randint(0, vocab, (batch, tokens), generator=g, device="cuda")
    at = torch.arange(tokens, device="cuda").view(1, -1)
    start = (_uniform(g, batch, 1) * (tokens // 2)).long()
    end = tokens - 1 - (_uniform(g, batch, 1) * (tokens // 4)).long()
    return t.masked_fill((at < start) | (at >= end.clamp(min=1)), -100)


def _logits(targets, vocab, g):
    """Scores in which the tokens that were drawn are likely ones."""
    x = _normal(g, *targets.shape, vocab).mul_(2.5)
    lift = 6.0 + 4.0 * _uniform(g, *targets.shape, 1)
    return x.scatter_add_(2, targets.clamp(min=0).unsqueeze(2), lift)


def _scored(x, targets, temperature):
    """Log probabilities of the targets in 64 bits' differences, 0 where there is none."""
    at = targets.clamp(min=0).unsqueeze(2)
    got = (x.gather(2, at).double() / temperature).squeeze(2) - torch.logsumexp(x.float() / temperature, dim=2).double()
    return torch.where(targets != -100, got, 0.0)


def _prepare_preference(case, seed):
    g = _generator(seed)
    targets = _sequences(2 * case["pairs"], case["tokens"], case["vocab"], g)
    logits = _logits(targets, case["vocab"], g).to(DTYPES[case["dtype"]])
    st = dict(logits=logits.requires_grad_(), targets=targets, reference=None, grad=_normal(g, case["pairs"]),
              grad_more=0.01 * _uniform(g, 2 * case["pairs"]) if case["more"] else None)
    if case["reference"]:
        total = _scored(logits.detach(), targets, 1.0).sum(dim=1)
        count = (targets != -100).sum(dim=1)
        if case["average"]:
            total, count = total / count, torch.ones_like(total)
        st["reference"] = (total + 0.4 * count.sqrt() * _normal(g, 2 * case["pairs"])).float()
    return st


def _prepare_policy(case, seed):
    g = _generator(seed)
    targets = _sequences(case["batch"], case["tokens"], case["vocab"], g)
    logits = _logits(targets, case["vocab"], g).to(DTYPES[case["dtype"]])
    rows = (case["batch"], case["tokens"])
    lp = _scored(logits, targets, case["temperature"])
    st = dict(logits=logits.requires_grad_(), targets=targets, old=None, ref=None, grad=_normal(g, *rows).abs(),
              advantages=_normal(g, case["batch"], case["tokens"] if case["each"] else 1))
    if case["drawn"]:
        d = 0.2 * _normal(g, *rows)                       # log ratios, none within 0.001 of a border
        for border in (math.log(1 - CLIP[0]), math.log(1 + CLIP[1])):
            d = torch.where((d - border).abs() < 0.001, d + 0.003, d)
        st["old"] = (lp - d).float()
    if case["kl"]:
        st["ref"] = (lp + 0.3 * _normal(g, *rows)).float()
    return st


def _count(shape):
    return math.prod(int(n) for n in shape.split("x"))


def _places(case):
    """Where each tensor begins, its shape, and where all end."""
    shapes = [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split()] * case["repeat"]
    at, places = 0, []
    for s in shapes:
        places.append((at, s))
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return places, at


def _views(flat, places):
    return [flat[at:at + math.prod(s)].view(s) for at, s in places]


def _real(places, n):
    """True for the elements of tensors, False for what fills their last 256."""
    edge = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    one = torch.ones(len(places), dtype=torch.int32, device="cuda")
    edge.index_add_(0, torch.tensor([at for at, _ in places], device="cuda"), one)
    edge.index_add_(0, torch.tensor([at + math.prod(s) for at, s in places], device="cuda"), -one)
    return edge.cumsum(0, dtype=torch.int32)[:n] > 0


def _gradients(case, places, n, g):
    """Gradients, all tensors' behind one another: each 256 of a size of their own, a few elements without any."""
    size = torch.exp(1.5 * _normal(g, n // BLOCK, 1)) * 1e-3
    x = _normal(g, n // BLOCK, BLOCK) * size
    x = x * (_uniform(g, n // BLOCK, BLOCK) > 0.02)
    return (x.view(-1) * _real(places, n)).to(DTYPES[case["dtype"]])


def _prepare_norm(case, seed):
    places, n = _places(case)
    flat = _gradients(case, places, n, _generator(seed))
    return dict(flat=flat, grads=_views(flat, places))


def _prepare_adamw(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    places, n = _places(case)
    real = _real(places, n)
    flat_g = _gradients(case, places, n, g)
    seen = flat_g.float()
    m = (0.5 * seen + 0.2 * _normal(g, n) * seen.abs()) * real
    v = (seen * (0.3 + _uniform(g, n))).square() + 1e-9 * seen.abs()
    wide = _normal(g, n).mul_(0.02) * real
    st = dict(flat_g=flat_g, grads=_views(flat_g, places), m_scale=None, v_scale=None, rest=None, norm=None, seed=int(seed) & 0xFFFF,
              step=(torch.rand(1, generator=g, device="cuda") * 2000).long())
    if case["master"] == "rest":
        st["flat"], st["rest"] = _split(wide)
    else:
        st["flat"] = wide.to(dt)
        st["rest"] = wide if case["master"] == "fp32" else None
    st["params"] = _views(st["flat"], places)
    if case["bits"] == 8:
        key = torch.zeros(n, dtype=torch.int64, device="cuda")
        st["m"], st["m_scale"] = _held_m(m, key + 0x8000)
        st["v"], st["v_scale"] = _held_v(v, key + 0x8000)
    else:
        st["m"], st["v"] = m, v
    if case["clip"]:
        st["norm"] = 2.0 * _norm(flat_g) * _uniform(g, 1).view(()) + 0.1
    return st


def prepare(case, seed):
    make = dict(preference=_prepare_preference, policy=_prepare_policy, norm=_prepare_norm, adamw=_prepare_adamw)[case["kind"]]
    with torch.no_grad():
        return dict(make(case, seed), case=case)


# ---- the plain forms, in 32 bits ------------------------------------------------------------------------------------------
def _log_softmax(logits, temperature):
    y = logits.float() / temperature
    y = y - y.amax(dim=-1, keepdim=True)
    return y - torch.log(torch.exp(y).sum(dim=-1, keepdim=True))


def _d_logits(logp, targets, by, temperature, dtype):
    """``by [...]`` times the gradient of the targets' log probabilities."""
    d = torch.exp(logp) * -by.unsqueeze(2)
    return (d.scatter_add_(2, targets.clamp(min=0).unsqueeze(2), by.unsqueeze(2)) / temperature).to(dtype)


def _plain_preference(st):
    case, targets, P, b = st["case"], st["targets"], st["case"]["pairs"], st["case"]["beta"]
    real = targets != -100
    logp = _log_softmax(st["logits"], 1.0)
    s = torch.where(real, logp.gather(2, targets.clamp(min=0).unsqueeze(2)).squeeze(2), 0.0).double().sum(dim=1)
    share = real.sum(dim=1).clamp(min=1).double().reciprocal() if case["average"] else torch.ones_like(s)
    s = s * share
    h = s if st["reference"] is None else s - st["reference"].double()
    h = h[:P] - h[P:]
    if case["form"] == "ipo":
        loss, slope = (h - 1 / (2 * b)).square(), 2 * (h - 1 / (2 * b))
    elif case["form"] == "hinge":
        loss, slope = (1 - b * h).clamp(min=0), torch.where(b * h < 1, -b, 0.0)
    else:
        z, e = b * h - case["margin"], case["smoothing"]
        loss = (1 - e) * torch.log1p(torch.exp(-z)) + e * torch.log1p(torch.exp(z))
        up = 1 / (1 + torch.exp(-z))
        slope = b * (e * up - (1 - e) * (1 - up))
    by = st["grad"] * slope
    by = torch.cat([by, -by])
    if st["grad_more"] is not None:
        by = by + st["grad_more"]
    by = torch.where(real, (by * share).unsqueeze(1), 0.0).float()
    return {"loss": loss.float(), "logprob": s.float(), "dlogits": _d_logits(logp, targets, by, 1.0, st["logits"].dtype)}


def _plain_policy(st):
    case, targets = st["case"], st["targets"]
    real = targets != -100
    logp = _log_softmax(st["logits"], case["temperature"])
    lp = torch.where(real, logp.gather(2, targets.clamp(min=0).unsqueeze(2)).squeeze(2), 0.0)
    old = lp if st["old"] is None else st["old"]
    a, ratio = st["advantages"], torch.exp(lp - old)
    held = ratio.clamp(1 - CLIP[0], 1 + CLIP[1])
    loss = -torch.minimum(ratio * a, held * a)
    clipped = (ratio * a > held * a) & real
    slope = torch.where(clipped, 0.0, -a * ratio)
    kl = torch.zeros_like(lp)
    if st["ref"] is not None:
        d = (st["ref"] - lp).double()
        kl = (torch.expm1(d) - d).float()
        loss, slope = loss + case["kl"] * kl, slope - case["kl"] * torch.expm1(d).float()
    loss, kl = torch.where(real, loss, 0.0), torch.where(real, kl, 0.0)
    by = torch.where(real, slope * st["grad"], 0.0)
    return {"loss": loss, "logprob": lp, "kl": kl, "clipped": clipped,
            "dlogits": _d_logits(logp, targets, by, case["temperature"], st["logits"].dtype)}


def _norm(flat):
    return flat.double().square().sum().sqrt().float()


def _plain_norm(st):
    return {"norm": _norm(st["flat"])}


def _split(wide):
    """32-bit numbers as the nearest bf16 (halves up) and the 16 bits that this leaves."""
    bits = wide.view(torch.int32).long() & 0xFFFFFFFF
    high = (bits + 0x8000) >> 16
    rest = (bits - (high << 16)).to(torch.int16)
    return _as_int16(high & 0xFFFF).view(torch.bfloat16), rest


def _as_int16(x):
    return torch.where(x >= 0x8000, x - 0x10000, x).to(torch.int16)


def _joined(high, rest):
    bits = ((high.view(torch.int16).long() << 16) + rest.long()) & 0xFFFFFFFF
    return torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32)


def _exponents(x):
    """The exponent of the largest of each 256, as in a 32-bit number's bits."""
    top = x.abs().view(-1, BLOCK).amax(dim=1)
    return (top.view(torch.int32) >> 23).clamp(LOW, 254)


def _power(e):
    """2^e, |e| up to 126."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _times(x, e):
    return (x.view(-1, BLOCK) * _power(e).unsqueeze(1)).view(-1)


def _held_m(m, chance):
    """e4m3 of m, the largest of each 256 in [2^7, 2^8); ``chance``: 16 random bits for each."""
    e = _exponents(m)
    bits = (_times(m.abs(), 134 - e) * 2.0 ** -120).view(torch.int32).long()
    code = (bits + (chance << 4) + 8) >> 20
    return torch.where(m < 0, code + 128, code).to(torch.uint8).view(torch.float8_e4m3fn), e.to(torch.uint8)


def _held_v(v, chance):
    """e5m2 of v, the largest of each 256 in [2^14, 2^15); what is not 0 does not become 0."""
    e = _exponents(v)
    bits = (_times(v, 141 - e) * 2.0 ** -112).view(torch.int32).long()
    code = (bits + (chance << 5) + 16) >> 21
    return torch.where(v > 0, code.clamp(min=1), code).to(torch.uint8).view(torch.float8_e5m2), e.to(torch.uint8)


def _mixed(x):
    """Bits of a hash of 32-bit numbers (in 64)."""
    for shift, by in ((16, 0xBB67AE85), (15, 0x6A09E667)):
        x = ((x ^ (x >> shift)) * by) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _chances(n, step, seed):
    """16 random bits for each moment of each element at step number ``step``."""
    key = _mixed((_mixed(step & 0xFFFFFFFF) + seed * 0x9E3779B1) & 0xFFFFFFFF)
    at = torch.arange(n, device="cuda")
    x = _mixed(((at & 0xFFFFFFFF) * 0x9E3779B1 + (at >> 32) * 0xBB67AE85 + key) & 0xFFFFFFFF)
    return x & 0xFFFF, x >> 16


def _plain_adamw(st):
    case, n, (b1, b2) = st["case"], st["flat"].numel(), BETAS
    st["step"] += 1
    t = st["step"].double()
    rate, root = (LR / (1 - b1 ** t)).float(), (1 - b2 ** t).rsqrt().float()
    g = st["flat_g"].float()
    if case["clip"]:
        g = g * (1.0 / (st["norm"] + 1e-6)).clamp(max=1.0)
    m, v = st["m"], st["v"]
    if case["bits"] == 8:
        m, v = _times(m.float(), st["m_scale"].int() - 134), _times(v.float(), st["v_scale"].int() - 141)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    p = st["flat"].float()
    if st["rest"] is not None:
        p = _joined(st["flat"], st["rest"]) if case["master"] == "rest" else st["rest"]
    p = p * (1 - LR * case["decay"]) - (m * rate) / (v.sqrt() * root + EPS)
    if case["bits"] == 8:
        for_m, for_v = _chances(n, st["step"], st["seed"])
        (m, e), (v, f) = _held_m(m, for_m), _held_v(v, for_v)
        st["m_scale"].copy_(e)
        st["v_scale"].copy_(f)
    st["m"].copy_(m)
    st["v"].copy_(v)
    if case["master"] == "rest":
        p, rest = _split(p)
        st["rest"].copy_(rest)
    elif case["master"] == "fp32":
        st["rest"].copy_(p)
    st["flat"].copy_(p)
    return _updated(st)


def _updated(st):
    got = {"params": st["flat"], "m": st["m"], "v": st["v"], "step": st["step"]}
    more = {"rest": st["rest"], "m_scale": st["m_scale"], "v_scale": st["v_scale"]}
    return dict(got, **{k: x for k, x in more.items() if x is not None})


# ---- the framework's operators ----------------------------------------------------------------------------------------
def _own_preference(st):
    from ipex_llm_b200.ops.preference import preference_loss
    case = st["case"]
    r = preference_loss(st["logits"], st["targets"], st["reference"], beta=case["beta"], form=case["form"],
                        label_smoothing=case["smoothing"], margin=case["margin"], average=case["average"])
    more = st["grad_more"] is not None
    dx, = torch.autograd.grad((r.loss, r.logprob) if more else (r.loss,), (st["logits"],),
                              (st["grad"], st["grad_more"]) if more else (st["grad"],))
    return {"loss": r.loss.detach(), "logprob": r.logprob.detach(), "dlogits": dx}


def _own_policy(st):
    from ipex_llm_b200.ops.preference import policy_loss
    case = st["case"]
    r = policy_loss(st["logits"], st["targets"], st["advantages"], old_logprobs=st["old"], ref_logprobs=st["ref"], clip=CLIP,
                    kl_weight=case["kl"], temperature=case["temperature"])
    dx, = torch.autograd.grad(r.loss, (st["logits"],), (st["grad"],))
    return {"loss": r.loss.detach(), "logprob": r.logprob, "kl": r.kl, "clipped": r.clipped, "dlogits": dx}


def _own_norm(st):
    from ipex_llm_b200.ops.adamw import grad_norm
    return {"norm": grad_norm(st["grads"])}


def _own_adamw(st):
    from ipex_llm_b200.ops.adamw import adamw_step
    adamw_step(st["params"], st["grads"], st["m"], st["v"], st["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=st["case"]["decay"],
               exp_avg_scale=st["m_scale"], exp_avg_sq_scale=st["v_scale"], rest=st["rest"], grad_norm=st["norm"],
               max_grad_norm=1.0 if st["case"]["clip"] else 0.0, seed=st["seed"])
    return _updated(st)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(preference=_own_preference, policy=_own_policy, norm=_own_norm, adamw=_own_adamw)[kind](state)
    with torch.no_grad():
        return dict(preference=_plain_preference, policy=_plain_policy, norm=_plain_norm, adamw=_plain_adamw)[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if case["kind"] in ("preference", "policy"):
        rows = case.get("batch", 2 * case.get("pairs", 0)) * case["tokens"]
        # about 5 / 8 of the positions have a target: a prompt of a quarter and padding of an eighth on average
        logits = rows * case["vocab"]
        return {"bytes": logits * size * 1.625 + rows * 24, "flops": logits * 5.0}
    n = sum(_count(s) for s in case["shapes"].split()) * case["repeat"]
    if case["kind"] == "norm":
        return {"bytes": n * size, "flops": 2.0 * n}
    each = 3 * size + {"none": 0, "rest": 4, "fp32": 8}[case["master"]] + (16 if case["bits"] == 32 else 4 + 4 / BLOCK)
    if case["master"] == "fp32":
        each -= size                                      # the 16-bit parameters are only written
    return {"bytes": n * each, "flops": 16.0 * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_logprobs(x, targets, temperature):
    """Log probabilities [rows] of rows that have a target, from x [rows, vocab] in 64 bits."""
    return (x.gather(1, targets.unsqueeze(1)).squeeze(1) / temperature) - torch.logsumexp(x / temperature, dim=1)


def _exact_rows(logits, targets, temperature, by=None):
    """Over the rows with a target, a GB at a time: their log probabilities, or with ``by`` those rows of its gradient."""
    flat, t = logits.detach().reshape(-1, logits.shape[-1]), targets.reshape(-1)
    rows = (t != -100).nonzero().squeeze(1)
    out = torch.zeros(t.shape if by is None else flat.shape, dtype=torch.float64, device="cuda")
    for part in rows.split(max(1, (1 << 27) // flat.shape[1])):
        x = flat[part].double().requires_grad_(by is not None)
        lp = _exact_logprobs(x, t[part], temperature)
        out[part] = lp if by is None else torch.autograd.grad(lp, (x,), (by.reshape(-1)[part],))[0]
    return out.view(targets.shape if by is None else logits.shape)


def _exact_preference(case, st):
    P, real = case["pairs"], st["targets"] != -100
    lp = _exact_rows(st["logits"], st["targets"], 1.0).requires_grad_()
    s = lp.sum(dim=1)
    if case["average"]:
        s = s / real.sum(dim=1).clamp(min=1)
    gap = s - (0 if st["reference"] is None else st["reference"].double())
    gap = gap[:P] - gap[P:]
    if case["form"] == "ipo":
        loss = (gap - 0.5 / case["beta"]) ** 2
    elif case["form"] == "hinge":
        loss = torch.relu(1 - case["beta"] * gap)
    else:
        z = case["beta"] * gap - case["margin"]
        loss = -((1 - case["smoothing"]) * torch.nn.functional.logsigmoid(z) + case["smoothing"] * torch.nn.functional.logsigmoid(-z))
    total = (loss * st["grad"].double()).sum()
    if case["more"]:
        total = total + (s * st["grad_more"].double()).sum()
    by, = torch.autograd.grad(total, (lp,))
    return {"loss": loss.detach(), "logprob": s.detach(), "dlogits": _exact_rows(st["logits"], st["targets"], 1.0, by)}


def _exact_policy(case, st):
    T, real = case["temperature"], st["targets"] != -100
    lp = _exact_rows(st["logits"], st["targets"], T).requires_grad_()
    ratio = torch.exp(lp - (lp.detach() if st["old"] is None else st["old"].double()))
    a = st["advantages"].double()
    gain = torch.minimum(ratio * a, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * a)
    kl = torch.zeros_like(lp)
    if case["kl"]:
        d = st["ref"].double() - lp
        kl = torch.exp(d) - d - 1
    loss = torch.where(real, case["kl"] * kl - gain, 0.0)
    by, = torch.autograd.grad((loss * st["grad"].double()).sum(), (lp,))
    return {"loss": loss.detach(), "logprob": lp.detach(), "kl": torch.where(real, kl, 0.0).detach(), "clipped": None,
            "dlogits": _exact_rows(st["logits"], st["targets"], T, by)}


def _exact_norm(case, st):
    return {"norm": torch.linalg.vector_norm(st["flat"].double())}


def _exact_adamw(case, st):
    t, (b1, b2) = int(st["step"]) + 1, BETAS
    g = st["flat_g"].double()
    if case["clip"]:
        g = g * min(1.0, 1.0 / (float(st["norm"]) + 1e-6))
    m, v = st["m"].double(), st["v"].double()
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK) * torch.exp2(st["m_scale"].double() - 134).unsqueeze(1)).view(-1)
        v = (v.view(-1, BLOCK) * torch.exp2(st["v_scale"].double() - 141).unsqueeze(1)).view(-1)
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    p = {"none": st["flat"], "fp32": st["rest"]}.get(case["master"])
    p = _joined(st["flat"], st["rest"]).double() if p is None else p.double()
    p = p - LR * case["decay"] * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    wide = case["bits"] == 32
    got = {"params": p, "m": m if wide else None, "v": v if wide else None, "step": None}
    if case["master"] != "none":
        got["rest"] = p if case["master"] == "fp32" else None
    return got if wide else dict(got, m_scale=None, v_scale=None)


def exact(case, seed):
    st = prepare(case, seed)
    return dict(preference=_exact_preference, policy=_exact_policy, norm=_exact_norm, adamw=_exact_adamw)[case["kind"]](case, st)
