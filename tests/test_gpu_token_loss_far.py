"""Losses from logits far from 0: masks that are finite numbers, and temperatures and logits that make exponents large."""
import math

import pytest
import torch

import token_loss_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
READERS = 224              # threads of a CTA that read a row


def _near(got, want, tol, what):
    got = got.detach()
    past = got.isinf() & (want.abs() > torch.finfo(got.dtype).max) & (want.sign() == got.sign())      # past the type's range
    got = got.double()
    same = past | (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() / tol)
    assert bool((off <= 1).all()), (what, float(off.max()), int(off.argmax()))


def _value_tol(V, exact):
    """`oracle.value_tol`, where the exact numbers are."""
    return oracle.U * (2 * oracle.sum_steps(V) + 4 * math.log(V) + 8 * exact.abs().masked_fill(exact.isinf(), 0.0) + 8)


def _logprobs(x, t, temperature, entropy=True, top=0):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import token_logprobs
    V = x.shape[-1]
    gen = torch.Generator(device="cuda").manual_seed(V)
    g, ge = (torch.randn(t.shape, generator=gen, device="cuda") for _ in range(2))
    ge = ge * entropy
    x = x.detach().requires_grad_()
    r = token_logprobs(x, t, temperature=temperature, entropy=entropy, top=top)
    # log_softmax takes the largest number out first: nothing cancels behind it
    wide = x.detach().double().requires_grad_()
    logp = torch.log_softmax(wide / temperature, -1)
    lp = logp.gather(-1, t.unsqueeze(-1)).squeeze(-1)
    ent = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0.0)).sum(-1)
    dx, = torch.autograd.grad((lp * g.double()).sum() + (ent * ge.double()).sum(), wide)
    lp, ent, logp = lp.detach(), ent.detach(), logp.detach()
    _near(r.logprob, lp, _value_tol(V, lp), "logprob")
    if entropy:
        _near(r.entropy, ent, _value_tol(V, ent), "entropy")
    if top:
        order = torch.sort(x.detach().float(), dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(r.top_ids, order)
        best = logp.gather(-1, order)
        _near(r.top_logprobs, best, _value_tol(V, best), "top")
    got, = torch.autograd.grad((r.logprob, r.entropy) if entropy else (r.logprob,), (x,), (g, ge) if entropy else (g,))
    size = (g.abs() + ge.abs()).double().unsqueeze(-1)
    _near(got, dx, oracle.grad_tol(dx, x.dtype, V, size, temperature), "dlogits")
    cuda_ops.check_error_flag(x.device)


def _distill(x, ids, values, lse, temperature):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import distill_loss
    V, K = x.shape[-1], ids.shape[-1]
    g = torch.randn(x.shape[:-1], generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
    x = x.detach().requires_grad_()
    loss = distill_loss(x, ids, values, temperature=temperature, teacher_logsumexp=lse)
    wide = x.detach().double().requires_grad_()
    logp = torch.log_softmax(wide / temperature, -1)
    v = values.double() / temperature
    logq = v - (torch.logsumexp(v, -1) if lse is None else lse.double()).unsqueeze(-1)
    q = logq.exp()
    want = (q * (logq - logp.gather(-1, ids))).sum(-1)
    if lse is not None:
        rest = (1 - q.sum(-1)).clamp(min=0)
        given = torch.zeros_like(x, dtype=torch.bool).scatter_(-1, ids, True)
        left = torch.logsumexp(logp.masked_fill(given, -1e300), -1)
        some = (rest > 0) & (left > -60)                 # the student has other tokens
        want = want + torch.where(some, torch.xlogy(rest, rest) - rest * torch.where(some, left, 0.0), 0.0)
    want = want * temperature ** 2
    dx, = torch.autograd.grad((want * g.double()).sum(), wide)
    # as for rows near 0: the teacher's exponents, the sums' relative errors, the terms of the sum over the teacher's tokens; and
    # the result's own rounding
    size = float(values.abs().max()) / temperature + math.log(V) + 20
    want = want.detach()
    _near(loss, want, oracle.U * ((4 * oracle.sum_steps(V) + K + 24 * size) * temperature ** 2 + 2 * want.abs()), "loss")
    got, = torch.autograd.grad(loss, (x,), (g,))
    scale = g.abs().double().unsqueeze(-1) * temperature ** 2
    _near(got, dx, oracle.grad_tol(dx, x.dtype, V, scale * (1 + (K + 2 * size) / 64), temperature), "dlogits")
    cuda_ops.check_error_flag(x.device)


def _hidden(where, V, vec):
    at = torch.arange(V, device="cuda")
    return {"one": at == V // 2, "head": at < 3, "tail": at >= V - 3, "ends": (at < 3) | (at >= V - 3),
            "threads": at // vec % READERS < 20, "batch": at < 4 * READERS * vec, "parts": (at < V // 4) | (at >= V - V // 4),
            "most": (at != 1) & (at != V - 2) & (at != V // 2), "half": at % 2 == 0, "nearly all": at != V - 1}[where]


@pytest.mark.parametrize("by", [-1e10, -1e30, "bf16", "fp32"])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 1.5, 2.0, 3.0])
@pytest.mark.parametrize("where", ["one", "head", "tail", "ends", "threads", "batch", "parts", "most", "half", "nearly all"])
def test_finite_masks(where, temperature, by):
    g = torch.Generator(device="cuda").manual_seed(11)
    value = {"bf16": torch.finfo(torch.bfloat16).min, "fp32": torch.finfo(torch.float32).min}.get(by, by)
    for dtype, V, rows in ((torch.bfloat16, 8197, 3), (torch.float32, 4101, 3), (torch.bfloat16, 1003, 300), (torch.float32, 9003, 150)):
        if dtype == torch.bfloat16 and by == "fp32":
            continue                                     # rounds to -inf
        wide = (torch.randn(rows, V + 5, generator=g, device="cuda") * 2.5).to(dtype)
        x = wide[:, 3:V + 3]                             # unaligned: elements in front of the first vector
        x = x.masked_fill_(_hidden(where, V, 16 // x.element_size()), value)
        left = (x[0] > value).nonzero().flatten()
        if len(left) == 0:
            continue                                     # rows of nothing else: below
        t = left[torch.randint(0, len(left), (rows,), generator=g, device="cuda")]
        t[0] = V // 2                                    # hidden in most of these
        _logprobs(x, t, temperature, True, 7)
        _logprobs(x, t, temperature, False)
        ids = left[torch.randint(0, len(left), (rows, 5), generator=g, device="cuda")]
        values = torch.randn(rows, 5, generator=g, device="cuda")
        _distill(x, ids, values, None, temperature)
        _distill(x, ids, values, torch.logsumexp(values / temperature, -1) + 0.5, temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("value", [-1e10, -1e30, 1e10, 1e30, -1.5e38, 1.5e38])
def test_rows_of_one_far_number(dtype, temperature, value):
    """All tokens are alike, however far: the uniform distribution."""
    g = torch.Generator(device="cuda").manual_seed(12)
    for rows, V in ((2, 5003), (160, 1001)):
        x = torch.full((rows, V), value, device="cuda").to(dtype)
        t = torch.randint(0, V, (rows,), generator=g, device="cuda")
        _logprobs(x, t, temperature, True, 3)
        _logprobs(x, t, temperature, False)
        ids = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(i))[:6] for i in range(rows)]).cuda()
        values = torch.randn(rows, 6, generator=g, device="cuda")
        _distill(x, ids, values, None, temperature)
        _distill(x, ids, values, torch.logsumexp(values / temperature, -1) + 0.5, temperature)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0])
def test_rows_of_lowest_values_have_no_token(dtype, temperature):
    from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs
    for rows, V in ((2, 5003), (160, 1001)):
        x = torch.full((rows, V), torch.finfo(dtype).min, dtype=dtype, device="cuda").requires_grad_()
        t = torch.zeros(rows, dtype=torch.int64, device="cuda")
        r = token_logprobs(x, t, temperature, entropy=True, top=2)
        assert bool((r.logprob == -math.inf).all()) and bool((r.entropy == 0).all()) and bool((r.top_logprobs == -math.inf).all())
        loss = distill_loss(x, t.view(-1, 1), torch.zeros(rows, 1, device="cuda"), temperature)
        assert bool((loss == math.inf).all())
        for d in torch.autograd.grad((r.logprob, r.entropy), (x,), (torch.ones(rows, device="cuda"),) * 2) + \
                torch.autograd.grad(loss, (x,), torch.ones(rows, device="cuda")):
            assert bool((d == 0).all())


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("rows,V", [(2, 20001), (170, 5001)])
@pytest.mark.parametrize("middle,temperature", [(2.0 ** 24 * math.log(2.0), 1.0), (2.0 ** 24 * math.log(2.0) * 3, 3.0),
                                                (2.0 ** 26, 1.0), (2.0 ** 27, 10.0), (2.0 ** 28, 64.0)])
def test_around_where_rows_are_far(sign, rows, V, middle, temperature):
    """Logits some 60 steps of 32 bits to either side of a number: exponents of all sizes, and maxima of threads, warps and CTAs
    on both sides of 2^24."""
    g = torch.Generator(device="cuda").manual_seed(13)
    middle = sign * middle
    step = 2.0 ** (math.floor(math.log2(abs(middle))) - 23)
    x = torch.full((rows, V), round(middle / step) * step, device="cuda")
    x = x + torch.randint(-60, 61, (rows, V), generator=g, device="cuda") * step
    x[:, ::7] = -math.inf
    t = torch.randint(0, V // 7, (rows,), generator=g, device="cuda") * 7 + 1
    _logprobs(x, t, temperature, True, 5)
    _logprobs(x, t, temperature, False)
    ids = torch.randint(0, V // 7, (rows, 9), generator=g, device="cuda") * 7 + 2
    values = torch.randn(rows, 9, generator=g, device="cuda")
    _distill(x, ids, values, None, temperature)
    _distill(x, ids, values, torch.logsumexp(values / temperature, -1) + 0.5, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1e-6, 1e-4, 1e-3])
def test_low_temperatures(dtype, temperature):
    g = torch.Generator(device="cuda").manual_seed(14)
    for rows, V in ((2, 5003), (160, 1001)):
        x = (torch.randn(rows, V, generator=g, device="cuda") * (3000.0 if dtype != torch.float32 else 30.0)).to(dtype)
        x[1, 5] = x[1, 500] = x[1].max()                 # two best
        best = x.float().argmax(-1)
        t = torch.where(torch.arange(rows, device="cuda") % 3 == 0, best, torch.randint(0, V, (rows,), generator=g, device="cuda"))
        _logprobs(x, t, temperature, True, 4)
        _logprobs(x, t, temperature, False)
