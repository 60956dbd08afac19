"""Log probabilities of given tokens and distillation on the CPU: the plain form, its gradients, and what is refused."""
import math

import pytest
import torch

import token_loss_oracle as oracle
from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs


def _case(seed, shape, k=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * 2.5
    t = torch.randint(0, shape[-1], shape[:-1], generator=g)
    teacher = torch.randn(shape, generator=g) * 2.5
    best = torch.topk(teacher, k, dim=-1)
    return g, x, t, best.indices, best.values, torch.logsumexp(teacher, dim=-1)


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_logprobs(temperature):
    g, x, t, *_ = _case(0, (2, 5, 37))
    t[0, 1] = -100
    x.requires_grad_()
    gl, ge = torch.randn(2, 5, generator=g), torch.randn(2, 5, generator=g)
    r = token_logprobs(x, t, temperature=temperature, entropy=True, top=4)
    lp, ent, logp, dx = oracle.logprobs(x, t, temperature, gl, ge)
    # 37 terms: sums and logarithms stay within 64 roundings of numbers below 32
    tol = 64 * 32 * oracle.U
    assert (r.logprob - lp).abs().max() < tol and (r.entropy - ent).abs().max() < tol
    assert torch.equal(r.top_ids, torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[..., :4])
    got, = torch.autograd.grad((r.logprob, r.entropy), (x,), (gl, ge))
    assert (got - dx).abs().max() < 4 * tol / temperature


def test_gradients_by_differences():
    g, x, t, ids, values, lse = _case(1, (3, 11), k=4)
    ids[1, 2] = ids[1, 3]
    lse = lse + 0.5
    x = x.double().requires_grad_()
    assert torch.autograd.gradcheck(lambda y: token_logprobs(y, t, temperature=0.8, entropy=True)[:2], (x,))
    assert torch.autograd.gradcheck(lambda y: distill_loss(y, ids, values, temperature=1.5), (x,))
    assert torch.autograd.gradcheck(lambda y: distill_loss(y, ids, values, teacher_logsumexp=lse), (x,))


@pytest.mark.parametrize("tail", [False, True])
def test_distill(tail):
    g, x, t, ids, values, lse = _case(2, (2, 3, 41))
    ids[0, 1, 2:] = -1
    ids[1, 2] = -1
    ids[1, 1, 0] = ids[1, 1, 5]
    lse = lse + 0.5 if tail else None
    x.requires_grad_()
    go = torch.randn(2, 3, generator=g)
    loss = distill_loss(x, ids, values, teacher_logsumexp=lse)
    want, dx = oracle.distill(x, ids, values, 1.0, lse, go)
    tol = 64 * 32 * oracle.U
    assert (loss - want).abs().max() < tol and loss[1, 2] == 0
    got, = torch.autograd.grad(loss, (x,), (go,))
    assert (got - dx).abs().max() < 4 * tol


def test_rows_without_any_token():
    x = torch.zeros(3, 9)
    x[0] = -math.inf
    x[1, 3:] = -math.inf
    x.requires_grad_()
    r = token_logprobs(x, torch.tensor([0, 5, -100]), entropy=True, top=2)
    assert r.logprob.tolist() == [-math.inf, -math.inf, 0.0] and r.entropy[0] == 0 and r.entropy[2] == 0
    assert abs(float(r.entropy[1]) - math.log(3)) < 1e-6
    dx, = torch.autograd.grad(r.entropy.sum(), (x,))
    assert bool(dx.isfinite().all())


def test_what_is_refused():
    x, t = torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64)
    ids, values = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for bad in (lambda: token_logprobs(x.to(torch.int32), t), lambda: token_logprobs(torch.zeros(()), t),
                lambda: token_logprobs(x, t[:1]), lambda: token_logprobs(x, t.float()),
                lambda: token_logprobs(x, t, temperature=0.0), lambda: token_logprobs(x, t, temperature=math.nan),
                lambda: token_logprobs(x, t, temperature=-1.0), lambda: token_logprobs(x, t, top=10),
                lambda: token_logprobs(torch.zeros(2, 99), t, top=33), lambda: token_logprobs(x, t, top=-1),
                lambda: token_logprobs(x, t + 9), lambda: token_logprobs(x, t - 1),
                lambda: distill_loss(x, ids[0], values[0]), lambda: distill_loss(x, ids, values[:, :2]),
                lambda: distill_loss(x, ids.float(), values), lambda: distill_loss(x, ids, ids),
                lambda: distill_loss(x, ids[:, :0], values[:, :0]), lambda: distill_loss(x, ids + 9, values),
                lambda: distill_loss(x, ids, values, temperature=math.inf),
                lambda: distill_loss(x, ids, values, teacher_logsumexp=values),
                lambda: distill_loss(x, ids.expand(2, 3).repeat(1, 400), values.repeat(1, 400))):
        with pytest.raises(RuntimeError):
            bad()
    # ids of other whole types, and negative ones as padding
    assert token_logprobs(x, t.int()).logprob.shape == (2,) and bool((distill_loss(x, ids - 1, values) == 0).all())
