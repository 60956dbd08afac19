"""Preference and policy losses on the CPU, against their definitions in 64 bits and against differences."""
import math

import pytest
import torch

import preference_oracle as oracle
from ipex_llm_b200.ops.preference import policy_loss, preference_loss


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _preference(seed=0, pairs=2, tokens=9, V=31, dtype=torch.float64):
    g = _gen(seed)
    x = (torch.randn(2 * pairs, tokens, V, generator=g, dtype=torch.float64) * 2).to(dtype)
    t = torch.randint(0, V, (2 * pairs, tokens), generator=g)
    t[0, :4] = t[1, 6:] = t[2, 0] = -100
    return x, t, torch.randn(2 * pairs, generator=g, dtype=torch.float64) * 3 - 20


FORMS = [dict(form="sigmoid"), dict(form="sigmoid", label_smoothing=0.3, margin=0.7), dict(form="hinge", beta=0.3), dict(form="ipo"),
         dict(form="ipo", average=True), dict(form="sigmoid", average=True, beta=2.0)]


@pytest.mark.parametrize("kw", FORMS)
@pytest.mark.parametrize("with_reference", [False, True])
@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
def test_preference_by_its_definition(kw, with_reference, dtype):
    x, t, ref = _preference(dtype=dtype)
    ref = ref if with_reference else None
    x.requires_grad_()
    g, gs = torch.randn(2, generator=_gen(5)), torch.randn(4, generator=_gen(6))
    got = preference_loss(x, t, ref, temperature=0.8, **kw)
    dx, = torch.autograd.grad((got.loss, got.logprob), x, (g.to(got.loss.dtype), gs.to(got.loss.dtype)))
    want = oracle.preference(x, t, ref, temperature=0.8, g=g, g_seq=gs, **kw)
    for a, (b, tol) in zip((got.loss, got.logprob, dx), want):
        assert a.shape == b.shape and ((a.detach().double() - b).abs() <= tol).all()


@pytest.mark.parametrize("kw", FORMS)
def test_preference_by_differences(kw):
    x, t, ref = _preference()
    x.requires_grad_()
    loss = preference_loss(x, t, ref, **kw).loss.sum()
    dx, = torch.autograd.grad(loss, x)
    d = torch.randn(x.shape, generator=_gen(3), dtype=torch.float64)
    h = 1e-6
    diff = (preference_loss(x + h * d, t, ref, **kw).loss.sum() - preference_loss(x - h * d, t, ref, **kw).loss.sum()) / (2 * h)
    assert abs(float((dx * d).sum() - diff.detach())) <= 1e-6 * max(1.0, abs(float(diff)))
    assert not dx[0, :4].any() and not dx[1, 6:].any()


@pytest.mark.parametrize("gap", [-1e4, -200.0, 0.0, 200.0, 1e4])
def test_preference_far_from_even(gap):
    """Sequences that are told apart by far, and the other way round: losses of log(1 + e^-z) neither overflow nor vanish early."""
    x = torch.zeros(2, 1, 2, dtype=torch.float64)
    x[0, 0, 0], x[1, 0, 0] = gap, -gap
    got = preference_loss(x, torch.zeros(2, 1, dtype=torch.int64), beta=1.0)
    z = float(got.logprob[0] - got.logprob[1])
    want = -z if z < -40 else math.log1p(math.exp(-z))
    assert float(got.loss) == pytest.approx(want, rel=1e-12, abs=1e-300)


def test_pairs_without_a_target():
    x, t, ref = _preference()
    t[:] = -100
    x.requires_grad_()
    got = preference_loss(x, t, average=True)
    assert torch.equal(got.logprob, torch.zeros(4, dtype=torch.float64)) and torch.allclose(got.loss, torch.full((2,), math.log(2.0), dtype=torch.float64))
    dx, = torch.autograd.grad(got.loss.sum(), x)
    assert not dx.any()


def _policy(seed=0, shape=(2, 7), V=23, dtype=torch.float64, temperature=1.0):
    g = _gen(seed)
    x = (torch.randn(*shape, V, generator=g, dtype=torch.float64) * 2).to(dtype)
    t = torch.randint(0, V, shape, generator=g)
    lp = torch.log_softmax(x.double() / temperature, -1).gather(-1, t.unsqueeze(-1)).squeeze(-1)
    old = lp + 0.3 * torch.randn(shape, generator=g, dtype=torch.float64)
    ref = lp + 0.5 * torch.randn(shape, generator=g, dtype=torch.float64)
    t.view(-1)[::3] = -100
    return x, t, torch.randn(shape, generator=g, dtype=torch.float64), old, ref


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16])
@pytest.mark.parametrize("case", ["plain", "reference", "first", "no clip", "one advantage", "one dimension"])
def test_policy_by_its_definition(dtype, case):
    x, t, adv, old, ref = _policy(dtype=dtype, temperature=0.7)
    kw = dict(kl_weight=0.0, clip=(0.2, 0.3))
    if case == "reference":
        kw["kl_weight"] = 0.4
    if case == "no clip":
        kw["clip"] = (1.0, 1e9)
    if case == "one advantage":
        adv = adv[:, :1]
    if case == "one dimension":
        x, t, adv, old, ref = x[0], t[0], adv[0], old[0], ref[0]
    old = None if case == "first" else old
    x = x.clone().requires_grad_()
    g = torch.rand(t.shape, generator=_gen(9), dtype=torch.float64)
    got = policy_loss(x, t, adv, old, ref, temperature=0.7, **kw)
    dx, = torch.autograd.grad(got.loss, x, g.to(got.loss.dtype))
    *want, clipped = oracle.policy(x, t, adv, old, ref, temperature=0.7, g=g, **kw)
    for a, (b, tol) in zip((got.loss, got.logprob, got.kl, dx), want):
        assert a.shape == b.shape and ((a.detach().double() - b).abs() <= tol).all()
    assert torch.equal(got.clipped, clipped) and bool(clipped.any()) == (case not in ("first", "no clip"))
    assert not got.logprob.requires_grad and not got.kl.requires_grad
    assert not got.loss[t == -100].any() and not dx[t == -100].any()


def test_policy_by_differences():
    x, t, adv, old, ref = _policy()
    x.requires_grad_()

    def f(x):
        return policy_loss(x, t, adv, old, ref, kl_weight=0.3).loss.sum()
    dx, = torch.autograd.grad(f(x), x)
    d = torch.randn(x.shape, generator=_gen(3), dtype=torch.float64)
    h = 1e-6
    assert abs(float((dx * d).sum() - ((f(x + h * d) - f(x - h * d)) / (2 * h)).detach())) <= 1e-6


def test_policy_of_one_step_moves_by_the_advantage():
    """Without old log probabilities the ratio is 1: the loss is -A, its gradient that of -A log p."""
    x, t, adv, _, _ = _policy()
    x.requires_grad_()
    got = policy_loss(x, t, adv)
    real = t != -100
    assert torch.equal(got.loss, torch.where(real, -adv, 0.0)) and not got.clipped.any()
    lp = torch.log_softmax(x, -1).gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    want, = torch.autograd.grad((-adv * lp)[real].sum(), x)
    dx, = torch.autograd.grad(got.loss.sum(), x)
    assert (dx - want).abs().max() <= 1e-14


def test_hidden_targets():
    x = torch.tensor([[0.0, 1.0, -math.inf]], dtype=torch.float64)
    got = policy_loss(x, torch.tensor([2]), torch.tensor([1.0]), torch.tensor([-1.0]), torch.tensor([-1.0]), kl_weight=0.1)
    assert got.logprob[0] == -math.inf and got.kl[0] == math.inf and got.loss[0] == math.inf
    got = policy_loss(x, torch.tensor([2]), torch.tensor([1.0]), torch.tensor([-1.0]))
    assert got.loss[0] == 0.0
    x.requires_grad_()
    for ref, weight in ((None, 0.0), (torch.tensor([-1.0]), 0.1)):
        got = policy_loss(x, torch.tensor([2]), torch.tensor([1.0]), torch.tensor([-1.0]), ref, kl_weight=weight)
        dx, = torch.autograd.grad(got.loss, x)
        assert torch.equal(dx, torch.zeros_like(x))
    got = policy_loss(x, torch.tensor([2]), torch.tensor([1.0]))
    assert got.loss[0] == -1.0 and not torch.autograd.grad(got.loss, x)[0].any()


def test_refusals():
    x, t, ref = _preference(dtype=torch.float32)

    def refused(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            preference_loss(*a, **kw)
    refused("2 pairs", x[:3], t[:3])
    refused("2 pairs", x[0], t[0])
    refused("2 pairs", x[:0], t[:0])
    refused("no tokens", x[:, :0], t[:, :0])
    refused("targets should have shape", x, t[:, :3])
    refused("targets should hold token ids", x, t.float())
    refused("reference should have shape", x, t, ref[:2])
    refused("reference should hold floating", x, t, ref.long())
    refused("form should be", x, t, form="square")
    refused("beta should be above", x, t, beta=0.0)
    refused("beta should be above", x, t, label_smoothing=1.5)
    refused("beta should be above", x, t, margin=math.inf)
    refused("belong to the form", x, t, form="ipo", margin=0.5)
    refused("belong to the form", x, t, form="hinge", label_smoothing=0.5)
    refused("temperature", x, t, temperature=0.0)
    refused("not supported", x.long(), t)
    refused("outside of the vocabulary", x, t.masked_fill(t == -100, 31))
    x, t, adv, old, ref = _policy(dtype=torch.float32)

    def refused(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            policy_loss(*a, **kw)
    refused("old_logprobs should have shape", x, t, adv, old[:1])
    refused("ref_logprobs should hold", x, t, adv, old, t)
    refused("do not fit", x, t, adv[:, :3])
    refused("do not fit", x, t, adv.unsqueeze(0).expand(3, -1, -1))
    refused("advantages should hold", x, t, t)
    refused("clip should hold", x, t, adv, old, clip=(1.5, 0.2))
    refused("clip should hold", x, t, adv, old, clip=(0.2, -0.1))
    refused("kl_weight be finite", x, t, adv, old, ref, kl_weight=-1.0)
    refused("needs ref_logprobs", x, t, adv, old, kl_weight=0.1)
    refused("outside of the vocabulary", x, torch.full_like(t, -1), adv)
