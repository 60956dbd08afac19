"""Forward-mode differentiation of the operators with a gradient of their own: the CPU's plain forms carry it, the GPU refuses it."""
import pytest
import torch
from torch.autograd import forward_ad

from ipex_llm_b200.ops.gradients import refuse_tangents
from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs
from ipex_llm_b200.ops.train_attn import attention


def test_tangents_are_refused():
    x = torch.randn(3)
    refuse_tangents("an operator", x, None)
    with forward_ad.dual_level():
        refuse_tangents("an operator", x, None)
        with pytest.raises(RuntimeError, match="an operator: forward-mode"):
            refuse_tangents("an operator", None, x, forward_ad.make_dual(x, x))

    def f(t):
        refuse_tangents("an operator", t)
        return t
    with pytest.raises(RuntimeError, match="an operator: forward-mode"):
        torch.func.jvp(f, (x,), (x,))


def _calls(device, dtype):
    g = torch.Generator().manual_seed(1)
    q, logits = (torch.randn(*s, generator=g, dtype=torch.float64).to(device, dtype) for s in ((1, 2, 5, 8), (5, 9)))
    ids = torch.arange(5, device=device)
    return [(q, lambda t: attention(t, q, q)), (q, lambda t: attention(q, t, q)), (q, lambda t: attention(q, q, t)),
            (logits, lambda t: token_logprobs(t, ids).logprob),
            (logits, lambda t: distill_loss(t, ids.unsqueeze(-1), logits[:, :1].float()))]


@pytest.mark.parametrize("i", range(5))
def test_the_cpu_carries_tangents(i):
    x, f = _calls("cpu", torch.float64)[i]
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    with forward_ad.dual_level():
        got = forward_ad.unpack_dual(f(forward_ad.make_dual(x, d))).tangent
    h = 1e-5
    assert (got - (f(x + h * d) - f(x - h * d)) / (2 * h)).abs().max() <= 1e-7      # h^2 of the third derivative, 2^-52 / h


@pytest.mark.gpu
@pytest.mark.parametrize("learns", [False, True])
@pytest.mark.parametrize("i", range(5))
def test_the_gpu_refuses_tangents(i, learns):
    x, f = _calls("cuda", torch.bfloat16)[i]
    x = x.clone().requires_grad_(learns)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        f(x)


@pytest.mark.parametrize("device,dtype", [("cpu", torch.float64), ("cpu", torch.float32),
                                          pytest.param("cuda", torch.float32, marks=pytest.mark.gpu),
                                          pytest.param("cuda", torch.bfloat16, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("other", [-40.0, -87.5, -100.0, -1000.0, -float("inf")])
@pytest.mark.parametrize("V", [40, 9000])
def test_students_that_give_nearly_nothing_to_other_tokens(V, other, device, dtype):
    """What the student gives to tokens that the teacher did not name falls to the end of 32 bits and past it."""
    x = torch.full((3, V), -float("inf"), dtype=dtype, device=device)
    x[:, 4:12] = 0.0
    x[:, 20] = other
    x.requires_grad_()
    ids = torch.arange(4, 12, device=device).expand(3, 8)
    values = torch.full((3, 8), 0.05 / 8, device=device).log()           # the teacher leaves 0.95 to others
    loss = distill_loss(x, ids, values, teacher_logsumexp=torch.zeros(3, device=device))
    dx, = torch.autograd.grad(loss.sum(), (x,))
    p = torch.full((V,), 0.0, dtype=torch.float64)
    p[4:12] = 0.125
    want, rest = 0.05 * torch.tensor(0.05 / 8 / 0.125, dtype=torch.float64).log(), 0.0
    if other == -40.0:                                                   # e^-40 / 8 is above 2^-100
        p[20] = torch.tensor(-40.0, dtype=torch.float64).exp() / 8
        rest = 0.95
        want = want + rest * (torch.tensor(rest, dtype=torch.float64).log() - p[20].log())
    d = (0.05 + rest) * p
    d[4:12] -= 0.05 / 8
    d[20] -= rest
    # numbers of up to 45 and 1, a few roundings of 32 bits each; the gradient's last rounding
    assert (loss.double().cpu() - want).abs().max() <= 16 * 45 * 2.0 ** -24
    assert (dx.double().cpu() - d).abs().max() <= 16 * 2.0 ** -24 + torch.finfo(dtype).eps / 2
