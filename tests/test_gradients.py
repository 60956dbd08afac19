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
