"""Whole steps of finetuning on the GPU: the clipped update, bit by bit as on the CPU."""
import pytest
import torch

from ipex_llm_b200.train import MultiTensorAdamW, optim, policy_lm_loss, preference_lm_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("policy", [False, True])
def test_clipped_steps_bit_by_bit(monkeypatch, dtype, bits, policy):
    """Loss, gradients, norm and update of a table of hidden states and an output layer.  The CPU's optimizer gets the same gradients
    and, as sums of squares are in another order there, the same norm: parameters, what is kept beside them, moments, exponents and
    counters are the same bits, and each step moves the parameters."""
    g = torch.Generator().manual_seed(0)
    B, S, H, V = 4, 37, 64, 1003
    params = [(torch.randn(B, S, H, generator=g)).to(dtype).cuda().requires_grad_(),
              (torch.randn(H, V, generator=g) * H ** -0.5).to(dtype).cuda().requires_grad_()]
    here = [p.detach().cpu().requires_grad_() for p in params]
    labels = torch.randint(0, V, (B, S), generator=g).cuda()
    labels[:, :9] = -100
    adv, old = ((torch.randn(B, S, generator=g) * 0.3 + m).cuda() for m in (0.0, -7.0))
    kw = dict(lr=1e-2, bits=bits, max_grad_norm=0.05, weight_decay=0.1, seed=3)
    opt, same = MultiTensorAdamW(params, **kw), MultiTensorAdamW(here, **kw)
    taken, norm_of = [], optim.grad_norm

    def norm(grads):
        if grads[0].is_cuda:
            taken.append(norm_of(grads))
            return taken[-1]
        want = float(norm_of(grads))
        assert abs(float(taken[-1]) - want) <= 2.0 ** -20 * want
        return taken[-1].cpu()
    monkeypatch.setattr(optim, "grad_norm", norm)
    for _ in range(4):
        logits = params[0] @ params[1]
        (policy_lm_loss(logits, labels, adv, old) if policy else preference_lm_loss(logits, labels, beta=0.5)).backward()
        before = [p.detach().clone() for p in params]
        for p, q in zip(params, here):
            q.grad = p.grad.cpu()
        opt.step()
        same.step()
        opt.zero_grad()
        assert not any(torch.equal(p, q) for p, q in zip(params, before))
        assert all(torch.equal(p.detach().cpu(), q.detach()) for p, q in zip(params, here))
        for b, c in zip(opt.buckets(), same.buckets()):
            for name, x, y in zip(b["state"]._fields, b["state"], c["state"]):
                assert x is None or torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8)), name
    assert len(taken) == 4 and float(taken[0]) > 0.05             # the factor takes part
