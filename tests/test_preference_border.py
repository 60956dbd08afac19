"""The border of the hinge: where its loss is 0, it does not pull any more."""
import pytest
import torch

from ipex_llm_b200.ops.preference import preference_loss


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("beyond,slope", [(-0.25, 1.0), (0.0, 0.0), (0.25, 0.0)])
def test_the_hinge_at_its_border(device, beyond, slope):
    """Both sequences have -log 2: the margin is what their reference makes of it, exactly."""
    s = -torch.tensor(2.0, dtype=torch.float64).log()
    assert float((s + 1.0) - s) == 1.0
    x = torch.zeros(2, 1, 2, device=device, requires_grad=True)
    got = preference_loss(x, torch.zeros(2, 1, dtype=torch.int64, device=device),
                          torch.tensor([-1.0 - beyond, 0.0], device=device), beta=1.0, form="hinge")
    dx, = torch.autograd.grad(got.loss.sum(), x)
    assert abs(float(got.loss.detach()) - max(0.0, -beyond)) <= 2.0 ** -24 and (beyond or float(got.loss.detach()) == 0.0)
    # -1 for the preferred one's log p, 1 for the other's; log p moves with the logits by half each
    want = torch.tensor([[[-0.5, 0.5]], [[0.5, -0.5]]]) * slope
    assert (dx.cpu() - want).abs().max() <= 2.0 ** -22
