"""Targets that a policy hides (a logit of -inf), beside old and reference policies that hide them or not."""
import math

import pytest
import torch

from ipex_llm_b200.ops.preference import policy_loss

HIDDEN = -math.inf


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("old", [None, -1.0, HIDDEN], ids=["no old", "old", "old hidden"])
@pytest.mark.parametrize("ref", [None, -1.0, HIDDEN], ids=["no ref", "ref", "ref hidden"])
def test_hidden_targets_of_a_policy(device, dtype, old, ref):
    """What both policies hide has a ratio of 1 and no KL term, as equal numbers have; no row has a gradient of NaN."""
    weight = 0.0 if ref is None else 0.25
    x = torch.zeros(4, 9, dtype=dtype, device=device)
    x[:3, 4] = HIDDEN
    x[2] = HIDDEN                                                 # a row without a token
    x.requires_grad_()
    t = torch.full((4,), 4, device=device)
    a = torch.tensor([2.0, -2.0, 2.0, 2.0], device=device)
    seen = -math.log(9.0)

    def rows(value):
        return None if value is None else torch.tensor([value] * 3 + [seen], device=device)
    got = policy_loss(x, t, a, rows(old), rows(ref), clip=(0.2, 0.3), kl_weight=weight)
    dx, = torch.autograd.grad(got.loss.sum(), x)
    w = 0.0 if old == -1.0 else 1.0
    kl = math.inf if ref == -1.0 else 0.0
    # -min(w A, clamp(w) A)
    want = [-min(w * v, min(max(w, 0.8), 1.3) * v) + (weight * kl if weight else 0.0) for v in (2.0, -2.0, 2.0)]
    assert got.logprob[:3].tolist() == [HIDDEN] * 3
    assert got.kl[:3].tolist() == [kl] * 3
    assert got.loss[:3].tolist() == pytest.approx(want)
    assert got.clipped.tolist() == [False, w == 0.0, False, False]
    assert not dx[:3].any()                                       # NaN counts as one that is there
    # the row beside them: w = 1, d = 0 but for the rounding of log 9 to 32 bits
    assert abs(float(got.loss[3]) + 2.0) <= 1e-5 and abs(float(got.kl[3])) <= 1e-6
    p = torch.full((9,), 1.0 / 9.0, dtype=torch.float64)
    p[4] -= 1.0
    assert (dx[3].double().cpu() - 2.0 * p).abs().max() <= 2.0 * torch.finfo(dtype).eps / 2 + 1e-5


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_target_that_the_reference_alone_hides(device):
    """e^d - d - 1 grows without end, its slope does not: e^d - 1 is -1."""
    x = torch.zeros(1, 8, device=device, requires_grad=True)
    got = policy_loss(x, torch.tensor([3], device=device), torch.zeros(1, device=device), None, torch.full((1,), HIDDEN, device=device),
                      kl_weight=0.5)
    assert got.loss.item() == got.kl.item() == math.inf
    dx, = torch.autograd.grad(got.loss.sum(), x)
    want = torch.full((8,), -0.5 / 8)
    want[3] += 0.5
    assert (dx[0].cpu() - want).abs().max() <= 1e-6
