"""Calls of the optimizer's operators that hold nothing, or less than usual."""
import pytest
import torch

from ipex_llm_b200.ops.adamw import adamw_state, adamw_step, grad_norm


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_without_any_gradient(device, bits):
    """The norm of no gradients has no device to be on but the CPU; a step that clips by it does nothing."""
    params, grads = [torch.ones(300, device=device), torch.ones(7, device=device)], [None, None]
    state = adamw_state(params, bits)
    adamw_step(params, grads, **state._asdict(), lr=1.0, grad_norm=grad_norm(grads), max_grad_norm=1.0)
    assert all(bool((p == 1.0).all()) for p in params) and state.step.tolist() == [0]
    with pytest.raises(RuntimeError, match="exp_avg should be"):
        adamw_step(params, grads, **state._replace(exp_avg=state.exp_avg[:256])._asdict(), lr=1.0, grad_norm=grad_norm(grads), max_grad_norm=1.0)
    if device == "cuda":                                          # of gradients that are there, it is read where they are
        with pytest.raises(RuntimeError, match="grad_norm should be"):
            adamw_step(params, [torch.ones_like(p) for p in params], **state._asdict(), lr=1.0, grad_norm=torch.ones(()), max_grad_norm=1.0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_the_clipping_factor_is_a_quotient_rounded_once(device):
    """With beta 0 and gradients of 1, the first moment is the factor: max_norm / (norm + 1e-6) in 32 bits, its sum and its quotient
    rounded to nearest, and 1 at most."""
    params, grads = [torch.zeros(1, device=device)], [torch.ones(1, device=device)]
    state = adamw_state(params)
    norms = (torch.rand(500, generator=torch.Generator().manual_seed(0)) * 3).tolist() + [0.0, 0.05, 1e30, float("inf")]
    for norm in norms:
        norm = torch.tensor(norm)
        adamw_step(params, grads, **state._asdict(), lr=0.0, betas=(0.0, 0.5), grad_norm=norm.to(device), max_grad_norm=0.05)
        # 64 bits hold the quotient of two 32-bit numbers to more than twice their places: rounding it again is rounding it once
        below = (norm + torch.tensor(1e-6)).double()
        want = min(1.0, float((torch.tensor(0.05).double() / below).float()))
        assert float(state.exp_avg[0]) == want, float(norm)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("largest", [0.0, 1.0, float("inf")])
def test_zeros_keep_their_sign(device, largest):
    """Of first moments in 8 bits, as in 32: codes are the same on both sides."""
    grads = [torch.zeros(300, device=device)]
    grads[0][1::2] = -0.0
    grads[0][0] = largest                                         # the block's exponent, or what does not count for it
    params = [torch.zeros(300, device=device)]
    state = adamw_state(params, 8)
    for _ in range(2):
        adamw_step(params, grads, **state._asdict(), lr=0.1, betas=(0.0, 0.5))
        codes = state.exp_avg.view(torch.uint8).tolist()
        # with beta 0, moments are (0 m) + g: of -0 after 0 it is 0, of -0 after -0 it is -0
        assert not any(codes[2:300:2]) and not any(codes[300:])
    state = adamw_state(params, 8)
    state.exp_avg.view(torch.uint8)[:300] = 0x80
    adamw_step(params, grads, **state._asdict(), lr=0.1, betas=(0.5, 0.5))
    codes = state.exp_avg.view(torch.uint8).tolist()
    assert codes[1:300:2] == [0x80] * 150 and not any(codes[2:300:2]) and not any(codes[300:])
