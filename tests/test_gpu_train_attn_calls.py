"""Calls of the attention with a gradient that its documentation allows, on the GPU."""
import math

import pytest
import torch

import train_attn_oracle as oracle

pytestmark = pytest.mark.gpu


def _inputs(B, Hq, Hkv, Sq, Skv, D, dtype, seed, grad_std=1.0 / 16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def heads(n, s, std):
        return (torch.randn(B, s, n, D, generator=g, device="cuda") * std).to(dtype).transpose(1, 2)
    return heads(Hq, Sq, 1.5), heads(Hkv, Skv, 1.0), heads(Hkv, Skv, 1.0), heads(Hq, Sq, grad_std)


def _run(q, k, v, g, **kw):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.train_attn import attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, **kw)
    grads = torch.autograd.grad(out, (q, k, v), g)
    cuda_ops.check_error_flag(q.device)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)))


def _check(got, q, k, v, g, scale=None, causal=True, window=0, key_mask=None):
    want = oracle.attention(q, k, v, g, scale or q.shape[-1] ** -0.5, causal, window, key_mask)
    for name, (exact, tol) in want.items():
        t = got[name]
        assert t.shape == exact.shape and t.dtype == q.dtype, name
        off = ((t.double() - exact).abs() / tol).nan_to_num(nan=math.inf)
        # what passes the type's range in the formula is infinite
        past = t.isinf() & (t.sign() == exact.sign()) & (exact.abs() + tol > torch.finfo(t.dtype).max)
        off = off.masked_fill(past, 0.0)
        assert float(off.max()) <= 1.0, (name, float(off.max()), (off > 1).sum().item(), off.argmax().item())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("offset", [1, 4, 7])
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "qkvg"])
def test_contiguous_tensors_at_any_address(which, offset, masked):
    """Views of a flat buffer that begin between two 16-byte boundaries."""
    given = dict(zip("qkvg", _inputs(2, 4, 2, 70, 70, 64, torch.bfloat16, 3)))
    kw = dict(key_mask=torch.arange(70, device="cuda") < torch.tensor([[70], [31]], device="cuda")) if masked else {}
    want = _run(*given.values(), **kw)

    def moved(t):
        flat = torch.zeros(offset + t.numel(), dtype=t.dtype, device="cuda")[offset:]
        return flat.view(t.shape).copy_(t)
    got = _run(*(moved(t) if n in which else t for n, t in given.items()), **kw)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Sq,Skv", [(300, 200), (513, 1), (200, 300), (40, 33), (1000, 128)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30, 1000])
def test_windows_of_more_than_all_keys(window, Sq, Skv, dtype):
    args = _inputs(2, 4, 2, Sq, Skv, 64, dtype, 5)
    got, want = _run(*args, window=window), _run(*args)
    assert all(torch.equal(got[n], want[n]) for n in want)
    _check(got, *args, window=window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 24, 2.0 ** 27, 2.0 ** 29, 2.0 ** 30.9])
def test_rows_whose_gradient_and_output_have_a_large_product(size, D, dtype):
    """As where a loss is scaled: delta of the first tokens, whose own dS is small, lies far past what one number of 16 bits holds."""
    q, k, v, g = _inputs(1, 4, 2, 150, 150, D, dtype, 6)
    v = v * 64
    for i in (0, 3):
        one = v[:, :, i].repeat_interleave(2, 1).float()                     # the output of row 0, and near that of row 3
        g[:, :, i] = (one * (size / one.square().sum(-1, keepdim=True))).clamp(-6e4, 6e4).to(dtype)
    got = _run(q, k, v, g)
    # (row 3 is no mean of equal values: its dS and with it dk pass the range of fp16 with the larger sizes)
    assert not any(bool(t.isnan().any()) for t in got.values())
    _check(got, q, k, v, g)
    delta = (g[:, :, 0].float() * got["out"][:, :, 0].float()).sum(-1)
    assert float(delta.max()) > 0.4 * min(size, 2.0 ** 26)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [2.0 ** 23, 2.0 ** 25, 2.0 ** 30])
def test_first_tokens_of_a_large_scaled_loss(size, D):
    """fp16, and all gradients within its range: of the first token alone, whose dS is 0, delta is up to 2^30."""
    q, k, v, g = _inputs(1, 2, 2, 150, 150, D, torch.float16, 6)
    v = v * 2048
    one = v[:, :, 0].float()
    g[:, :, 0] = (one * (size / one.square().sum(-1, keepdim=True))).half()
    got = _run(q, k, v, g)
    assert all(bool(t.isfinite().all()) for t in got.values())
    _check(got, q, k, v, g)
