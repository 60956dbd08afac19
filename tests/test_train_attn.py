"""Attention with a gradient on the CPU: the plain form, its gradients, and what is refused."""
import math

import pytest
import torch

import train_attn_oracle as oracle
from ipex_llm_b200.ops.train_attn import attention


def _inputs(B, Hq, Hkv, Sq, Skv, D, dtype=torch.float64):
    g = torch.Generator().manual_seed(Sq + Skv)
    return [torch.randn(B, h, s, D, generator=g, dtype=torch.float64).to(dtype).requires_grad_()
            for h, s in ((Hq, Sq), (Hkv, Skv), (Hkv, Skv))]


@pytest.mark.parametrize("Sq,Skv,causal,window", [(5, 5, True, 0), (3, 7, True, 2), (6, 4, True, 0), (4, 6, False, 0)])
def test_gradients_by_differences(Sq, Skv, causal, window):
    q, k, v = _inputs(2, 4, 2, Sq, Skv, 8)
    mask = torch.ones(2, Skv, dtype=torch.bool)
    mask[0, 1] = mask[1, 0] = False
    assert torch.autograd.gradcheck(lambda *t: attention(*t, causal=causal, window=window, key_mask=mask), (q, k, v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_definition(dtype):
    q, k, v = _inputs(2, 4, 2, 9, 12, 16, dtype)
    mask = torch.arange(12) < torch.tensor([[7], [12]])
    g = torch.randn(2, 4, 9, 16, generator=torch.Generator().manual_seed(1)).to(dtype)
    want = oracle.attention(q, k, v, g, 0.25, True, 5, mask)
    out = attention(q, k, v, scale=0.25, window=5, key_mask=mask)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, (q, k, v), g))))
    for n, (exact, tol) in want.items():
        if dtype == torch.float64:
            tol = 1e-12
        assert bool(((got[n].double() - exact).abs() <= tol).all()), n


def test_rows_that_see_nothing_and_hidden_rows_that_hold_anything():
    q, k, v = _inputs(1, 2, 1, 6, 6, 8)
    with torch.no_grad():
        k[0, 0, :3] = math.nan
        v[0, 0, :3] = math.inf
    mask = torch.arange(6).view(1, -1) >= 3
    out = attention(q, k, v, key_mask=mask)
    assert bool((out[:, :, :3] == 0).all()) and bool(out.isfinite().all())
    for d in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)):
        assert bool(d.isfinite().all()) and bool((d[:, :, :3] == 0).all())


def test_what_is_refused():
    q, k, v = (t.detach() for t in _inputs(2, 4, 2, 5, 5, 8))
    for bad in (lambda: attention(q[0], k[0], v[0]), lambda: attention(q, k, v[:, :, :4]), lambda: attention(q, k[:1], v[:1]),
                lambda: attention(q[:, :3], k, v), lambda: attention(q, k.float(), v), lambda: attention(q, k, v, scale=0.0),
                lambda: attention(q, k, v, scale=-1.0), lambda: attention(q, k, v, scale=math.nan),
                lambda: attention(q, k, v, window=-1), lambda: attention(q, k, v, causal=False, window=3),
                lambda: attention(q, k, v, key_mask=torch.ones(2, 4, dtype=torch.bool)),
                lambda: attention(q, k, v, key_mask=torch.ones(2, 5)), lambda: attention(q.int(), k.int(), v.int())):
        with pytest.raises(RuntimeError):
            bad()
