"""Calls of the attention with a gradient that its documentation allows, on the CPU."""
import pytest
import torch

from ipex_llm_b200.ops import train_attn


@pytest.mark.parametrize("D", [8, 64])
@pytest.mark.parametrize("layout", ["contiguous", "token-major", "one head", "expanded", "rows apart"])
@pytest.mark.parametrize("offset", [0, 1, 4, 7, 8])
def test_tensors_at_any_address_fit(layout, offset, D):
    n = 2 * 4 * 6 * (D + 8)
    flat = torch.arange(offset + n + 8).to(torch.float16)[offset:]
    t = {"contiguous": lambda: flat[:2 * 4 * 6 * D].view(2, 4, 6, D),
         "token-major": lambda: flat[:2 * 4 * 6 * D].view(2, 6, 4, D).transpose(1, 2),
         "one head": lambda: flat[:2 * 6 * D].view(2, 6, 1, D).transpose(1, 2),
         "expanded": lambda: flat[:2 * 6 * D].view(2, 1, 6, D).expand(2, 4, 6, D),
         "rows apart": lambda: flat[:2 * 4 * 6 * (D + 8)].view(2, 4, 6, D + 8)[..., :D]}[layout]()
    at, b, h, s, fit = train_attn._fit(t)
    assert torch.equal(fit, t) and at == fit.data_ptr() and at % 16 == 0 and fit.stride(-1) == 1
    B, H, S, _ = t.shape
    for size, stride in ((B, b), (H, h), (S, s)):
        assert stride > 0 and stride % 8 == 0
    strides = [x for n, x in zip((B, H, S), fit.stride()) if n > 1]
    assert strides == [x for n, x in zip((B, H, S), (b, h, s)) if n > 1]


@pytest.mark.parametrize("Sq,Skv", [(6, 4), (4, 6)])
def test_windows_of_more_than_all_keys(Sq, Skv):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, s, 8, generator=g, dtype=torch.float64) for s in (Sq, Skv, Skv))
    assert torch.equal(train_attn.attention(q, k, v, window=2 ** 31 - 1), train_attn.attention(q, k, v))
