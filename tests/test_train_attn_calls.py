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


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("Sq,Skv", [(5, 5), (1, 5), (5, 0), (0, 5)])
def test_outputs_are_views_of_token_major_ones(device, Sq, Skv):
    """As attention modules go on with them: `out.transpose(1, 2).view(batch, tokens, -1)`."""
    q, k = (torch.randn(2, 4, s, 8, device=device, dtype=torch.bfloat16) for s in (Sq, Skv))
    for learns in (False, True):
        out = train_attn.attention(q.requires_grad_(learns), k, k, causal=False)
        assert out.shape == (2, 4, Sq, 8) and out.transpose(1, 2).is_contiguous()


def test_modules_that_view_the_attention():
    """Its result in a model whose attention takes it by `view`, on the CPU."""
    import transformers as tr
    from ipex_llm_b200.models.train_attention import use_train_attention
    cfg = tr.AfmoeConfig(hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         head_dim=8, vocab_size=50, num_experts=4, num_experts_per_tok=2, moe_intermediate_size=16,
                         max_position_embeddings=64, attn_implementation="sdpa")
    torch.manual_seed(0)
    model = tr.AfmoeForCausalLM(cfg)
    ids = torch.randint(1, 50, (2, 9), generator=torch.Generator().manual_seed(2))
    want = model(ids).logits
    assert use_train_attention(model)
    # 32 bits on both sides: some 100 roundings a layer on a path, two layers, either side, four for what they amplify
    assert (model(ids).logits - want).abs().max() <= 2 * 2 * 100 * 4 * 2.0 ** -24 * want.abs().max()
