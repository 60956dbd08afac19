"""Finetuning steps of models whose attention is the one with a gradient, on the GPU: loaded with and without optimisations, with
windows and padding, against the usual path of the same model."""
import pytest
import torch

from ipex_llm_b200.ops import cuda_ops
from ipex_llm_b200.train import causal_lm_loss

pytestmark = pytest.mark.gpu


def _model(kind, optimised, fused, **kw):
    import transformers as tr
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import LoraConfig, cast_lora_weight, get_peft_model, prepare_model_for_kbit_training
    cfg = getattr(tr, kind + "Config")(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                                       num_key_value_heads=2, vocab_size=1000, max_position_embeddings=512,
                                       tie_word_embeddings=False, **kw)
    model = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.bfloat16, device="cuda",
                                             modules_to_not_convert=["lm_head"], optimize_model=optimised, seed=0)
    model = prepare_model_for_kbit_training(model, use_gradient_checkpointing=fused, use_fused_attention=fused)
    pm = get_peft_model(model, LoraConfig(r=8, lora_alpha=16, lora_dropout=0.0, target_modules=["o_proj", "up_proj", "down_proj"]))
    cast_lora_weight(pm, torch.bfloat16)
    for i, p in enumerate(p for p in pm.parameters() if p.requires_grad):
        p.data.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.05)
    return pm.train()


@pytest.mark.parametrize("kind,kw,window", [("Llama", {}, 0), ("Mistral", dict(sliding_window=40), 40)])
@pytest.mark.parametrize("optimised", [False, True])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("pad", ["none", "ones", "left", "right"])
def test_steps(kind, kw, window, optimised, batch, pad, monkeypatch):
    from ipex_llm_b200.models import train_attention
    calls, kernel = [], train_attention.attention
    monkeypatch.setattr(train_attention, "attention", lambda *a: calls.append(a[5]) or kernel(*a))
    ids = torch.randint(0, 1000, (batch, 150), generator=torch.Generator().manual_seed(1)).cuda()
    real = torch.ones_like(ids)
    if pad == "left":
        real[-1, :37] = 0
    if pad == "right":
        real[-1, 99:] = 0
    labels = ids.masked_fill(real == 0, -100)
    if pad == "left":
        labels[-1, 37] = -100            # it would be predicted by a query that sees nothing: the library makes something up there
    args = dict(input_ids=ids, use_cache=False, **({} if pad == "none" else dict(attention_mask=real)))
    losses, grads = [], []
    for fused in (False, True):
        model = _model(kind, optimised, fused, **kw)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = causal_lm_loss(model(**args).logits, labels)
        loss.backward()
        losses.append(loss.detach())
        grads.append({n: p.grad for n, p in model.named_parameters() if p.requires_grad})
    assert calls == [window] * 4                       # two layers, each once more for its checkpoint
    cuda_ops.check_error_flag(ids.device)
    # Two paths in bf16 (2^-8 for a rounding) over the same weights: a layer rounds its seven products' results, their sums with
    # the adapters', rope, the attention and the residuals, about 16 numbers on a path forward and as many backward; errors of
    # single roundings are independent, so their norms add up in squares: sqrt(2 layers x 32) roundings of either path.
    tol = 2 * (2 * 32) ** 0.5 * 2.0 ** -8
    assert abs(float(losses[0] - losses[1])) <= tol * float(losses[0])
    for n, a in grads[0].items():
        b = grads[1][n]
        assert torch.isfinite(b).all() and (a - b).float().norm() <= tol * a.float().norm(), n


@pytest.mark.parametrize("optimised", [False, True])
@pytest.mark.parametrize("pad", ["none", "ones"])
def test_no_logit_depends_on_a_later_token(optimised, pad):
    model = _model("Llama", optimised, True)
    ids = torch.randint(0, 1000, (1, 150), generator=torch.Generator().manual_seed(1)).cuda()
    args = {} if pad == "none" else dict(attention_mask=torch.ones_like(ids))
    out = []
    for last in (7, 500):
        ids[0, -1] = last
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out.append(model(input_ids=ids, use_cache=False, **args).logits.detach())
    assert torch.equal(out[0][:, :-1], out[1][:, :-1]) and not torch.equal(out[0][:, -1], out[1][:, -1])


@pytest.mark.parametrize("optimised", [False, True])
@pytest.mark.parametrize("window", [0, 40])
def test_generation_after_finetuning(optimised, window):
    """Evaluation leaves the gradient's kernels.  A model that was optimised computes what it did without them; the others' attention
    goes from the library's to this package's."""
    kind, kw = ("Mistral", dict(sliding_window=window)) if window else ("Llama", {})
    ids = torch.randint(0, 1000, (2, 60), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones_like(ids)
    mask[1, :11] = 0
    out = []
    for fused in (False, True):
        model = _model(kind, optimised, fused, **kw).eval()
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            out.append(model(input_ids=ids, attention_mask=mask, use_cache=False).logits)
    see = mask.bool().unsqueeze(-1)
    a, b = (o.masked_fill(~see, 0).float() for o in out)
    if optimised:
        assert torch.equal(a, b)
    assert (a - b).norm() <= 2 * (2 * 16) ** 0.5 * 2.0 ** -8 * a.norm()          # as in test_steps, forward alone
