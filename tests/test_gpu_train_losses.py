"""Attention with a gradient and the losses from logits, together: in a chain of their own and in a finetuning step."""
import pytest
import torch

from ipex_llm_b200.ops import cuda_ops
from ipex_llm_b200.train import causal_lm_loss, distill_lm_loss, next_tokens, teacher_tokens

pytestmark = pytest.mark.gpu


def _chain(attend, lm_loss, distill, q, k, v, w, labels, mask, teacher):
    out = attend(q, k, v, mask)
    logits = out.transpose(1, 2).flatten(2) @ w
    return lm_loss(logits, labels) + 0.5 * distill(logits, labels, teacher)


def _formula_attention(q, k, v, mask):
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5
    see = torch.ones(s.shape[-2:], dtype=torch.bool, device=s.device).tril() & mask[:, None, None, :]
    p = torch.softmax(s.masked_fill(~see, -1e30), -1) * see
    return p @ v


def _formula_loss(logits, labels):
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), next_tokens(labels).flatten())


def _formula_distill(logits, labels, t):
    real = next_tokens(labels) != -100
    q = t.teacher_logits.double().exp()
    logp = torch.log_softmax(logits, -1).gather(-1, t.teacher_ids)
    rest, left = 1 - q.sum(-1), 1 - logp.exp().sum(-1)
    kl = (q * (q.log() - logp)).sum(-1) + rest * (rest.log() - left.log())
    return kl[real].sum() / real.sum()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,Hkv,S,D,V", [(2, 4, 4, 37, 64, 1000), (3, 8, 2, 190, 128, 515)])
def test_chain_and_its_gradients(dtype, B, Hq, Hkv, S, D, V):
    from ipex_llm_b200.ops.train_attn import attention
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(B, h, S, D, generator=g).to("cuda", dtype).requires_grad_() for h in (Hq, Hkv, Hkv))
    w = (torch.randn(Hq * D, V, generator=g) * (Hq * D) ** -0.5).to("cuda", dtype).requires_grad_()
    labels = torch.randint(0, V, (B, S), generator=g).cuda()
    mask = torch.ones(B, S, dtype=torch.bool, device="cuda")
    mask[1, S - 11:] = False
    labels[1, S - 11:] = -100
    t = teacher_tokens(torch.randn(B, S, V, generator=g).cuda(), 16)
    loss = _chain(lambda a, b, c, m: attention(a, b, c, key_mask=m), causal_lm_loss,
                  lambda x, y, z: distill_lm_loss(x, y, *z), q, k, v, w, labels, mask, t)
    own = torch.autograd.grad(loss, (q, k, v, w))
    cuda_ops.check_error_flag(q.device)
    wide = [x.detach().double().requires_grad_() for x in (q, k, v, w)]
    ref = _chain(_formula_attention, _formula_loss, _formula_distill, *wide, labels, mask, t)
    want = torch.autograd.grad(ref, wide)
    # Half a step of the type for each rounding on a path: the attention's output, the logits, their two gradients and their sum,
    # the output's gradient, and in the attention's backward pass p, ds, dq or dk: nine, of which each moves a gradient's norm by no
    # more than its own size (a logit's rounding changes p by |logit| times that: logits are below 4, so it counts four times).
    half = torch.finfo(dtype).eps / 2
    assert abs(float((loss.detach() - ref.detach()))) <= 9 * half * float(ref.detach())
    for n, a, b in zip("qkvw", own, want):
        assert a.dtype == dtype and torch.isfinite(a).all()
        assert (a.double() - b).norm() <= 12 * half * b.norm(), n


def _model(fused):
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import LoraConfig, cast_lora_weight, get_peft_model, prepare_model_for_kbit_training
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      vocab_size=1000, max_position_embeddings=256, tie_word_embeddings=False)
    model = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.bfloat16, device="cuda",
                                             modules_to_not_convert=["lm_head"], optimize_model=False, seed=0)
    model = prepare_model_for_kbit_training(model, use_gradient_checkpointing=fused, use_fused_attention=fused)
    pm = get_peft_model(model, LoraConfig(r=8, lora_alpha=16, lora_dropout=0.0, target_modules=["q_proj", "v_proj", "up_proj"]))
    cast_lora_weight(pm, torch.bfloat16)
    for i, p in enumerate(p for p in pm.parameters() if p.requires_grad):
        p.data.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.05)
    return pm.train()


@pytest.mark.parametrize("pad", [False, True])
def test_finetuning_step(tmp_path, pad):
    from ipex_llm.transformers.qlora import TrainingArguments
    from ipex_llm_b200.models import train_attention
    from ipex_llm_b200.train import Trainer, default_collator
    g = torch.Generator().manual_seed(1)
    data = []
    for i in range(4):
        ids = torch.randint(0, 1000, (150 - (17 * i if pad else 0),), generator=g)
        teacher = teacher_tokens(torch.randn(len(ids), 1000, generator=g).cuda(), 8)
        data.append({"input_ids": ids.tolist(), "labels": ids.tolist(), "attention_mask": [1] * len(ids), **teacher._asdict()})
    fused, usual = _model(True), _model(False)
    args = TrainingArguments(output_dir=str(tmp_path), per_device_train_batch_size=4, max_steps=3, logging_steps=1,
                             optim="fused_lora_adamw", fused_loss=True, distill_weight=0.25)
    tr = Trainer(fused, args, train_dataset=data)
    batch = default_collator(data)
    calls, kernel = [], train_attention.attention
    train_attention.attention = lambda *a: calls.append(a) or kernel(*a)
    try:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = tr.compute_loss(fused, dict(batch))
        loss.backward()
    finally:
        train_attention.attention = kernel
    assert len(calls) == 4                            # two layers, each once more for its checkpoint
    cuda_ops.check_error_flag(loss.device)
    batch = {n: t.cuda() for n, t in batch.items()}
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = usual(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    labels = batch["labels"]
    t = type(teacher)(batch["teacher_ids"].clamp(min=0), batch["teacher_logits"], batch["teacher_logsumexp"])
    want = 0.75 * _formula_loss(logits.double(), labels) + 0.25 * _formula_distill(logits.double(), labels, t)
    want.backward()
    # Two paths in bf16 (2^-8 for a rounding) over the same weights: a layer rounds its seven products' results, their sums with
    # the adapters', rope, the attention and the residuals, about 16 numbers on a path forward and as many backward; errors of
    # single roundings are independent, so their norms add up in squares: sqrt(2 layers x 32) roundings of either path.
    tol = 2 * (2 * 32) ** 0.5 * 2.0 ** -8
    assert abs(float(loss.detach() - want.detach())) <= tol * float(want.detach())
    for (n, a), b in zip(fused.named_parameters(), usual.parameters()):
        if a.requires_grad:
            assert torch.isfinite(a.grad).all() and (a.grad - b.grad).float().norm() <= tol * b.grad.float().norm(), n
    fused.zero_grad()
    metrics = tr.train()
    assert metrics["train_loss"] == metrics["train_loss"] and tr.state.global_step == 3


def test_scores_of_tokens_on_a_device():
    from ipex_llm_b200.benchmark.perplexity import BigDLPPL
    model = _model(False).eval()
    ppl = BigDLPPL(model=model)
    ids = torch.randint(0, 1000, (1, 40), generator=torch.Generator().manual_seed(2))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        total, n = ppl.nll(ids)
        got = ppl.token_scores(ids, entropy=True, top=3)
    assert got.logprob.shape == (1, 39) and n == 39
    # the logits are the same: 32-bit sums on both sides (2^-24 for each of some 64 roundings of 1000 terms' tree)
    assert abs(float(-got.logprob.sum()) - total) <= 64 * 2.0 ** -24 * total
