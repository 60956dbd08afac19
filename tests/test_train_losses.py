"""Losses from logits and the attention with a gradient inside models, on the CPU in 64 bits."""
import copy

import pytest
import torch
import torch.nn.functional as F

from ipex_llm_b200.models.train_attention import TRAIN_INTERFACE_NAME, use_train_attention
from ipex_llm_b200.train import causal_lm_loss, default_collator, distill_lm_loss, next_tokens, teacher_tokens

# Sums of a few hundred terms in 64 bits.
EXACT = 1e-12
# Norms compute in 32 bits inside a 64-bit model: a difference in the last bits of their inputs may turn any of their roundings
# (2^-24 each) the other way.  Two layers have five norms, each rounding three numbers on a path and entering up to two products
# of a gradient: 5 * 3 * 2 roundings, doubled for what the layers between them amplify.
NORMS = 64 * 2.0 ** -24


def _labels(batch, tokens, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    labels = torch.randint(0, vocab, (batch, tokens), generator=g)
    labels[0, : tokens // 3] = -100
    labels[-1, tokens - tokens // 4:] = -100
    return labels


@pytest.mark.parametrize("batch,tokens,vocab", [(1, 1, 5), (1, 2, 7), (3, 17, 211)])
def test_causal_lm_loss(batch, tokens, vocab):
    g = torch.Generator().manual_seed(3)
    labels = _labels(batch, tokens, vocab, 4)
    a = torch.randn(batch, tokens, vocab, generator=g, dtype=torch.float64, requires_grad=True)
    b = a.detach().clone().requires_grad_()
    own = causal_lm_loss(a, labels)
    own.backward()
    if tokens == 1:
        assert float(own.detach()) == 0 and not a.grad.any()
        return
    ref = F.cross_entropy(b[:, :-1].flatten(0, 1), labels[:, 1:].flatten())
    ref.backward()
    assert abs(float((own - ref).detach())) <= EXACT * max(1.0, abs(float(ref.detach())))
    assert (a.grad - b.grad).abs().max() <= EXACT
    assert not a.grad[:, -1].any()


def test_no_label_is_left():
    logits = torch.randn(2, 4, 9, requires_grad=True)
    labels = torch.full((2, 4), -100)
    t = teacher_tokens(logits.detach(), top=3)
    loss = causal_lm_loss(logits, labels) + distill_lm_loss(logits, labels, *t)
    loss.backward()
    assert float(loss.detach()) == 0 and not logits.grad.any()


@pytest.mark.parametrize("temperature", [1.0, 2.5])
@pytest.mark.parametrize("top", [1, 6, 23])
def test_distill_of_a_recorded_teacher(temperature, top):
    """Against the divergence of the coarsened distributions: the recorded tokens, and all others as one."""
    g = torch.Generator().manual_seed(5)
    V = 23
    teacher, student = (torch.randn(2, 6, V, generator=g, dtype=torch.float64) * 2 for _ in range(2))
    student.requires_grad_()
    labels = _labels(2, 6, V, 6)
    t = teacher_tokens(teacher, top, temperature)
    loss = distill_lm_loss(student, labels, *t, temperature=temperature)
    (own,) = torch.autograd.grad(loss, student)
    q, logp = torch.softmax(teacher / temperature, -1), torch.log_softmax(student / temperature, -1)
    at = torch.sort(teacher, dim=-1, descending=True, stable=True).indices[..., :top]
    qk, pk = q.gather(-1, at), logp.exp().gather(-1, at)
    kl = (qk * (qk.log() - pk.log())).sum(-1)
    if top < V:
        rest = 1 - qk.sum(-1)
        kl = kl + rest * (rest.log() - (1 - pk.sum(-1)).log())
    real = next_tokens(labels) != -100
    ref = (kl * real).sum() / real.sum() * temperature ** 2
    (grad,) = torch.autograd.grad(ref, student)
    # a teacher is kept in 32 bits: q is off by 2^-24 of log q, at most 8 * 2^-24 in all with its rounding, and what is left of 1
    # by as much; both enter the loss times a difference of logarithms of up to 16, times temperature^2
    tol = 2 * 16 * 8 * 2.0 ** -24 * temperature ** 2
    assert abs(float(loss - ref)) <= tol
    assert (own - grad).abs().max() <= tol
    same = distill_lm_loss(teacher, labels, *t, temperature=temperature)
    assert abs(float(same)) <= tol


def test_losses_refuse():
    logits = torch.randn(2, 4, 9)
    for labels in (torch.zeros(2, 3, dtype=torch.long), torch.zeros(8, dtype=torch.long)):
        with pytest.raises(RuntimeError, match="labels"):
            causal_lm_loss(logits, labels)
    with pytest.raises(RuntimeError, match="teacher_ids"):
        distill_lm_loss(logits, torch.zeros(2, 4, dtype=torch.long), torch.zeros(2, 3, 2, dtype=torch.long), torch.zeros(2, 3, 2))


def _llama(kind="llama", **kw):
    import transformers as tr
    base = dict(hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                vocab_size=97, max_position_embeddings=128, tie_word_embeddings=False, attn_implementation="sdpa")
    if kind == "gemma2":
        base.update(head_dim=16, sliding_window=5)
    if kind == "qwen2":
        base.update(use_sliding_window=True, sliding_window=5, max_window_layers=1)
    base.update(kw)
    name = {"llama": "Llama", "mistral": "Mistral", "gemma2": "Gemma2", "qwen2": "Qwen2", "phi3": "Phi3",
            "starcoder2": "Starcoder2"}[kind]
    if kind == "phi3":
        base.update(pad_token_id=0)
    torch.manual_seed(1)
    return getattr(tr, name + "ForCausalLM")(getattr(tr, name + "Config")(**base)).double()


@pytest.mark.parametrize("kind,kw", [("llama", {}), ("llama", dict(attention_dropout=0.0, num_key_value_heads=4)),
                                     ("mistral", dict(sliding_window=5)), ("mistral", dict(sliding_window=64)), ("qwen2", {}),
                                     ("phi3", dict(sliding_window=7)), ("starcoder2", dict(sliding_window=3)), ("gemma2", {}),
                                     ("gemma2", dict(attn_logit_softcapping=None))])
@pytest.mark.parametrize("pad", ["none", "left", "right", "packed"])
def test_models_give_the_same(kind, kw, pad, monkeypatch):
    from ipex_llm_b200.models import train_attention
    calls, usual = [], train_attention.attention
    monkeypatch.setattr(train_attention, "attention", lambda *a: calls.append(a[5]) or usual(*a))
    model = _llama(kind, **kw)
    own = copy.deepcopy(model)
    assert use_train_attention(own) and own.config._attn_implementation == TRAIN_INTERFACE_NAME
    ids = torch.randint(1, 97, (2, 13), generator=torch.Generator().manual_seed(2))
    args = dict(input_ids=ids, use_cache=False)
    real = torch.ones_like(ids)
    if pad in ("left", "right"):
        real[1, slice(0, 4) if pad == "left" else slice(9, 13)] = 0
        args["attention_mask"] = real
    if pad == "packed":
        args["position_ids"] = torch.cat([torch.arange(6), torch.arange(7)]).expand(2, -1)
    for m in (model, own):
        m.train()
    out = [m(**args).logits for m in (model, own)]
    soft = kind == "gemma2" and not kw                 # soft-capped scores and packed sequences stay on the usual path
    window = kw.get("sliding_window", 5 if kind in ("gemma2", "qwen2") else 0) % 64
    both = [0, window] if kind == "qwen2" else [window, 0] if kind == "gemma2" else [window, window]
    assert calls == ([] if pad == "packed" or soft else both)
    see = real.bool().unsqueeze(-1)
    scale = out[0].abs().max()
    assert ((out[0] - out[1]) * see).abs().max() <= NORMS * scale
    for m, o in zip((model, own), out):
        causal_lm_loss(o, ids.masked_fill(real == 0, -100)).backward()
    for (n, a), b in zip(model.named_parameters(), own.parameters()):
        assert (a.grad - b.grad).abs().max() <= NORMS * a.grad.abs().max() + NORMS * 1e-2, n


@pytest.mark.parametrize("kind", ["llama", "mistral"])
def test_generation_goes_on(kind):
    model = _llama(kind, **(dict(sliding_window=5) if kind == "mistral" else {}))
    own = copy.deepcopy(model)
    use_train_attention(own)
    ids = torch.randint(1, 97, (2, 9), generator=torch.Generator().manual_seed(2))
    mask = torch.ones_like(ids)
    mask[1, :3] = 0
    a, b = (m.eval().generate(ids, attention_mask=mask, max_new_tokens=7, do_sample=False, pad_token_id=0) for m in (model, own))
    assert torch.equal(a, b)


def test_encoder():
    import transformers as tr
    torch.manual_seed(1)
    cfg = tr.BertConfig(hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, vocab_size=50,
                        hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0, attn_implementation="sdpa")
    model = tr.BertModel(cfg).double()
    own = copy.deepcopy(model)
    assert use_train_attention(own)
    ids = torch.randint(1, 50, (2, 9), generator=torch.Generator().manual_seed(2))
    for mask in (None, torch.tensor([[1] * 9, [1] * 5 + [0] * 4])):
        a, b = (m.train()(input_ids=ids, attention_mask=mask).last_hidden_state for m in (model, own))
        see = slice(None) if mask is None else mask.bool()
        assert (a[see] - b[see]).abs().max() <= 1e-11


def test_refused_where_nothing_dispatches():
    from ipex_llm_b200.transformers.qlora import prepare_model_for_kbit_training
    with pytest.raises(RuntimeError, match="registry"):
        prepare_model_for_kbit_training(torch.nn.Sequential(torch.nn.Linear(3, 3)), False, use_fused_attention=True)


def _adapters(fused):
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import LoraConfig, get_peft_model, prepare_model_for_kbit_training
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      vocab_size=256, max_position_embeddings=128, tie_word_embeddings=False)
    torch.manual_seed(0)
    model = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.float32,
                                             modules_to_not_convert=["lm_head"], optimize_model=False, device="cpu")
    model = prepare_model_for_kbit_training(model, use_gradient_checkpointing=fused, use_fused_attention=fused)
    return get_peft_model(model, LoraConfig(r=4, lora_alpha=8, lora_dropout=0.0, target_modules=["q_proj", "v_proj"]))


def _samples(n, vocab, top=0):
    g = torch.Generator().manual_seed(1)
    out = []
    for i in range(n):
        ids = torch.randint(0, vocab, (5 + i % 4,), generator=g)
        s = {"input_ids": ids.tolist(), "labels": ids.tolist(), "attention_mask": [1] * len(ids)}
        if top:
            s.update(teacher_tokens(torch.randn(len(ids), vocab, generator=g), top)._asdict())
        out.append(s)
    return out


def test_collator_pads_teacher():
    batch = default_collator(_samples(2, 40, 3))
    assert batch["teacher_ids"].shape == (2, 6, 3) and batch["teacher_logits"].shape == (2, 6, 3)
    assert batch["teacher_logsumexp"].shape == (2, 6)
    assert (batch["teacher_ids"][0, 5:] == -1).all() and (batch["teacher_ids"][1] >= 0).all()
    assert batch["teacher_ids"].dtype == torch.long and batch["teacher_logits"].dtype == torch.float32


@pytest.mark.parametrize("top", [0, 8])
def test_trainer_runs_them_together(tmp_path, top):
    """A step with attention, loss and teacher: its gradients are those of the formula on the usual path."""
    from ipex_llm.transformers.qlora import TrainingArguments
    from ipex_llm_b200.train import Trainer
    data = _samples(4, 256, top)
    pm, ref = _adapters(True), _adapters(False)
    args = TrainingArguments(output_dir=str(tmp_path), per_device_train_batch_size=4, max_steps=2, logging_steps=1, bf16=False,
                             optim="adamw_torch", fused_loss=True, distill_weight=0.25, distill_temperature=1.0)
    tr = Trainer(pm, args, train_dataset=data)
    batch = default_collator(data)
    for m in (pm, ref):
        for i, p in enumerate(p for p in m.parameters() if p.requires_grad):
            torch.nn.init.normal_(p, std=0.05, generator=torch.Generator().manual_seed(i))
    pm.train(), ref.train()
    loss = tr.compute_loss(pm, dict(batch))
    labels = batch["labels"]
    logits = ref(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    want = F.cross_entropy(logits[:, :-1].flatten(0, 1), labels[:, 1:].flatten())
    if top:
        real = labels[:, 1:] != -100
        q = batch["teacher_logits"][:, :-1].exp()
        logp = torch.log_softmax(logits[:, :-1], -1)
        own = logp.gather(-1, batch["teacher_ids"][:, :-1].clamp(min=0))
        rest, left = 1 - q.sum(-1), 1 - own.exp().sum(-1)
        kl = (q * (q.log() - own)).sum(-1) + rest * (rest.log() - left.log())
        want = 0.75 * want + 0.25 * kl[real].sum() / real.sum()
    loss.backward()
    want.backward()
    # 32 bits all through: NORMS, and sums of up to 256 terms
    tol = NORMS + 256 * 2.0 ** -24
    assert abs(float(loss - want)) <= tol * max(1.0, abs(float(want)))
    for (n, a), b in zip(pm.named_parameters(), ref.parameters()):
        if a.requires_grad:
            assert (a.grad - b.grad).abs().max() <= tol * b.grad.abs().max() + 1e-6 * tol, n
    metrics = tr.train()
    assert metrics["train_loss"] == metrics["train_loss"] and tr.state.global_step == 2


def test_scores_of_tokens():
    from ipex_llm_b200.benchmark.perplexity import BigDLPPL
    model = _llama().float()
    ppl = BigDLPPL(model=model)
    ids = torch.randint(0, 97, (1, 12), generator=torch.Generator().manual_seed(2))
    got = ppl.token_scores(ids, entropy=True, top=3)
    total, n = ppl.nll(ids)
    assert got.logprob.shape == (1, 11) and got.top_ids.shape == (1, 11, 3) and n == 11
    assert abs(float(-got.logprob.sum()) - total) <= 64 * 2.0 ** -24 * total
    assert (got.entropy > 0).all() and (got.top_logprobs[..., 0] >= got.logprob).all()
