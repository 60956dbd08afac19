"""Preference and policy finetuning: losses on labels, pairs in batches, the optimizer over many tensors, and all of it in the trainer."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from ipex_llm_b200.train import (MultiTensorAdamW, Trainer, default_collator, next_tokens, policy_lm_loss, preference_lm_loss,
                                 sequence_logprobs)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _sums(logits, labels, average=False):
    t = next_tokens(labels)
    lp = torch.log_softmax(logits.double(), -1).gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    n = (t != -100).sum(1).clamp(min=1)
    s = torch.where(t != -100, lp, 0.0).sum(1)
    return s / n if average else s


@pytest.mark.parametrize("average", [False, True])
def test_preference_of_labels(average):
    logits = torch.randn(4, 9, 17, generator=_gen(0), dtype=torch.float64).requires_grad_()
    labels = torch.randint(0, 17, (4, 9), generator=_gen(1))
    labels[:, :3] = -100
    labels[2, 7:] = -100
    reference = sequence_logprobs(torch.randn(4, 9, 17, generator=_gen(2), dtype=torch.float64), labels, average)
    got = preference_lm_loss(logits, labels, reference, beta=0.3, average=average, likelihood_weight=0.5)
    s = _sums(logits, labels, average)
    h = s - reference.double()
    n = (next_tokens(labels) != -100).sum(1)
    want = -F.logsigmoid(0.3 * (h[:2] - h[2:])).mean() - 0.5 * (s[:2] / (1 if average else n[:2])).mean()
    assert torch.allclose(got, want, atol=1e-12)
    a, = torch.autograd.grad(got, logits)
    b, = torch.autograd.grad(want, logits)
    assert torch.allclose(a, b, atol=1e-12)


def test_policy_of_labels():
    logits = torch.randn(2, 7, 13, generator=_gen(0), dtype=torch.float64).requires_grad_()
    labels = torch.randint(0, 13, (2, 7), generator=_gen(1))
    labels[0, :2] = -100
    adv, old, ref = (torch.randn(2, 7, generator=_gen(i), dtype=torch.float64) - (3 if i > 2 else 0) for i in (2, 3, 4))
    got = policy_lm_loss(logits, labels, adv, old, ref, clip=(0.2, 0.3), kl_weight=0.1)
    t = next_tokens(labels)
    real = t != -100
    lp = torch.log_softmax(logits, -1).gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    w = torch.exp(lp - old)
    each = -torch.minimum(w * adv, w.clamp(0.8, 1.3) * adv) + 0.1 * (torch.exp(ref - lp) - (ref - lp) - 1)
    want = each[real].sum() / real.sum()
    assert torch.allclose(got, want, atol=1e-12)
    assert torch.allclose(torch.autograd.grad(got, logits)[0], torch.autograd.grad(want, logits)[0], atol=1e-12)


def _pairs(n, vocab, reference=False):
    out = []
    for i in range(n):
        g = _gen(i)
        prompt, a, b = (torch.randint(0, vocab, (k,), generator=g).tolist() for k in (3 + i % 2, 4, 2 + i))
        s = {"chosen_input_ids": prompt + a, "chosen_labels": [-100] * len(prompt) + a, "rejected_input_ids": prompt + b,
             "rejected_labels": [-100] * len(prompt) + b}
        if reference:
            s["reference_logprobs"] = [-20.0 - i, -15.0 + i]
        out.append(s)
    return out


def test_pairs_become_a_batch():
    batch = default_collator(_pairs(3, 50, True))
    assert batch["input_ids"].shape == batch["labels"].shape == batch["attention_mask"].shape == (6, 8)
    assert batch["reference_logprobs"].tolist() == [-20.0, -21.0, -22.0, -15.0, -14.0, -13.0]
    assert batch["input_ids"][1, :8].tolist()[:8] == _pairs(3, 50)[1]["chosen_input_ids"]
    assert (batch["labels"][0, :3] == -100).all() and (batch["labels"][3, 5:] == -100).all() and batch["attention_mask"][3].sum() == 5


def test_a_policys_columns_are_padded():
    samples = [{"input_ids": [1, 2, 3], "labels": [1, 2, 3], "advantages": 0.5, "old_logprobs": [-1.0, -2.0, 0.0]},
               {"input_ids": [1, 2], "labels": [1, 2], "advantages": [-1.5], "old_logprobs": [-3.0, 0.0]}]
    batch = default_collator(samples)
    assert batch["advantages"].tolist() == [[0.5], [-1.5]] and batch["old_logprobs"].tolist() == [[-1.0, -2.0, 0.0], [-3.0, 0.0, 0.0]]


def _adapters(seed=0):
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import LoraConfig, get_peft_model, prepare_model_for_kbit_training
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      vocab_size=256, max_position_embeddings=128, tie_word_embeddings=False)
    torch.manual_seed(0)
    model = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.float32,
                                             modules_to_not_convert=["lm_head"], optimize_model=False, device="cpu")
    model = get_peft_model(prepare_model_for_kbit_training(model, use_gradient_checkpointing=False),
                           LoraConfig(r=4, lora_alpha=8, lora_dropout=0.0, target_modules=["q_proj", "v_proj"]))
    for i, p in enumerate(p for p in model.parameters() if p.requires_grad):
        torch.nn.init.normal_(p, std=0.05, generator=_gen(seed + i))
    return model


def _args(tmp_path, **kw):
    from ipex_llm.transformers.qlora import TrainingArguments
    return TrainingArguments(output_dir=str(tmp_path), per_device_train_batch_size=4, max_steps=3, logging_steps=1, bf16=False,
                             fused_loss=True, learning_rate=1e-3, **kw)


@pytest.mark.parametrize("given", [False, True])
def test_trainer_on_pairs(tmp_path, given):
    """Its loss and gradients are those of the formula, with the batch's reference or the model without adapters."""
    data = _pairs(4, 256, given)
    model = _adapters()
    tr = Trainer(model, _args(tmp_path, optim="adamw_8bit", preference_form="sigmoid", preference_beta=0.4), train_dataset=data)
    batch = default_collator(data)
    reference = batch.get("reference_logprobs")
    if reference is None:
        model.disable_adapter_layers(True)
        with torch.no_grad():
            reference = _sums(model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits, batch["labels"])
        model.disable_adapter_layers(False)
    loss = tr.compute_loss(model, dict(batch))
    h = _sums(model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits, batch["labels"]) - reference.double()
    want = -F.logsigmoid(0.4 * (h[:4] - h[4:])).mean()
    params = [p for p in model.parameters() if p.requires_grad]
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5
    for a, b in zip(torch.autograd.grad(loss, params), torch.autograd.grad(want, params)):
        assert (a - b).norm() <= 1e-4 * b.norm() + 1e-7
    out = tr.train()
    assert isinstance(tr.optimizer, MultiTensorAdamW) and tr.optimizer.bits == 8 and math.isfinite(out["train_loss"])


def test_trainer_on_a_policys_batch(tmp_path):
    g = _gen(0)
    data = [{"input_ids": (ids := torch.randint(0, 256, (6 + i,), generator=g).tolist()), "labels": [-100] * 2 + ids[2:],
             "attention_mask": [1] * len(ids), "advantages": float(i - 1.5), "old_logprobs": [-5.0] * len(ids),
             "ref_logprobs": [-5.5] * len(ids)} for i in range(4)]
    model = _adapters()
    tr = Trainer(model, _args(tmp_path, optim="adamw_multi", policy_clip=(0.1, 0.3), policy_kl_weight=0.05), train_dataset=data)
    batch = default_collator(data)
    loss = tr.compute_loss(model, dict(batch))
    logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    want = policy_lm_loss(logits.double(), batch["labels"], batch["advantages"].double(), batch["old_logprobs"].double(),
                          batch["ref_logprobs"].double(), (0.1, 0.3), 0.05)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5
    assert math.isfinite(tr.train()["train_loss"]) and tr.optimizer.bits == 32


def test_trainer_refuses(tmp_path):
    data = _pairs(4, 256)
    for k, s in enumerate(data):
        s.pop("chosen_labels")
    model = _adapters()
    plain = torch.nn.Module()
    plain.register_parameter("w", torch.nn.Parameter(torch.zeros(1)))
    with pytest.raises(RuntimeError, match="pairs of samples need"):
        Trainer(model, _args(tmp_path), train_dataset=data)
    plain_loss = _args(tmp_path, preference_form="ipo")
    plain_loss.fused_loss = False
    with pytest.raises(RuntimeError, match="needs fused_loss"):
        Trainer(model, plain_loss, train_dataset=data)
    tr = Trainer(model, _args(tmp_path, preference_form="ipo"), train_dataset=data)
    with pytest.raises(RuntimeError, match="disable_adapter|adapters"):
        tr._preference_loss(plain, {"labels": torch.zeros(2, 3, dtype=torch.int64)})
    with pytest.raises(RuntimeError, match="no labels"):
        tr._preference_loss(model, {})
    with pytest.raises(RuntimeError, match="no labels"):
        tr._policy_loss(model, {"advantages": torch.zeros(1)})


# ---- the optimizer -----------------------------------------------------------------------------------------------------------
def _params(dtypes=(torch.float32,), seed=0):
    g = _gen(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.5).to(d)) for d in dtypes for s in ((7, 33), (300,), (1,))]


def _set_grads(params, seed, none=()):
    g = _gen(seed)
    for i, p in enumerate(params):
        d = torch.randn(p.shape, generator=g).to(p.dtype)
        p.grad = None if i in none else d


def test_optimizer_is_the_librarys():
    mine, theirs = _params(), [torch.nn.Parameter(p.detach().double()) for p in _params()]
    groups = [[0, 2], [1]]

    def of(ps, cls, **kw):
        return cls([{"params": [ps[i] for i in groups[0]], "weight_decay": 0.1}, {"params": [ps[i] for i in groups[1]], "lr": 3e-2}],
                   lr=1e-2, weight_decay=0.0, **kw)
    a, b = of(mine, MultiTensorAdamW, max_grad_norm=2.0), of(theirs, torch.optim.AdamW)
    for t in range(12):
        none = (1,) if t % 3 == 1 else ()
        _set_grads(mine, t, none)
        for p, q in zip(mine, theirs):
            q.grad = None if p.grad is None else p.grad.double()
        torch.nn.utils.clip_grad_norm_(theirs, 2.0)
        a.step()
        b.step()
    # 12 steps of some ten roundings of numbers below 4, and of changes of up to 3e-2
    for p, q in zip(mine, theirs):
        assert (p.double() - q).abs().max() <= 12 * 20 * 2.0 ** -24 * 4


@pytest.mark.parametrize("bits", [8, 32])
def test_state_is_saved_and_resumed(bits, tmp_path):
    dtypes = (torch.float32, torch.bfloat16, torch.float16)
    a, b = _params(dtypes), _params(dtypes)
    one, other = (MultiTensorAdamW(ps, lr=1e-2, bits=bits, max_grad_norm=1.0) for ps in (a, b))
    for t in range(3):
        _set_grads(a, t)
        one.step()
    torch.save(one.state_dict(), tmp_path / "o.pt")
    other.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=False))
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    for t in range(3, 6):
        _set_grads(a, t)
        _set_grads(b, t)
        one.step()
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(RuntimeError, match="other bits"):
        MultiTensorAdamW(_params(dtypes), bits=40 - bits).load_state_dict(one.state_dict())
    with pytest.raises(RuntimeError, match="before the first step"):
        one.add_param_group({"params": _params()})
    with pytest.raises(RuntimeError, match="32 or 8 bits"):
        MultiTensorAdamW(_params(), bits=16)
    with pytest.raises(RuntimeError, match="'copy' or None"):
        MultiTensorAdamW(_params(), rest="low")


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_that_change_and_moments_that_are_pruned(bits):
    """As a restart of the adapters does it."""
    from ipex_llm.transformers.relora import reset_optimizer
    ps = _params((torch.bfloat16, torch.float16))
    opt = MultiTensorAdamW(ps, lr=1e-3, bits=bits)
    for t in range(2):
        _set_grads(ps, t)
        opt.step()
    with torch.no_grad():
        for p in ps:
            p.fill_(0.75)
    opt.parameters_changed()
    reset_optimizer(opt, 0.9)
    for b in opt.buckets():
        m = b["state"].exp_avg.float()
        assert 0 < int((m != 0).sum()) <= 0.1 * m.numel() + 1
        # what is kept beside 0.75: nothing below bf16, or its copy
        kept, n = b["state"].rest, sum(p.numel() for p in b["params"])
        assert not kept.any() if kept.dtype == torch.int16 else int((kept == 0.75).sum()) == n


def test_trainer_resumes_with_it(tmp_path):
    data = _pairs(8, 256, True)
    args = _args(tmp_path, optim="adamw_8bit", preference_form="ipo", preference_average=True)
    args.max_steps, args.save_steps = 4, 2
    one = _adapters()
    Trainer(one, args, train_dataset=data).train()
    two = _adapters(50)
    tr = Trainer(two, copy.deepcopy(args), train_dataset=data)
    tr.train(resume_from_checkpoint=str(tmp_path / "checkpoint-2"))
    for (k, a), (_, b) in zip(one.state_dict().items(), two.state_dict().items()):
        if "lora_" in k:
            assert torch.equal(a, b), k


def test_layers_that_take_turns(tmp_path):
    """Layer-wise sampling: layers without a gradient stay, moments and step counters too."""
    from ipex_llm.transformers.lisa import DynamicLayerActivationCallback
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(hidden_size=32, intermediate_size=64, num_hidden_layers=3, num_attention_heads=2,
                                         num_key_value_heads=2, vocab_size=64, tie_word_embeddings=False))
    before = {k: v.clone() for k, v in model.state_dict().items()}
    data = [{"input_ids": torch.randint(0, 64, (9,), generator=_gen(i)).tolist()} for i in range(8)]
    args = _args(tmp_path, optim="adamw_8bit")
    args.max_steps = 2
    turns = DynamicLayerActivationCallback(n_layers=1, interval_steps=1, model=model, seed=1)
    tr = Trainer(model, args, train_dataset=data, callbacks=[turns])
    tr.create_optimizer()
    seen = set()
    turns.switch = turns.switch_active_layers
    turns.switch_active_layers = lambda: (turns.switch(), seen.update(turns.active_layers_indices))
    tr.train()
    (b,) = tr.optimizer.buckets()
    for (name, p), steps in zip(((n, p) for n, p in model.named_parameters()), b["state"].step.tolist()):
        layer = int(name.split(".")[2]) if ".layers." in name else None
        if layer is None:
            assert steps == 2
        else:
            assert (steps > 0) == (layer in seen)
            assert torch.equal(p, before[name]) == (layer not in seen), name
