"""Calls of preference and policy finetuning that are easy to make and hard to notice: references that move, batches of another kind."""
import pytest
import torch
import torch.nn.functional as F

from ipex_llm_b200.train import Trainer, TrainerCallback, default_collator, sequence_logprobs


def _gen(seed):
    return torch.Generator().manual_seed(seed)


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
    kw = {"fused_loss": True, "max_steps": 5, "per_device_train_batch_size": 4, "optim": "adamw_multi", **kw}
    return TrainingArguments(output_dir=str(tmp_path), logging_steps=1, bf16=False, learning_rate=1e-2, **kw)


def _pairs(n=4, vocab=256):
    out = []
    for i in range(n):
        g = _gen(i)
        prompt, a, b = (torch.randint(0, vocab, (k,), generator=g).tolist() for k in (3, 4, 2 + i))
        out.append({"chosen_input_ids": prompt + a, "chosen_labels": [-100] * 3 + a, "rejected_input_ids": prompt + b,
                    "rejected_labels": [-100] * 3 + b})
    return out


def _with_reference(model, data):
    """Pairs with the log probabilities of the model without its adapters, as it is now."""
    batch = default_collator(data)
    model.disable_adapter_layers(True)
    with torch.no_grad():
        got = sequence_logprobs(model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits, batch["labels"])
    model.disable_adapter_layers(False)
    return [dict(s, reference_logprobs=[float(got[i]), float(got[len(data) + i])]) for i, s in enumerate(data)]


# ---- the reference of pairs --------------------------------------------------------------------------------------------------
def test_a_reference_that_restarts_would_move(tmp_path):
    """Restarts fold the adapters into the base, which then is no reference any more: it has to be given with the pairs."""
    from ipex_llm.transformers.relora import ReLoRATrainer
    model, data = _adapters(), _pairs()
    args = _args(tmp_path, preference_form="sigmoid", preference_beta=0.5)
    before = [p.detach().clone() for p in model.parameters() if p.requires_grad]
    with pytest.raises(RuntimeError, match="fold"):
        ReLoRATrainer(model, args, train_dataset=data, relora_steps=2).train()
    assert all(torch.equal(p, q) for p, q in zip((p for p in model.parameters() if p.requires_grad), before))
    args.preference_reference = False
    assert ReLoRATrainer(_adapters(), args, train_dataset=data, relora_steps=2).train()["train_loss"] > 0
    args.preference_reference = True
    given = _with_reference(model, data)
    batch = default_collator(given)
    seen = []

    class Watch(TrainerCallback):
        """The loss of the batch by its definition, before each step."""

        def on_step_begin(self, args, state, control, model=None, **kw):
            with torch.no_grad():
                logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
            h = sequence_logprobs(logits, batch["labels"]) - batch["reference_logprobs"]
            seen.append(float(-F.logsigmoid(0.5 * (h[:4] - h[4:])).mean()))
    trainer = ReLoRATrainer(model, args, train_dataset=given, relora_steps=2)
    trainer.callbacks.append(Watch())                 # behind the restarts
    trainer.train()
    assert trainer.relora.num_restarts == 2
    losses = [r["loss"] for r in trainer.state.log_history]
    # the batch's order is the only difference: sums of 32-bit numbers below 100
    assert losses == pytest.approx(seen, abs=1e-4)


def test_a_reference_whose_base_is_trained_would_move(tmp_path):
    model, data = _adapters(), _pairs()
    model.base_model.get_output_embeddings().weight.requires_grad_(True)
    trainer = Trainer(model, _args(tmp_path, preference_form="sigmoid"), train_dataset=data)
    with pytest.raises(RuntimeError, match="outside of the adapters.*lm_head"):
        trainer.compute_loss(model, default_collator(data))
    trainer.compute_loss(model, default_collator(_with_reference(model, data))).backward()
    trainer.args.preference_reference = False
    trainer.compute_loss(model, default_collator(data)).backward()


def test_a_base_that_took_the_adapters_in_is_no_reference(tmp_path):
    """Whoever folds the adapters in; a base that had them before the first loss is what finetuning begins with."""
    from ipex_llm.transformers.relora import merge_and_requantize
    model, data = _adapters(), _pairs()
    merge_and_requantize(model, reinit=True)
    trainer = Trainer(model, _args(tmp_path, preference_form="sigmoid"), train_dataset=data)
    trainer.compute_loss(model, default_collator(data)).backward()
    merge_and_requantize(model, reinit=True)
    with pytest.raises(RuntimeError, match="fold"):
        trainer.compute_loss(model, default_collator(data))
    trainer.compute_loss(model, default_collator(_with_reference(model, data))).backward()


# ---- batches of a policy -----------------------------------------------------------------------------------------------------
def _drawn(n=4, **kw):
    out = []
    for i in range(n):
        ids = torch.randint(0, 256, (6 + i,), generator=_gen(i)).tolist()
        out.append({"input_ids": ids, "labels": [-100] * 2 + ids[2:], "attention_mask": [1] * len(ids), "advantages": float(i - 1.5), **kw})
    return out


@pytest.mark.parametrize("args,match", [(dict(fused_loss=False), "fused_loss=True"), (dict(preference_form="sigmoid"), "preference_form")],
                         ids=["usual loss", "pairs"])
@pytest.mark.parametrize("columns", [("advantages",), ("advantages", "old_logprobs", "ref_logprobs"), ("old_logprobs",)], ids=str)
def test_a_policys_numbers_are_not_passed_over(tmp_path, args, match, columns):
    """A loss that does not know them would make completions of a negative advantage more likely."""
    model = _adapters()
    batch = default_collator(_drawn())
    for k in ("old_logprobs", "ref_logprobs"):
        batch[k] = torch.full(batch["input_ids"].shape, -5.0)
    batch = {k: v for k, v in batch.items() if k in columns or k in ("input_ids", "labels", "attention_mask")}
    trainer = Trainer(model, _args(tmp_path, **args), train_dataset=None, data_collator=lambda s: batch)
    with pytest.raises(RuntimeError, match=match):
        trainer.compute_loss(model, dict(batch))
    assert set(batch) == {"input_ids", "labels", "attention_mask", *columns}
    if "advantages" in columns:
        Trainer(model, _args(tmp_path)).compute_loss(model, dict(batch)).backward()


def test_old_log_probabilities_need_advantages(tmp_path):
    model = _adapters()
    batch = default_collator(_drawn(old_logprobs=[-5.0] * 6))
    del batch["advantages"]
    with pytest.raises(RuntimeError, match="without advantages"):
        Trainer(model, _args(tmp_path)).compute_loss(model, batch)


def test_a_teachers_tokens_and_references_are_not_passed_over(tmp_path):
    model = _adapters()
    batch = default_collator(_drawn())
    batch["teacher_ids"] = torch.zeros(*batch["input_ids"].shape, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no teacher"):
        Trainer(model, _args(tmp_path)).compute_loss(model, batch)
    batch = default_collator(_with_reference(model, _pairs()))
    for args in (dict(fused_loss=False), dict()):
        with pytest.raises(RuntimeError, match="reference_logprobs in the batch"):
            Trainer(model, _args(tmp_path, **args)).compute_loss(model, dict(batch))


def test_a_model_with_a_loss_of_its_own_gets_them(tmp_path):
    class Own(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.ones(1))

        def forward(self, input_ids, labels, attention_mask=None, advantages=None):
            return ((self.w * advantages).sum(),)
    batch = default_collator(_drawn())
    loss = Trainer(Own(), _args(tmp_path, fused_loss=False)).compute_loss(Own(), batch)
    assert float(loss.detach()) == float(batch["advantages"].sum())


def test_advantages_of_both_kinds_in_a_batch():
    """One number for a sample counts at each of its positions, also where another sample has one for each."""
    samples = [{"input_ids": [1, 2, 3], "labels": [1, 2, 3], "advantages": -1.0},
               {"input_ids": [1, 2, 3, 4], "labels": [1, 2, 3, 4], "advantages": [1.0, 2.0, 3.0, 4.0]},
               {"input_ids": [5], "labels": [5], "advantages": [0.5]}]
    assert default_collator(samples)["advantages"].tolist() == [[-1.0, -1.0, -1.0, 0.0], [1.0, 2.0, 3.0, 4.0], [0.5, 0.0, 0.0, 0.0]]
    assert default_collator([samples[0], samples[2]])["advantages"].tolist() == [[-1.0], [0.5]]


def test_columns_that_some_samples_lack():
    plain, drawn = {"input_ids": [1, 2], "labels": [1, 2]}, {"input_ids": [1, 2], "labels": [1, 2], "advantages": 1.0}
    pairs = _pairs(2)
    pairs[1]["reference_logprobs"] = [-1.0, -2.0]
    for samples, match in (([plain, drawn], "advantages"), ([drawn, plain], "advantages"), ([drawn, dict(drawn, ref_logprobs=[0.0, 0.0])],
                                                                                           "ref_logprobs"),
                           (pairs, "reference_logprobs"), (pairs[::-1], "reference_logprobs")):
        with pytest.raises(RuntimeError, match=f"{match} of some samples"):
            default_collator(samples)


def test_the_temperature_a_policy_was_sampled_at(tmp_path):
    from ipex_llm_b200.train import policy_lm_loss
    model = _adapters()
    batch = default_collator(_drawn(old_logprobs=[-5.0] * 6, ref_logprobs=[-5.5] * 6))
    trainer = Trainer(model, _args(tmp_path, policy_temperature=0.7, policy_kl_weight=0.1))
    loss = trainer.compute_loss(model, dict(batch))
    logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    numbers = [batch[k] for k in ("advantages", "old_logprobs", "ref_logprobs")]
    assert torch.equal(loss, policy_lm_loss(logits, batch["labels"], *numbers, kl_weight=0.1, temperature=0.7))
    assert not torch.equal(loss, policy_lm_loss(logits, batch["labels"], *numbers, kl_weight=0.1))


# ---- optimizers of the caller's own ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("own", [0.0, 1e-3])
def test_gradients_are_clipped_for_an_optimizer_that_does_not(tmp_path, own):
    from ipex_llm_b200.train import MultiTensorAdamW

    class Watch(MultiTensorAdamW):
        def step(self, closure=None):
            self.norm = float(torch.cat([p.grad.flatten() for g in self.param_groups for p in g["params"]]).norm())
            return super().step(closure)
    norms = []
    for limit in (0.0, 1e-3):
        model = _adapters()
        opt = Watch([p for p in model.parameters() if p.requires_grad], max_grad_norm=own)
        args = _args(tmp_path, max_grad_norm=limit, max_steps=1)
        Trainer(model, args, train_dataset=_drawn(), optimizers=(opt, None)).train()
        norms.append(opt.norm)
    # an optimizer that clips gets its gradients as they are
    assert norms[0] > 1e-2 and norms[1] == (norms[0] if own else pytest.approx(1e-3, rel=1e-3))


# ---- datasets ----------------------------------------------------------------------------------------------------------------
def test_datasets_without_a_length_or_places(tmp_path):
    """A trainer can be made of them, as for a loop of one's own over compute_loss."""
    class Stream(torch.utils.data.IterableDataset):
        def __iter__(self):
            return iter(_drawn())

    class Places(torch.utils.data.Dataset):
        def __len__(self):
            return 4
    model = _adapters()
    for data in (Stream(), iter(_drawn()), Places(), [], None):
        trainer = Trainer(model, _args(tmp_path), train_dataset=data)
    trainer.compute_loss(model, default_collator(list(Stream()))).backward()


def test_pairs_are_not_made_of_single_samples(tmp_path):
    """Halves of a shuffled batch of samples are no preferred and rejected ones."""
    model = _adapters()
    args = _args(tmp_path, preference_form="sigmoid")
    single = [{k: v for k, v in s.items() if k != "advantages"} for s in _drawn()]
    with pytest.raises(RuntimeError, match="needs pairs"):
        Trainer(model, args, train_dataset=single)
    # a collator of one's own makes them of what it is given
    given = default_collator(_pairs())
    trainer = Trainer(model, args, train_dataset=single, data_collator=lambda samples: given)
    trainer.compute_loss(model, trainer.collate(single)).backward()
