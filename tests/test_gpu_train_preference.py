"""A finetuning step on the GPU, all its operators together: loss of pairs or of a policy, its gradients, their norm, the update."""
import math

import pytest
import torch
import torch.nn.functional as F

from ipex_llm_b200.ops import cuda_ops
from ipex_llm_b200.train import MultiTensorAdamW, Trainer, default_collator, next_tokens, policy_lm_loss, preference_lm_loss

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _sums(logits, labels):
    t = next_tokens(labels)
    lp = torch.log_softmax(logits, -1).gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return torch.where(t != -100, lp, 0.0).sum(1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("policy", [False, True])
def test_steps_of_a_small_model(dtype, bits, policy):
    """A table of hidden states and an output layer: the loss's gradients by the formula in 64 bits, the update bit by bit as on the
    CPU, over several steps."""
    g = _gen(0)
    B, S, H, V = 4, 37, 64, 1003
    make = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype)      # noqa: E731
    params = [make(B, S, H).cuda().requires_grad_(), make(H, V, std=H ** -0.5).cuda().requires_grad_()]
    here = [p.detach().cpu().requires_grad_() for p in params]
    labels = torch.randint(0, V, (B, S), generator=g)
    labels[:, :9] = -100
    labels[1, 30:] = -100
    dev = labels.cuda()
    reference = (torch.randn(B, generator=g) * 3 - 180).cuda()
    adv, old, ref = (torch.randn(B, S, generator=g) * 0.3 + m for m in (0.0, -7.0, -7.0))

    def loss_of(h, w, y, where):
        logits = h @ w
        if policy:
            return policy_lm_loss(logits, y, *(x.to(where, torch.float64 if h.dtype == torch.float64 else torch.float32)
                                               for x in (adv, old, ref)), kl_weight=0.1)
        return preference_lm_loss(logits, y, reference.to(where), beta=0.05, likelihood_weight=0.1)

    opt, same = (MultiTensorAdamW(ps, lr=1e-2, bits=bits, max_grad_norm=0.5, weight_decay=0.1, seed=3) for ps in (params, here))
    for _ in range(4):
        loss = loss_of(*params, dev, "cuda")
        loss.backward()
        wide = [p.detach().cpu().double().requires_grad_() for p in params]
        want = loss_of(*wide, labels, "cpu")
        exact = torch.autograd.grad(want, wide)
        # half a step of the type for the logits, their gradient, and the products' results: four roundings; logits reach 5 in size
        # and move a probability by that many times their rounding, the loss's slope by less
        tol = (4 + 5) * torch.finfo(dtype).eps / 2 + (2.0 ** -10 if dtype == torch.float32 else 0.0)      # tf32 or not
        for p, e in zip(params, exact):
            assert (p.grad.double().cpu() - e).norm() <= tol * e.norm()
        for p, q in zip(params, here):
            q.grad = p.grad.cpu()
        opt.step()
        same.step()
        opt.zero_grad()
        cuda_ops.check_error_flag(loss.device)
        for p, q in zip(params, here):
            # the norm's last bits may differ between the two, and so the clipping factor's
            assert (p.detach().cpu().float() - q.detach().float()).abs().max() <= 2 * torch.finfo(dtype).eps * q.detach().float().abs().max()
            with torch.no_grad():
                q.copy_(p)
        for b, c in zip(opt.buckets(), same.buckets()):
            for x, y in zip(b["state"], c["state"]):
                if x is not None:
                    raw = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[y.element_size()]
                    y.view(raw).copy_(x.view(raw))


def test_optimizer_over_types_groups_and_orders():
    """Parameters of three types, one of another order in memory, gradients of another order than theirs, none for some."""
    def make(where):
        g = _gen(1)
        out = []
        for d in (torch.float32, torch.bfloat16, torch.float16):
            for s in ((7, 33), (300,), (6, 50), (1,)):
                p = torch.randn(s, generator=g).to(where, d)
                out.append((p.t().contiguous().t() if s == (6, 50) else p).requires_grad_())
        return out
    a, b = make("cuda"), make("cpu")
    opts = [MultiTensorAdamW([{"params": ps[:5]}, {"params": ps[5:], "lr": 1e-3, "weight_decay": 0.1}], lr=1e-2, bits=8) for ps in (a, b)]
    for t in range(4):
        g = _gen(10 + t)
        for i, (p, q) in enumerate(zip(a, b)):
            d = torch.randn(p.shape, generator=g).to(p.dtype)
            p.grad = q.grad = None
            if i % 3 != t % 3:
                q.grad = d
                p.grad = d.cuda().t().contiguous().t() if i % 4 == 0 else d.cuda()
        for o in opts:
            o.step()
        for p, q in zip(a, b):
            assert torch.equal(p.detach().cpu(), q.detach())
    for x, y in zip(opts[0].buckets(), opts[1].buckets()):
        assert all(s is None or torch.equal(s.cpu().view(torch.uint8), c.view(torch.uint8)) for s, c in zip(x["state"], y["state"]))


def test_a_captured_step_of_everything():
    """Loss, gradients, norm and update in one graph: replays go on from where the last one ended, as eager steps do."""
    g = _gen(2)
    labels = torch.randint(0, 515, (2, 20), generator=g).cuda()
    x = torch.randn(2, 20, 32, generator=g).cuda()
    w0 = torch.randn(32, 515, generator=g).cuda() * 0.2

    def build():
        w = w0.clone().requires_grad_()
        return w, MultiTensorAdamW([w], lr=1e-2, bits=8, max_grad_norm=1.0)

    def step(w, opt):
        w.grad, = torch.autograd.grad(preference_lm_loss(x @ w, labels), w)
        opt.step()

    eager, opt = build()
    for _ in range(5):
        step(eager, opt)
    captured, opt = build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, opt)
        step(captured, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, opt)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, captured) and opt.buckets()[0]["state"].step.tolist() == [5]


@pytest.mark.parametrize("optim", ["adamw_8bit", "adamw_multi"])
def test_trainer_on_pairs(tmp_path, optim):
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import LoraConfig, TrainingArguments, cast_lora_weight, get_peft_model, prepare_model_for_kbit_training
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      vocab_size=1000, max_position_embeddings=256, tie_word_embeddings=False)
    model = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.bfloat16, modules_to_not_convert=["lm_head"],
                                             optimize_model=False, device="cuda")
    model = get_peft_model(prepare_model_for_kbit_training(model, use_gradient_checkpointing=True),
                           LoraConfig(r=8, lora_alpha=16, lora_dropout=0.0, target_modules=["q_proj", "v_proj", "down_proj"]))
    cast_lora_weight(model, torch.bfloat16)
    data = []
    for i in range(8):
        g = _gen(i)
        ids = [torch.randint(0, 1000, (k,), generator=g).tolist() for k in (5, 30 + i, 21)]
        data.append({"chosen_input_ids": ids[0] + ids[1], "chosen_labels": [-100] * 5 + ids[1], "rejected_input_ids": ids[0] + ids[2],
                     "rejected_labels": [-100] * 5 + ids[2]})
    args = TrainingArguments(output_dir=str(tmp_path), per_device_train_batch_size=4, max_steps=4, logging_steps=1, optim=optim,
                             fused_loss=True, preference_form="sigmoid", preference_beta=0.2, gradient_accumulation_steps=2)
    tr = Trainer(model, args, train_dataset=data)
    batch = {k: v.cuda() for k, v in default_collator(data[:4]).items()}
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = tr.compute_loss(model, dict(batch))
    # adapters begin at 0: the model is its own reference
    assert float(loss.detach()) == pytest.approx(math.log(2.0), abs=1e-4)
    params = [p for p in model.parameters() if p.requires_grad]
    own = torch.autograd.grad(loss, params)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = model(input_ids=batch["input_ids"], attention_mask=batch["attention_mask"]).logits
    s = _sums(logits.double(), batch["labels"])
    h = s - s.detach()
    want = torch.autograd.grad(-F.logsigmoid(0.2 * (h[:4] - h[4:])).mean(), params)
    own, want = (torch.cat([x.flatten().double() for x in xs]) for xs in (own, want))
    # both pass through the same bf16 layers; the logits' gradient is rounded to bf16 once on either side, two halves of a step
    assert (own - want).norm() <= 2 * 2.0 ** -8 * 4 * want.norm()
    out = tr.train()
    assert math.isfinite(out["train_loss"]) and isinstance(tr.optimizer, MultiTensorAdamW)
    assert tr.optimizer.bits == (8 if optim == "adamw_8bit" else 32)
    assert all(torch.isfinite(p).all() for p in params)
