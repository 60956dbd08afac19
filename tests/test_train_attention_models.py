"""The attention with a gradient inside models of other kinds and makes than plain decoders: what they compute stays what the
library's attention computes, on the CPU."""
import copy

import pytest
import torch

from ipex_llm_b200.models import train_attention
from ipex_llm_b200.models.train_attention import TRAIN_INTERFACE_NAME, use_train_attention

# Two paths in 32 bits over the same weights: a layer of these rounds some 100 numbers on a path (norms, products of up to 96
# terms, soft-max, residuals), each by 2^-24 of the largest number at hand; two layers, both paths, and 4 for what they amplify.
TOL = 2 * 2 * 100 * 4 * 2.0 ** -24


@pytest.fixture
def calls(monkeypatch):
    """The windows that the attention with a gradient was called with."""
    got, usual = [], train_attention.attention
    monkeypatch.setattr(train_attention, "attention", lambda *a: got.append(a[5]) or usual(*a))
    return got


BASE = dict(hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=97,
            max_position_embeddings=128, tie_word_embeddings=False, attn_implementation="sdpa", pad_token_id=0)


def _model(name, **kw):
    import transformers as tr
    torch.manual_seed(1)
    return getattr(tr, name + "ForCausalLM")(getattr(tr, name + "Config")(**{**BASE, **kw})).train()


def _inputs(pad, batch=2, tokens=13):
    ids = torch.randint(1, 97, (batch, tokens), generator=torch.Generator().manual_seed(2))
    if pad == "none":
        return dict(input_ids=ids)
    real = torch.ones_like(ids)
    if pad == "left":
        real[-1, :4] = 0
    if pad == "right":
        real[-1, 9:] = 0
    return dict(input_ids=ids, attention_mask=real)


def _same(model, own, args):
    x, y = (m(**args).logits for m in (model, own))
    off = (x - y).abs()
    if "attention_mask" in args:
        off = off * args["attention_mask"].unsqueeze(-1)
    assert off.max() <= TOL * x.abs().max()


def _optimised(model):
    from ipex_llm_b200.transformers.convert import _optimize_post, _optimize_pre
    return _optimize_post(_optimize_pre(model))


@pytest.mark.parametrize("name,kw", [("Llama", {}), ("Mistral", dict(sliding_window=64)), ("Qwen2", {}), ("Gemma", dict(head_dim=16)),
                                     ("Phi3", {}), ("Glm4", dict(head_dim=16))])
@pytest.mark.parametrize("use_cache", [False, True])
@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("pad", ["none", "ones", "left", "right"])
def test_optimised_models(name, kw, use_cache, batch, pad, calls):
    """Models loaded with their optimisations run this package's decoder forward: it takes the attention with a gradient, too."""
    model = _optimised(_model(name, **kw))
    own = copy.deepcopy(model)
    assert use_train_attention(own) and own.config._attn_implementation == TRAIN_INTERFACE_NAME
    _same(model, own, dict(_inputs(pad, batch), use_cache=use_cache))
    assert calls == [0, 0]


@pytest.mark.parametrize("pad", ["none", "ones"])
def test_no_logit_depends_on_a_later_token(pad, calls):
    own = _optimised(_model("Llama"))
    assert use_train_attention(own)
    args = dict(_inputs(pad, batch=1), use_cache=False)
    first = own(**args).logits
    args["input_ids"] = args["input_ids"].clone()
    args["input_ids"][0, -1] = args["input_ids"][0, -1] % 96 + 1
    again = own(**args).logits
    assert torch.equal(first[:, :-1], again[:, :-1]) and not torch.equal(first[:, -1], again[:, -1]) and len(calls) == 4


def test_optimised_models_by_the_public_calls(calls):
    """As a user loads and prepares one: the mask of ones that the collator gives, one sequence and several."""
    from transformers import LlamaConfig
    from ipex_llm.transformers import AutoModelForCausalLM
    from ipex_llm.transformers.qlora import prepare_model_for_kbit_training

    def load(fused):
        torch.manual_seed(0)
        cfg = LlamaConfig(**{**BASE, "attn_implementation": None})
        m = AutoModelForCausalLM.from_config(cfg, load_in_low_bit="nf4", torch_dtype=torch.float32, device="cpu", seed=0,
                                             modules_to_not_convert=["lm_head"])
        return prepare_model_for_kbit_training(m, use_gradient_checkpointing=False, use_fused_attention=fused).train()

    usual, fused = load(False), load(True)
    for batch in (1, 2):
        for pad in ("none", "ones", "right"):
            args = _inputs(pad, batch)
            calls.clear()
            _same(usual, fused, args)
            assert calls == [0, 0]


def test_generation_of_optimised_models():
    own = _optimised(_model("Llama"))
    usual = copy.deepcopy(own)
    assert use_train_attention(own)
    args = _inputs("left")
    a, b = (m.eval().generate(**args, max_new_tokens=7, do_sample=False) for m in (usual, own))
    assert torch.equal(a, b)


def test_attention_forwards_of_other_makes_are_left_alone():
    """A forward bound to the attention modules that does not reach the interface keeps its masks."""
    import types
    model = _model("Llama")

    def forward(self, hidden_states, position_embeddings=None, attention_mask=None, **kwargs):
        return type(self).forward(self, hidden_states, position_embeddings, attention_mask, **kwargs)

    model.model.layers[1].self_attn.forward = types.MethodType(forward, model.model.layers[1].self_attn)
    assert not use_train_attention(model) and model.config._attn_implementation == "sdpa"
    alibi = _model("Llama")
    alibi.config.ipex_alibi = True
    assert not use_train_attention(alibi)


def test_padding_is_no_mask_of_scores():
    """What carries padding cannot be added to scores, multiplied with them or handed to the library's attention."""
    mask = train_attention._compact(torch.ones(1, 5, dtype=torch.long))
    scores, q = torch.zeros(1, 2, 5, 5), torch.zeros(1, 2, 5, 8)
    for use in (lambda: scores + mask, lambda: scores * mask, lambda: (1.0 - mask) * -1e4, lambda: scores.masked_fill(mask, 0.0),
                lambda: torch.where(mask, scores, 0.0), lambda: mask[:, :, :, :5],
                lambda: torch.nn.functional.scaled_dot_product_attention(q, q, q, attn_mask=mask)):
        with pytest.raises((RuntimeError, NotImplementedError, IndexError)):
            use()


# Attention dropout this rare drops nothing in a few thousand numbers (chance 1e-5), but takes the path that drops.
RARELY = 1e-9


@pytest.mark.parametrize("name,kw,window", [("Llama", {}, 0), ("Mistral", dict(sliding_window=5), 5), ("Phi3", dict(sliding_window=7), 7)])
@pytest.mark.parametrize("pad", ["none", "ones", "left", "right"])
def test_dropout_keeps_the_mask(name, kw, window, pad, calls):
    model = _model(name, attention_dropout=RARELY, **kw)
    own = copy.deepcopy(model)
    assert use_train_attention(own)
    _same(model, own, dict(_inputs(pad), use_cache=False))
    assert calls == []


@pytest.mark.parametrize("Sq,Skv,window", [(9, 9, 4), (5, 12, 0), (5, 12, 3), (5, 12, 100)])
def test_dropout_of_windows_and_of_queries_behind_earlier_keys(Sq, Skv, window):
    from ipex_llm_b200.models.train_attention import train_attention_interface
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, h, s, 16, generator=g, dtype=torch.float64) for h, s in ((4, Sq), (2, Skv), (2, Skv)))
    module = torch.nn.Module().train()
    for d in (0.0, RARELY):
        got, _ = train_attention_interface(module, q, k, v, None, dropout=d, sliding_window=window or None)
        last, key = torch.arange(Skv - Sq, Skv).view(-1, 1), torch.arange(Skv)
        see = (key <= last) & (key > last - (window or Skv))
        s = (q @ k.repeat_interleave(2, 1).transpose(-1, -2) / 4).masked_fill(~see, -torch.inf)
        want = (torch.softmax(s, -1) @ v.repeat_interleave(2, 1)).transpose(1, 2)
        # sums of a few numbers in 64 bits; what is kept is scaled by 1 / (1 - RARELY)
        assert (got - want).abs().max() <= 1e-13 + 10 * RARELY * bool(d)


MOE = dict(num_experts=4, num_local_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, sliding_window=5)


@pytest.mark.parametrize("name,kw", [("Qwen2Moe", dict(use_sliding_window=True, max_window_layers=0, layer_types=["sliding_attention"] * 2,
                                                       shared_expert_intermediate_size=32)),
                                     ("Phimoe", {}), ("Mixtral", {})])
@pytest.mark.parametrize("optimised", [False, True])
@pytest.mark.parametrize("pad", ["none", "ones", "left", "right"])
def test_windows_that_only_the_mask_knows(name, kw, optimised, pad, calls):
    """Attention modules that do not hand their window to the interface: it comes with the mask."""
    model = _model(name, **{**MOE, **kw})
    if optimised:
        model = _optimised(model)
    own = copy.deepcopy(model)
    assert use_train_attention(own)
    _same(model, own, dict(_inputs(pad), use_cache=False))
    assert calls == [5, 5]
    _same(model.eval(), own.eval(), dict(_inputs(pad), use_cache=False))
    with torch.no_grad():
        _same(model, own, dict(_inputs(pad), use_cache=False))
    assert len(calls) == 4


@pytest.mark.parametrize("optimised", [False, True])
@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("pad", ["none", "left"])
def test_windows_behind_checkpoints(optimised, reentrant, pad, calls):
    """Checkpoints hand detached tensors on: the window is in their shape."""
    model = _model("Mistral", sliding_window=5)
    if optimised:
        model = _optimised(model)
    own = copy.deepcopy(model)
    assert use_train_attention(own)
    own.gradient_checkpointing_enable({"use_reentrant": reentrant})
    own.enable_input_require_grads()
    args = _inputs(pad)
    _same(model, own, dict(args, use_cache=False))
    assert calls and set(calls) == {5}
    see = args.get("attention_mask", torch.ones(2, 13)).unsqueeze(-1)
    for m in (model, own):
        (m(**args, use_cache=False).logits * see).square().mean().backward()
    for (n, a), b in zip(model.named_parameters(), own.parameters()):
        if a.grad is not None:
            assert (a.grad - b.grad).abs().max() <= 2 * TOL * a.grad.abs().max() + TOL * 1e-3, n


@pytest.mark.parametrize("window", [0, 4, 9, 100])
@pytest.mark.parametrize("Sq,Skv", [(9, 9), (4, 9)])
def test_what_masks_stand_for(window, Sq, Skv):
    real = torch.arange(Skv) >= torch.tensor([[0], [3]])
    last, key = torch.arange(Skv - Sq, Skv).view(-1, 1), torch.arange(Skv)
    see = (key <= last) & (key > last - (window or Skv))
    for padding in (real, real.long(), None):
        mask = train_attention._compact(padding, window, Skv)
        if mask is None:
            assert padding is None and window == 0
            continue
        want = see[None, None] if padding is None else see & real[:, None, None, :]
        assert torch.equal(train_attention.whole_mask(mask, Sq), want)
        assert torch.equal(train_attention.whole_mask(mask.detach(), Sq), want)


@pytest.mark.parametrize("q_length,kv_length", [(50, 50), (31, 50), (1, 7)])
@pytest.mark.parametrize("differs", [None, (0, 0), (13, 20), (30, 49)])
def test_windows_are_told_by_some_rows_at_a_time(q_length, kv_length, differs, monkeypatch):
    """Nothing of the size of queries x keys is made for long sequences, and every pair counts."""
    monkeypatch.setattr(train_attention, "_LOOKED_AT", 120)
    pairs = []

    def mask(batch, head, q, key):
        own = (key <= q) & (key > q - 9)
        pairs.append(own.numel())
        if differs is not None:
            own = own ^ ((q == differs[0] + kv_length - q_length) & (key == differs[1]))
        return own
    inside = differs is not None and differs[0] < q_length and differs[1] < kv_length
    assert train_attention._is_window(mask, q_length, kv_length, 9, "cpu") == (not inside)
    assert max(pairs) <= 120 and sum(pairs) == q_length * kv_length
    assert q_length == 1 or not train_attention._is_window(lambda b, h, q, k: True, q_length, kv_length, 9, "cpu")


@pytest.mark.parametrize("name,kw", [("Llama", {}), ("Mistral", dict(sliding_window=5)), ("Qwen2Moe", dict(
    MOE, use_sliding_window=True, max_window_layers=0, layer_types=["sliding_attention"] * 2, shared_expert_intermediate_size=32))])
@pytest.mark.parametrize("packed", [(0,), (1,), (0, 1)])
def test_sequences_packed_into_some_rows(name, kw, packed, calls):
    """A row that is one sequence says nothing about the others."""
    model = _model(name, **kw)
    own = copy.deepcopy(model)
    assert use_train_attention(own)
    at = torch.arange(13).repeat(2, 1)
    for i in packed:
        at[i, 4 + i:] = torch.arange(9 - i)
    _same(model, own, dict(_inputs("none"), position_ids=at, use_cache=False))
    assert calls == []


@pytest.mark.parametrize("optimised", [False, True])
def test_hooks_around_an_attention_are_looked_through(optimised, calls):
    """As device maps put them: the module's forward is a function of its own around the former one."""
    model = _model("Llama")
    if optimised:
        model = _optimised(model)
    own = copy.deepcopy(model)
    for layer in own.model.layers:
        m = layer.self_attn
        m._old_forward = m.forward
        m.forward = lambda *a, _m=m, **kw: _m._old_forward(*a, **kw)
    assert use_train_attention(own)
    _same(model, own, dict(_inputs("left"), use_cache=False))
    assert calls == [0, 0]


class _OtherLength:
    """A cache that keeps fewer keys than the mask was made for, or gives more."""

    def __init__(self, kept):
        self.kept = kept

    def update(self, k, v, layer_idx, **kw):
        return tuple(torch.cat([t, t], 2)[:, :, :self.kept] for t in (k, v))


@pytest.mark.parametrize("kept", [9, 13, 17])
@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("pad", [False, True])
def test_caches_of_another_length_than_the_mask(kept, window, pad):
    own = _optimised(_model("Llama")).eval()
    usual = copy.deepcopy(own)
    assert use_train_attention(own)
    x = torch.randn(2, 13, 64, generator=torch.Generator().manual_seed(3))
    rope = own.model.rotary_emb(x, torch.arange(13).unsqueeze(0))
    real = torch.arange(13) >= torch.tensor([[0], [3]])
    mask = train_attention._compact(real if pad else None, window, 13)
    whole = train_attention.whole_mask(mask, 13)
    with torch.no_grad():
        a, b = (m.model.layers[0].self_attn(x, position_embeddings=rope, attention_mask=t, past_key_values=_OtherLength(kept))[0]
                for m, t in ((usual, whole), (own, mask)))
    # rows that see nothing apart, the same operations
    assert (a - b).abs().max() <= TOL * a.abs().max()
