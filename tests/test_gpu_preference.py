"""Preference and policy losses on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import preference_oracle as oracle
from ipex_llm_b200.ops import cuda_ops
from ipex_llm_b200.ops.preference import policy_loss, preference_loss

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# odd vocabularies, rows of one batch and of many, fewer elements than a vector has, more rows than warps
SHAPES = [(2, 1, 1), (2, 3, 5), (4, 9, 33), (2, 40, 1000), (6, 17, 1029), (2, 5, 32000), (4, 33, 32003), (2, 700, 517), (2, 2, 128256),
          (10, 250, 2050)]


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) % (1 << 31))


def _logits(shape, dtype, g, std=2.5):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _targets(rows, V, g, kind="some"):
    t = torch.randint(0, V, rows, generator=g, device="cuda")
    if kind == "some":
        t[torch.rand(rows, generator=g, device="cuda") < 0.4] = -100
    elif kind == "prompts":
        t[:, :rows[1] // 3] = -100
    elif kind == "none":
        t[:] = -100
    elif kind == "one":
        keep = t[-1, 0].clone()
        t[:] = -100
        t[-1, 0] = keep
    return t


def _near(got, want, tol, what):
    got = got.detach().double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() / tol)
    assert bool((off <= 1).all()), (what, float(off.max()), int(off.argmax()))


def _check_preference(x, t, ref=None, more=True, **kw):
    P = x.shape[0] // 2
    x = x.detach().requires_grad_()
    g, gs = torch.randn(P, generator=_gen(1), device="cuda"), torch.randn(2 * P, generator=_gen(2), device="cuda") * 0.1
    got = preference_loss(x, t, ref, **kw)
    outs, grads = ((got.loss, got.logprob), (g, gs)) if more else ((got.loss,), (g,))
    dx, = torch.autograd.grad(outs, (x,), grads)
    assert dx.dtype == x.dtype and dx.shape == x.shape and not bool(dx[t == kw.get("ignore_index", -100)].any())
    want = oracle.preference(x, t, ref, g=g, g_seq=gs if more else None, **kw)
    for a, (b, tol), name in zip((got.loss, got.logprob, dx), want, ("loss", "logprob", "dlogits")):
        _near(a, b, tol, name)
    cuda_ops.check_error_flag(x.device)
    return dx


def _check_policy(x, t, adv, old=None, ref=None, **kw):
    x = x.detach().requires_grad_()
    g = torch.randn(t.shape, generator=_gen(3), device="cuda")
    got = policy_loss(x, t, adv, old, ref, **kw)
    dx, = torch.autograd.grad(got.loss, (x,), (g,))
    assert dx.dtype == x.dtype and not bool(dx[t == -100].any()) and not got.logprob.requires_grad
    *want, clipped = oracle.policy(x, t, adv, old, ref, g=g, **kw)
    sure = torch.ones(t.shape, dtype=torch.bool)
    if old is not None:
        sure = ~oracle.near_border(x, t, old, kw.get("clip", (0.2, 0.2)), kw.get("temperature", 1.0))
    assert torch.equal(got.clipped.cpu()[sure], clipped[sure])
    for a, (b, tol), name in zip((got.loss, got.logprob, got.kl, dx), want, ("loss", "logprob", "kl", "dlogits")):
        _near(a[sure.to(a.device)], b[sure], tol[sure], name)
    cuda_ops.check_error_flag(x.device)
    return got, dx


def _policy_inputs(x, t, g, temperature=1.0):
    lp = torch.log_softmax(x.float() / temperature, -1).gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    return torch.randn(t.shape, generator=g, device="cuda"), lp + 0.3 * torch.randn(t.shape, generator=g, device="cuda"), \
        lp + 0.5 * torch.randn(t.shape, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_preference_by_size(dtype, shape):
    g = _gen(shape)
    x = _logits(shape, dtype, g)
    t = _targets(shape[:2], shape[2], g)
    _check_preference(x, t, torch.randn(shape[0], generator=g, device="cuda") * shape[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_by_size(dtype, shape):
    g = _gen(shape)
    x = _logits(shape, dtype, g)
    t = _targets(shape[:2], shape[2], g)
    _check_policy(x, t, *_policy_inputs(x, t, g), kl_weight=0.2)


@pytest.mark.parametrize("tokens", [1, 127, 128, 129, 1023, 1024, 1025, 2048, 2049, 5000])
def test_lists_of_rows(tokens):
    """Around the number of rows up to which each CTA lists them for itself, and that which one pass over the targets takes."""
    g = _gen(tokens)
    x, t = _logits((2, tokens, 40), torch.float32, g), _targets((2, tokens), 40, g)
    _check_preference(x, t, average=True)
    _check_policy(x, t, *_policy_inputs(x, t, g), kl_weight=0.2)
    t[:] = -100
    t[1, -1] = 3
    _check_preference(x, t)


@pytest.mark.parametrize("kind", ["some", "prompts", "none", "one", "all"])
def test_which_rows_have_a_target(kind):
    g = _gen(kind)
    x = _logits((4, 300, 1003), torch.bfloat16, g)
    t = _targets((4, 300), 1003, g, kind)
    x[t == -100] = math.nan                               # their logits are not read
    y = x.nan_to_num(0.0)
    dx = _check_preference(y, t, average=True)
    z = x.detach().requires_grad_()
    got = preference_loss(z, t, average=True)
    same, = torch.autograd.grad((got.loss, got.logprob), (z,), (torch.randn(2, generator=_gen(1), device="cuda"),
                                                                 torch.randn(4, generator=_gen(2), device="cuda") * 0.1))
    assert torch.equal(dx, same)
    _, dx = _check_policy(y, t, *_policy_inputs(y, t, g), kl_weight=0.2)


@pytest.mark.parametrize("kw", [dict(form="sigmoid", label_smoothing=0.2, margin=0.5, beta=0.5), dict(form="hinge", beta=0.02), dict(form="ipo"),
                                dict(form="ipo", average=True, beta=0.5), dict(form="sigmoid", temperature=0.5),
                                dict(form="sigmoid", ignore_index=7)])
@pytest.mark.parametrize("more", [False, True])
def test_preference_forms(kw, more):
    g = _gen(str(kw))
    x, t = _logits((6, 50, 2003), torch.float32, g), _targets((6, 50), 2003, g, "all")
    t[t == 3] = 4
    t[:, :9] = kw.get("ignore_index", -100)
    _check_preference(x, t, None, more=more, **kw)
    _check_preference(x, t, torch.randn(6, generator=g, device="cuda") * 50 - 400, more=more, **kw)


@pytest.mark.parametrize("gap", [-3e4, -200.0, 200.0, 3e4])
@pytest.mark.parametrize("form", ["sigmoid", "hinge", "ipo"])
def test_preference_far_from_even(gap, form):
    x = torch.zeros(2, 1, 2, device="cuda")
    x[0, 0, 0], x[1, 0, 0] = gap, -gap
    _check_preference(x, torch.zeros(2, 1, dtype=torch.int64, device="cuda"), form=form, beta=0.9, label_smoothing=0.1 if form == "sigmoid" else 0.0)


@pytest.mark.parametrize("case", ["first", "no clip", "one advantage", "temperature", "one dimension", "four dimensions", "reference without weight"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_policy_cases(case, dtype):
    g = _gen(case)
    shape = {"one dimension": (33,), "four dimensions": (2, 3, 5)}.get(case, (3, 40))
    x, t = _logits((*shape, 1501), dtype, g), torch.randint(0, 1501, shape, generator=g, device="cuda")
    t.view(-1)[::4] = -100
    kw = dict(kl_weight=0.1, clip=(0.1, 0.4), temperature=1.7 if case == "temperature" else 1.0)
    adv, old, ref = _policy_inputs(x, t, g, kw["temperature"])
    if case == "first":
        old = None
    if case == "no clip":
        kw["clip"] = (1.0, 1e30)
    if case == "one advantage":
        adv = adv[:, :1]
    if case == "four dimensions":
        adv = adv[:, :1, :1]
    if case == "reference without weight":
        kw["kl_weight"] = 0.0
    got, _ = _check_policy(x, t, adv, old, ref, **kw)
    assert bool(got.clipped.any()) == (case not in ("first", "no clip"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [-math.inf, "lowest", -3e4])
def test_hidden_tokens(dtype, value):
    """Masks of -inf, of the type's lowest value and of a far number, a row that they leave one token of, and one of none."""
    g = _gen(dtype)
    value = torch.finfo(dtype).min if value == "lowest" else value
    x = _logits((2, 20, 700), dtype, g)
    t = torch.randint(0, 300, (2, 20), generator=g, device="cuda")
    x[:, :, 300:] = value
    x[0, 3, :300], x[1, 5] = value, value
    x[0, 3, 7] = 1.0
    t[0, 3] = 7
    if value != -3e4 and (value == -math.inf or dtype != torch.float16):
        t[1, 5] = -100                                   # no token at all is left: tested below
    _check_preference(x, t)
    adv, old, ref = _policy_inputs(x, t, g)
    _check_policy(x, t, adv, old, ref, kl_weight=0.1)


def test_rows_without_a_token_and_hidden_targets():
    x = torch.full((2, 2, 9), -math.inf, device="cuda")
    x[:, 1, :4] = torch.randn(2, 4, device="cuda")
    t = torch.tensor([[1, 7], [-100, 2]], device="cuda")
    x.requires_grad_()
    got = policy_loss(x, t, torch.ones(2, 2, device="cuda"), torch.full((2, 2), -1.0, device="cuda"), torch.full((2, 2), -1.0, device="cuda"),
                      kl_weight=0.1)
    dx, = torch.autograd.grad(got.loss.sum(), x)
    assert torch.equal(got.logprob[0], torch.full((2,), -math.inf, device="cuda")) and torch.isfinite(got.loss[1]).all()
    assert (got.kl[0] == math.inf).all() and (got.loss[0] == math.inf).all() and not dx[0].any() and bool(dx[1, 1, :4].all())
    got = policy_loss(x, t, torch.ones(2, 2, device="cuda"), torch.full((2, 2), -1.0, device="cuda"))
    assert (got.loss[0] == 0.0).all()
    got = policy_loss(x, t, torch.ones(2, 2, device="cuda"))
    assert (got.loss[0] == -1.0).all() and not torch.autograd.grad(got.loss.sum(), x)[0][0].any()


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_is_not_finite_stays_in_its_row(value):
    g = _gen(5)
    x, t = _logits((2, 30, 5003), torch.bfloat16, g), _targets((2, 30), 5003, g, "all")
    adv, old, ref = _policy_inputs(x, t, g)
    x[0, 4, 4001] = value
    x.requires_grad_()
    got = policy_loss(x, t, adv, old)
    dx, = torch.autograd.grad(got.loss.sum(), x)
    bad = torch.zeros(2, 30, dtype=torch.bool, device="cuda")
    bad[0, 4] = True
    assert torch.equal(got.loss.isnan(), bad) and torch.equal(dx.isnan().any(-1), bad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_logits(dtype):
    """Logits whose exponents pass 2^24, and a temperature that takes them there."""
    g = _gen(8)
    x, t = _logits((2, 9, 600), dtype, g), _targets((2, 9), 600, g, "all")
    far = x + (3e4 if dtype == torch.float16 else 1e9)
    t2 = far.float().argmax(-1)
    _check_preference(far, t2, temperature=1.0)
    _check_preference((x * 100).to(dtype), x.float().argmax(-1), temperature=1e-3)


def test_strided_and_shifted_logits():
    g = _gen(6)
    whole = _logits((2, 41, 1007), torch.bfloat16, g)
    x = whole[:, :-1]
    t = _targets((2, 40), 1007, g)
    a = _check_preference(x, t)
    assert torch.equal(a, _check_preference(x.contiguous(), t))
    wide = _logits((2, 40, 1100), torch.float32, g)
    for part in (wide[..., 3:1010], wide[:, ::2, :1007], wide[..., ::2]):
        t = _targets(part.shape[:2], part.shape[2], g)
        # where a row lies decides which lane adds what: each is near the definition, not bit by bit the other
        _check_preference(part, t)
        _check_preference(part.contiguous(), t)
        _check_policy(part, t, *_policy_inputs(part, t, g), kl_weight=0.1)
    same = _logits((1, 40, 1007), torch.float32, g).expand(2, -1, -1)
    _check_preference(same, _targets((2, 40), 1007, g))


def test_repeatable_and_independent_of_the_batch():
    g = _gen(7)
    x, t = _logits((2, 200, 3001), torch.bfloat16, g), _targets((2, 200), 3001, g)
    a, b = _check_preference(x, t), _check_preference(x, t)
    assert torch.equal(a, b)


def test_gradients_that_are_broadcast():
    g = _gen(9)
    x, t = _logits((4, 30, 1003), torch.float32, g).requires_grad_(), _targets((4, 30), 1003, g)
    adv, old, ref = _policy_inputs(x.detach(), t, g)
    a, = torch.autograd.grad(policy_loss(x, t, adv, old).loss.mean(), x)
    b, = torch.autograd.grad(policy_loss(x, t, adv, old).loss, x, torch.full((4, 30), 1 / 120, device="cuda"))
    assert torch.equal(a, b)
    a, = torch.autograd.grad(preference_loss(x, t).loss.sum(), x)
    b, = torch.autograd.grad(preference_loss(x, t).loss, x, torch.ones(2, device="cuda"))
    assert torch.equal(a, b)
    a, = torch.autograd.grad(preference_loss(x, t).logprob[2], x)
    assert not a[[0, 1, 3]].any()


def test_backward_twice_and_captured():
    g = _gen(10)
    x, t = _logits((2, 30, 1003), torch.bfloat16, g).requires_grad_(), _targets((2, 30), 1003, g)
    ref = torch.randn(2, generator=g, device="cuda")
    eager = preference_loss(x, t, ref).loss.sum()
    want, = torch.autograd.grad(eager, x, retain_graph=True)
    again, = torch.autograd.grad(eager, x, retain_graph=True)
    assert torch.equal(want, again)
    del eager                        # a leaf's graph on another stream would end the capture, whatever its operators
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(preference_loss(x, t, ref).loss.sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = preference_loss(x, t, ref).loss
        dx, = torch.autograd.grad(loss.sum(), x)
    with torch.no_grad():
        keep = x.clone()
        x.copy_(_logits((2, 30, 1003), torch.bfloat16, g))
        x[0, 3] = keep[0, 3]
    t[:, 5:9] = -100
    graph.replay()
    torch.cuda.synchronize()
    now, = torch.autograd.grad(preference_loss(x, t, ref).loss.sum(), x)
    assert torch.equal(dx, now) and not torch.equal(dx, want)


@pytest.mark.parametrize("bad", [300, -1, 1 << 40])
def test_targets_outside_of_the_vocabulary(bad):
    """Their pair is NaN, or their row; the others are not."""
    g = _gen(11)
    x, t = _logits((4, 9, 300), torch.bfloat16, g).requires_grad_(), _targets((4, 9), 300, g, "all")
    t[0, 3] = bad
    for pairs in (True, False):
        loss = preference_loss(x, t).loss if pairs else policy_loss(x, t, torch.ones(4, 9, device="cuda")).loss
        with pytest.raises(RuntimeError, match="61"):
            cuda_ops.check_error_flag(x.device)
        dx, = torch.autograd.grad(loss.sum(), x)
        cuda_ops.check_error_flag(x.device)
        spoiled = torch.zeros(4, 9, dtype=torch.bool, device="cuda")
        if pairs:
            spoiled[[0, 2]] = True
            assert loss.isnan().tolist() == [True, False]
        else:
            spoiled[0, 3] = True
            assert torch.equal(loss.isnan(), spoiled)
        assert torch.equal(dx.isnan().all(-1), spoiled) and torch.equal(dx.isnan().any(-1), spoiled)


def test_another_stream_and_grad_modes():
    g = _gen(12)
    x, t = _logits((2, 9, 300), torch.bfloat16, g), _targets((2, 9), 300, g, "all")
    want = preference_loss(x, t)
    assert not want.loss.requires_grad
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        got = preference_loss(x.clone().requires_grad_(), t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.loss, want.loss) and not got.loss.requires_grad
    empty = policy_loss(x[:, :0], t[:, :0], torch.ones(2, 0, device="cuda"))
    assert empty.loss.shape == (2, 0)


def test_rows_past_32_bits():
    """Rows whose elements begin past 2^32."""
    V = (1 << 25) + 9
    x = torch.zeros(2, 70, V, dtype=torch.bfloat16, device="cuda")
    t = torch.full((2, 70), -100, device="cuda")
    t[0, 1], t[1, 69] = 5, V - 1
    x[1, 69, V - 1] = 10.0
    x.requires_grad_()
    got = preference_loss(x, t)
    lse = math.log(V - 1 + math.exp(10.0))
    # 2^20 batches to a lane at most: 32-bit sums of equal terms, each rounded
    assert abs(float(got.logprob[0]) + math.log(V)) <= 1e-4 and abs(float(got.logprob[1]) - 10.0 + lse) <= 1e-4
    dx, = torch.autograd.grad(got.logprob, x, torch.tensor([1.0, 2.0], device="cuda"))
    assert float(dx[0, 1, 5]) == 1.0 and float(dx[1, 69, V - 1]) == pytest.approx(2 * (1 - math.exp(10.0 - lse)), rel=2.0 ** -8)
    assert int((dx != 0).sum()) == 2 * V


def test_a_gradients_gradient_is_refused():
    x, t = torch.randn(2, 3, 9, device="cuda", requires_grad=True), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for call in (lambda: preference_loss(x, t).loss, lambda: policy_loss(x, t, torch.ones(2, 3, device="cuda")).loss):
        want, = torch.autograd.grad(call().sum(), x)
        dx, = torch.autograd.grad(call().sum(), x, create_graph=True)
        assert torch.equal(dx.detach(), want)
        with pytest.raises(RuntimeError, match="used in the graph"):
            torch.autograd.grad(dx.sum(), x, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            dx.sum().backward()


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_a_dominant_token_among_many(rows):
    """One logit 60 octaves above thousands that come before it, and after it: the sums' reference moves once, or not at all."""
    g = _gen(rows)
    x = _logits((2, rows, 40000), torch.float32, g)
    t = torch.randint(0, 40000, (2, rows), generator=g, device="cuda")
    for at in (0, 20011, 39999):
        y = x.clone()
        y[:, :, at] += 42.0
        _check_preference(y, t)
        y[:, :, at] = 9.0                                  # a few octaves above the largest others
        _check_preference(y, torch.full_like(t, at))


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    x, t = torch.randn(2, 3, 9, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            preference_loss(d, t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy_loss(d, t, torch.ones(2, 3, device="cuda"))


def test_refusals_on_the_gpu():
    x, t = torch.randn(2, 3, 9, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="on cuda"):
        preference_loss(x, t.cpu())
    with pytest.raises(RuntimeError, match="advantages should hold"):
        policy_loss(x, t, torch.ones(2, 3))
    with pytest.raises(RuntimeError, match="not supported"):
        preference_loss(x.double(), t)
    with pytest.raises(RuntimeError, match="no tokens"):
        preference_loss(x[:, :0], t[:, :0])
