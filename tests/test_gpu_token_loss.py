"""Log probabilities of given tokens and distillation on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import token_loss_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(hash(key) % (1 << 31))


def _logits(shape, dtype, g, std=2.5):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _near(got, want, tol, what):
    got, want = got.detach().double().cpu(), want
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs() / tol)
    assert bool((off <= 1).all()), (what, float(off.max()), int(off.argmax()))


def _check_logprobs(x, t, temperature, top, grads=True):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import token_logprobs
    V = x.shape[-1]
    g = torch.randn(t.shape, generator=_gen(V, 1), device="cuda")
    ge = torch.randn(t.shape, generator=_gen(V, 2), device="cuda")
    x = x.detach().requires_grad_(grads)
    r = token_logprobs(x, t, temperature=temperature, entropy=True, top=top)
    lp, ent, logp, dx = oracle.logprobs(x, t, temperature, g if grads else None, ge)
    _near(r.logprob, lp, oracle.value_tol(V, lp, temperature), "logprob")
    _near(r.entropy, ent, oracle.value_tol(V, ent, temperature), "entropy")
    if top:
        order = torch.sort(x.detach().float(), dim=-1, descending=True, stable=True).indices[..., :top]
        assert torch.equal(r.top_ids, order)
        best = logp.gather(-1, order.cpu())
        _near(r.top_logprobs, best, oracle.value_tol(V, best, temperature), "top")
        assert not r.top_logprobs.requires_grad
    if grads:
        got, = torch.autograd.grad((r.logprob, r.entropy), (x,), (g, ge))
        assert got.dtype == x.dtype and got.shape == x.shape
        size = (g.abs() + ge.abs()).double().cpu().unsqueeze(-1)
        _near(got, dx, oracle.grad_tol(dx, x.dtype, V, size, temperature), "dlogits")
        only, = torch.autograd.grad(token_logprobs(x, t, temperature=temperature).logprob, (x,), (g,))
        zero = torch.zeros_like(ge)
        want = oracle.logprobs(x, t, temperature, g, zero)[3]
        _near(only, want, oracle.grad_tol(want, x.dtype, V, g.abs().double().cpu().unsqueeze(-1), temperature), "dlogits of logprob")
    cuda_ops.check_error_flag(x.device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 33), (1, 32000), (5, 32003), (150, 1000), (300, 517), (2, 128256),
                                   (20, 4100)])
def test_logprobs_by_size(dtype, shape):
    g = _gen(shape)
    x = _logits(shape, dtype, g)
    t = torch.randint(0, shape[1], (shape[0],), generator=g, device="cuda")
    _check_logprobs(x, t, 1.0, min(20, shape[1]))


@pytest.mark.parametrize("temperature", [0.5, 0.7, 3.0])
@pytest.mark.parametrize("top", [0, 1, 32])
def test_logprobs_by_temperature(temperature, top):
    g = _gen(top)
    x = _logits((2, 9, 5003), torch.float16, g)
    t = torch.randint(0, 5003, (2, 9), generator=g, device="cuda")
    t[0, 3] = t[1, 8] = -100
    _check_logprobs(x, t, temperature, top)


@pytest.mark.parametrize("rows", [2, 200])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "one thread", "two values"])
def test_best_tokens_in_awkward_orders(kind, rows):
    V = 40000
    at = torch.arange(V, device="cuda")
    x = {"equal": torch.zeros(V, device="cuda"), "rising": at / 1000.0, "falling": -at / 1000.0,
         # 16-byte vectors of 512 threads: columns whose vector belongs to a few of them hold all large values
         "one thread": torch.where(at // 4 % 512 < 40, 5.0 + (at * 7919 % 1000) / 500.0, (at * 104729 % 1000) / 500.0),
         "two values": (at * 7919 % 3 == 0).float()}[kind]
    x = x.float().expand(rows, V).contiguous()
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    _check_logprobs(x, t, 1.0, 32, grads=False)
    _check_logprobs(x.to(torch.bfloat16), t, 1.0, 32, grads=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_tokens_and_rows_without_any(dtype):
    from ipex_llm_b200.ops.token_loss import token_logprobs
    g = _gen(5)
    x = _logits((6, 1003), dtype, g)
    x[0, 17:] = -math.inf                       # a few are left
    x[1] = -math.inf                            # none is left
    x[2, ::2] = torch.finfo(dtype).min          # the type's lowest value
    x[3, 5] = -math.inf                         # the target is hidden
    x[4] = math.nan                             # no target: what the row holds does not matter
    t = torch.tensor([3, 3, 7, 5, -100, 0], device="cuda")
    keep = torch.tensor([0, 2, 5], device="cuda")
    _check_logprobs(x[keep], t[keep], 1.0, 16)
    x.requires_grad_()
    r = token_logprobs(x, t, entropy=True, top=20)
    assert r.logprob[1] == -math.inf and r.entropy[1] == 0 and r.logprob[3] == -math.inf and r.entropy[3] > 0
    assert r.logprob[4] == 0 and r.entropy[4] == 0 and bool((r.top_logprobs[1] == -math.inf).all())
    assert torch.equal(r.top_ids[1], torch.arange(20, device="cuda")) and torch.equal(r.top_ids[0, :17].sort().values, torch.arange(17, device="cuda"))
    dx, = torch.autograd.grad((r.logprob.sum() + r.entropy.sum()), (x,))
    assert bool((dx[1] == 0).all()) and bool((dx[4] == 0).all()) and bool(dx.isfinite().all())


def test_nan_and_infinity_are_not_swallowed():
    from ipex_llm_b200.ops.token_loss import token_logprobs
    x = torch.zeros(3, 5000, device="cuda")
    x[0, 4321], x[1, 17] = math.nan, math.inf
    r = token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"), entropy=True, top=2)
    assert r.logprob[:2].isnan().all() and r.entropy[:2].isnan().all() and r.logprob[2].isfinite()
    assert r.top_ids[:, 0].tolist() == [4321, 17, 0]


def test_target_outside_of_the_vocabulary():
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import token_logprobs
    x = torch.zeros(2, 50, device="cuda", requires_grad=True)
    cuda_ops.check_error_flag(x.device)
    r = token_logprobs(x, torch.tensor([50, 1], device="cuda"), entropy=True)
    assert r.logprob[0].isnan() and r.entropy[0].isnan() and r.logprob[1].isfinite()
    dx, = torch.autograd.grad(r.logprob.sum(), (x,))
    assert dx[0].isnan().all() and dx[1].isfinite().all()
    with pytest.raises(RuntimeError, match="61"):
        cuda_ops.check_error_flag(x.device)


def test_rows_of_any_stride():
    g = _gen(9)
    base = _logits((3, 11, 1009 + 6), torch.bfloat16, g)
    t = torch.randint(0, 1009, (3, 10), generator=g, device="cuda")
    _check_logprobs(base[:, :-1, 3:1012], t, 1.0, 5)                          # unaligned, a gap behind every row and sequence
    _check_logprobs(base[:, :-1, :2018:2][..., :505], t % 505, 1.0, 5)        # no unit stride
    _check_logprobs(base[:1, :1, :1009].expand(3, 10, 1009), t, 1.0, 5)       # one row for all
    _check_logprobs(base[0, 0, :1009], t[0, 0], 1.0, 5)                       # a single row
    _check_logprobs(base[:, :10, :1000].reshape(3, 2, 5, 1000), t.reshape(3, 2, 5) % 1000, 1.0, 5)


def _teacher(x, k, temperature, g):
    teacher = 1.1 * x.float() + torch.randn(x.shape, generator=g, device="cuda") * 0.5
    best = torch.topk(teacher, k, dim=-1)
    return best.indices, best.values, torch.logsumexp(teacher / temperature, dim=-1)


def _check_distill(x, ids, values, lse, temperature):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import distill_loss
    V = x.shape[-1]
    g = torch.randn(x.shape[:-1], generator=_gen(V, 3), device="cuda")
    x = x.detach().requires_grad_()
    loss = distill_loss(x, ids, values, temperature=temperature, teacher_logsumexp=lse)
    want, dx = oracle.distill(x, ids, values, temperature, lse, g)
    # log q - log p: both as log probabilities are, weighted by q, and T^2 in front; the teacher's exponents |t / T - lse| are
    # rounded like them; rest = 1 - sum q and `left` add their own relative errors times their logarithms' slope of 1
    size = float(values.abs().max()) / temperature + math.log(V) + 20
    tol = oracle.U * (4 * oracle.sum_steps(V) + ids.shape[-1] + 24 * size) * temperature ** 2
    _near(loss, want, tol, "loss")
    got, = torch.autograd.grad(loss, (x,), (g,))
    assert got.dtype == x.dtype
    # rest / left is as exact as the cancellation 1 - sum q, which belongs to the inputs' 32 bits: K + 2 |t / T| units of U,
    # divided by left and multiplied by p_j <= left
    scale = g.abs().double().cpu().unsqueeze(-1) * temperature ** 2
    _near(got, dx, oracle.grad_tol(dx, x.dtype, V, scale * (1 + (ids.shape[-1] + 2 * size) / 64), temperature), "dlogits")
    cuda_ops.check_error_flag(x.device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("shape,k", [((1, 40), 5), ((3, 33), 33), ((2, 32000), 64), ((5, 32003), 8), ((160, 1001), 1),
                                     ((2, 128256), 100), ((3, 5000), 1024)])
def test_distill_by_size(dtype, tail, shape, k):
    g = _gen(shape, k)
    x = _logits(shape, dtype, g)
    for temperature in (1.0, 2.0):
        ids, values, lse = _teacher(x, k, temperature, g)
        if tail and k == shape[1]:
            lse = lse + 0.125                    # the teacher knows a token more than the student
        _check_distill(x, ids, values, lse if tail else None, temperature)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_padding_and_repeated_ids(tail):
    from ipex_llm_b200.ops.token_loss import distill_loss
    g = _gen(21)
    x = _logits((2, 4, 2051), torch.bfloat16, g)
    ids, values, lse = _teacher(x, 12, 1.0, g)
    ids[0, 1, 5:] = -1
    ids[0, 2, 3] = ids[0, 2, 4] = ids[0, 2, 11]            # three of one
    ids[1, 0] = ids[1, 0, :1]                              # all of one
    if tail:
        lse = lse + 1.0                                    # so that repeated ids leave something
    _check_distill(x, ids, values, lse if tail else None, 1.0)
    ids[1, 3] = -1                                         # a row without a teacher
    x = x.requires_grad_()
    loss = distill_loss(x, ids, values, teacher_logsumexp=lse if tail else None)
    assert loss[1, 3] == 0
    dx, = torch.autograd.grad(loss.sum(), (x,))
    assert bool((dx[1, 3] == 0).all()) and bool((dx[1, 2] != 0).any())


def test_distill_hidden_tokens():
    from ipex_llm_b200.ops.token_loss import distill_loss
    g = _gen(22)
    x = _logits((3, 1500), torch.float32, g)
    ids, values, lse = _teacher(x, 10, 1.0, g)
    hide = torch.ones_like(x, dtype=torch.bool).scatter_(1, ids, False)
    hide[:, ::2] = False
    _check_distill(x.masked_fill(hide, -math.inf), ids, values, None, 1.0)
    _check_distill(x.masked_fill(hide, -math.inf), ids, values, lse, 1.0)
    # a token of the teacher that the student cannot give: infinitely far
    x[0, ids[0, 0]] = -math.inf
    assert distill_loss(x, ids, values)[0] == math.inf


def test_distill_id_outside_of_the_vocabulary():
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import distill_loss
    x = torch.zeros(2, 50, device="cuda")
    cuda_ops.check_error_flag(x.device)
    loss = distill_loss(x, torch.tensor([[1, 50], [1, 2]], device="cuda"), torch.zeros(2, 2, device="cuda"))
    assert loss[0].isnan() and loss[1].isfinite()
    with pytest.raises(RuntimeError, match="61"):
        cuda_ops.check_error_flag(x.device)


def test_no_rows():
    from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs
    x = torch.zeros(0, 4, 100, device="cuda", requires_grad=True)
    t = torch.zeros(0, 4, dtype=torch.int64, device="cuda")
    r = token_logprobs(x, t, entropy=True, top=3)
    assert r.logprob.shape == (0, 4) and r.top_ids.shape == (0, 4, 3)
    dx, = torch.autograd.grad(r.logprob.sum() + distill_loss(x, r.top_ids, r.top_logprobs).sum(), (x,))
    assert dx.shape == x.shape


def test_captured_and_replayed_on_another_stream():
    from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs
    g = _gen(31)
    x = _logits((4, 1003), torch.float16, g).requires_grad_()
    t = torch.randint(0, 1003, (4,), generator=g, device="cuda")
    ids, values, lse = _teacher(x.detach(), 8, 1.0, g)

    def step():
        r = token_logprobs(x, t, entropy=True, top=4)
        loss = distill_loss(x, ids, values, teacher_logsumexp=lse)
        dx, = torch.autograd.grad(r.logprob.sum() + r.entropy.sum() + loss.sum(), (x,))
        return r.logprob.detach(), r.top_ids, loss.detach(), dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        x.copy_(_logits((4, 1003), torch.float16, g))
        t.copy_(torch.randint(0, 1003, (4,), generator=g, device="cuda"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(out, step()):
        assert torch.equal(got, want)


def test_offsets_past_32_bits():
    """2.2e9 logits and their gradients: the last rows."""
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import distill_loss, token_logprobs
    R, V = 17_000, 131_072
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(R, V, dtype=torch.bfloat16, device="cuda").normal_(std=2.5, generator=g).requires_grad_()
    t = torch.randint(0, V, (R,), generator=g, device="cuda")
    up = torch.randn(R, generator=g, device="cuda")
    r = token_logprobs(x, t, entropy=True, top=4)
    got, = torch.autograd.grad((r.logprob, r.entropy), (x,), (up, up))
    lp, ent, logp, dx = oracle.logprobs(x[-2:], t[-2:], 1.0, up[-2:], up[-2:])
    _near(r.logprob[-2:], lp, oracle.value_tol(V, lp, 1.0), "logprob")
    _near(r.entropy[-2:], ent, oracle.value_tol(V, ent, 1.0), "entropy")
    assert torch.equal(r.top_ids[-2:], torch.sort(x.detach()[-2:].float(), dim=-1, descending=True, stable=True).indices[:, :4])
    size = 2 * up[-2:].abs().double().cpu().unsqueeze(-1)
    _near(got[-2:], dx, oracle.grad_tol(dx, x.dtype, V, size, 1.0), "dlogits")
    del got
    ids = r.top_ids
    values = r.top_logprobs.detach()
    loss = distill_loss(x, ids, values)
    got, = torch.autograd.grad(loss, (x,), (up,))
    want, dx = oracle.distill(x[-2:], ids[-2:], values[-2:], 1.0, None, up[-2:])
    _near(loss[-2:], want, oracle.U * (4 * oracle.sum_steps(V) + 4 + 24 * (20 + math.log(V) + 20)), "loss")
    _near(got[-2:], dx, oracle.grad_tol(dx, x.dtype, V, up[-2:].abs().double().cpu().unsqueeze(-1) * 2, 1.0), "dlogits")
    cuda_ops.check_error_flag(x.device)
