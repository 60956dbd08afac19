"""AdamW over many tensors and the norm of all gradients on the CPU: the arithmetic that the GPU's kernels follow bit by bit."""
import math

import pytest
import torch

import adamw_oracle as oracle
from ipex_llm_b200.ops.adamw import AdamWState, adamw_state, adamw_step, flat_size, grad_norm, moments

KW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8)


def _tensors(sizes, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(dtype) for s in sizes]


def _step(params, grads, state, **kw):
    adamw_step(params, grads, state.exp_avg, state.exp_avg_sq, state.step, exp_avg_scale=state.exp_avg_scale,
               exp_avg_sq_scale=state.exp_avg_sq_scale, rest=state.rest, **{**KW, **kw})


def _near(got, want, tol, what):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


@pytest.mark.parametrize("decay,max_norm", [(0.0, 0.0), (0.1, 0.0), (0.01, 0.5), (0.0, 1e6)])
def test_steps_follow_the_definition(decay, max_norm):
    sizes = [(1,), (255,), (256,), (3, 171), (0,), (2, 5, 61)]
    params, state = _tensors(sizes), None
    state = adamw_state(params)
    m = [torch.zeros(s).double() for s in sizes]
    v = [torch.zeros(s).double() for s in sizes]
    for t in range(1, 5):
        grads = _tensors(sizes, seed=t, std=0.1 * t)
        norm = grad_norm(grads)
        assert abs(float(norm) - oracle.norm(grads)) <= float(norm) * 1.01 * oracle.U
        want = [oracle.step(p, g, a, b, t, KW["lr"], KW["betas"], KW["eps"], decay, float(norm) if max_norm else None, max_norm)
                for p, g, a, b in zip(params, grads, m, v)]
        _step(params, grads, state, weight_decay=decay, grad_norm=norm, max_grad_norm=max_norm)
        assert int(state.step) == t
        at = 0
        for i, (p, w) in enumerate(zip(params, want)):
            n = p.numel()
            m[i], v[i] = (x[at:at + n].view(p.shape).double() for x in (state.exp_avg, state.exp_avg_sq))
            for got, (value, tol) in zip((p, m[i], v[i]), w):
                _near(got, value, tol, (t, i))
            assert not state.exp_avg[at + n:at + flat_size([n])].any()
            at += flat_size([n])


def test_it_is_the_librarys_adamw():
    sizes = [(7, 33), (300,)]
    a, b = _tensors(sizes, torch.float32), [p.double().requires_grad_() for p in _tensors(sizes, torch.float32)]
    state, other = adamw_state(a), torch.optim.AdamW(b, lr=KW["lr"], betas=KW["betas"], eps=KW["eps"], weight_decay=0.1)
    for t in range(20):
        grads = _tensors(sizes, seed=t + 1)
        for p, g in zip(b, grads):
            p.grad = g.double()
        other.step()
        _step(a, grads, state, weight_decay=0.1)
    for p, q in zip(a, b):
        # 20 steps of some roundings each of numbers up to 4 and changes up to 20 lr
        assert (p.double() - q).abs().max() <= 20 * 20 * oracle.U * 4


@pytest.mark.parametrize("bits", [8, 32])
def test_bf16_and_its_rest_are_the_32_bit_parameters(bits):
    """As with a copy in 32 bits, and as parameters in 32 bits, whose gradients are bf16 numbers."""
    sizes = [(300,), (2, 129)]
    low = _tensors(sizes, torch.bfloat16)
    copied, wide = [p.clone() for p in low], [p.float() for p in low]
    states = [adamw_state(low, bits, "low"), adamw_state(copied, bits, "copy"), adamw_state(wide, bits)]
    for t in range(6):
        grads = _tensors(sizes, torch.bfloat16, seed=t + 1)
        for params, state in zip((low, copied, wide), states):
            _step(params, [g.to(params[0].dtype) for g in grads], state, lr=1e-5, weight_decay=0.1)
    assert (states[0].rest != 0).any()
    at = 0
    for p, q, w in zip(low, copied, wide):
        n = p.numel()
        bits32 = (p.view(torch.int16).long() << 16) + states[0].rest[at:at + n].view(p.shape).long()
        assert torch.equal(bits32 & 0xFFFFFFFF, w.view(torch.int32).long() & 0xFFFFFFFF)
        assert torch.equal(states[1].rest[at:at + n].view(p.shape), w)
        assert ((p.float() - w).abs() <= w.abs() * 2.0 ** -8).all() and torch.equal(q, w.to(torch.bfloat16))
        at += flat_size([n])
    for x, y, z in zip(*(s[:2] for s in states)):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and torch.equal(x.view(torch.uint8), z.view(torch.uint8))


def test_steps_below_a_16_bit_place_are_not_lost():
    p, q = [torch.ones(256, dtype=torch.bfloat16)], [torch.ones(256, dtype=torch.bfloat16)]
    kept, none = adamw_state(p, rest="low"), adamw_state(q)
    for _ in range(200):
        g = [torch.ones(256, dtype=torch.bfloat16)]
        _step(p, g, kept, lr=1e-4)
        _step(q, g, none, lr=1e-4)
    assert (q[0] == 1.0).all()                                    # 1e-4 is below half of 2^-8
    assert ((p[0].float() - 0.98).abs() <= 2.0 ** -8).all()


def _held(m, v, step=1, seed=0, params=None):
    """8-bit moments of given 32-bit ones, by a step that leaves them as they are but for the rounding."""
    n = m.numel()
    state = adamw_state([torch.zeros(n)], 8)
    from ipex_llm_b200.ops import adamw
    cm, em, cv, ev = adamw._to_small(m, v, *adamw._chances(0, flat_size([n]), step, seed))
    state.exp_avg.copy_(cm)
    state.exp_avg_sq.copy_(cv)
    state.exp_avg_scale.copy_(em)
    state.exp_avg_sq_scale.copy_(ev)
    return state


def test_8_bit_moments_are_neighbours_with_the_right_mean():
    g = torch.Generator().manual_seed(0)
    m = torch.randn(512, generator=g) * torch.exp2(torch.randint(-6, 1, (512,), generator=g))
    v = m.square() * torch.rand(512, generator=g)
    total = [torch.zeros(512, dtype=torch.float64) for _ in range(2)]
    rounds = 400
    for k in range(rounds):
        s = _held(m, v, step=k + 1)
        got = moments(*s[:2], s.exp_avg_scale, s.exp_avg_sq_scale)
        for i, (x, y, eps) in enumerate(((got[0], m, 2.0 ** -3), (got[1], v, 2.0 ** -2))):
            # one step of the format: eps of the value, or of the smallest normal number (2^-6, 2^-14) where the block's largest
            # lies at 2^7, 2^14
            floor = torch.exp2(torch.floor(torch.log2(y.abs().view(-1, 256).amax(1)))).repeat_interleave(256)
            one = torch.maximum(torch.exp2(torch.floor(torch.log2(y.abs()))), floor * 2.0 ** (-13 if i == 0 else -28)) * eps
            assert ((x - y).abs() < one * (1 + 1e-6)).all()
            total[i] += (x - y).double() / one
    for i, t in enumerate(total):
        # a mean of `rounds` numbers of at most a step's spread: five deviations of half a step / sqrt(rounds)
        keep = torch.ones(512, dtype=torch.bool) if i == 0 else v > 2.0 ** -25 * v.view(-1, 256).amax(1).repeat_interleave(256)
        assert (t[keep] / rounds).abs().max() <= 5 * 0.5 / math.sqrt(rounds)


def test_a_second_moment_is_never_held_as_nothing():
    v = torch.full((256,), 1e-30)
    v[7] = 1.0
    v[9] = 0.0
    s = _held(torch.zeros(256), v)
    got = moments(*s[:2], s.exp_avg_scale, s.exp_avg_sq_scale)[1]
    assert (got[v > 0] > 0).all() and got[9] == 0


@pytest.mark.parametrize("where", ["nan", "inf", "-inf"])
def test_what_is_not_finite_stays_in_its_place(where):
    p = _tensors([(300,)])
    state, clean = adamw_state(p, 8), adamw_state(p, 8)
    grads = _tensors([(300,)], seed=1)
    grads[0][0] = 0.0                                              # the largest elements are the others' in any case
    q = [p[0].clone()]
    bad = [grads[0].clone()]
    bad[0][0] = float(where)
    _step(p, bad, state)
    _step(q, grads, clean)
    assert p[0][0].isnan() and torch.equal(p[0][1:], q[0][1:])
    a, b = (moments(*s[:2], s.exp_avg_scale, s.exp_avg_sq_scale) for s in (state, clean))
    for x, y in zip(a, b):
        assert not x[0].isfinite() and torch.equal(x[1:], y[1:])


@pytest.mark.parametrize("each", [False, True])
def test_parameters_without_a_gradient_stay(each):
    sizes = [(300,), (5,), (256,)]
    p = _tensors(sizes)
    state, before = adamw_state(p, each=each), [x.clone() for x in p]
    _step(p, [None, *_tensors(sizes[1:], seed=1)], state)
    assert torch.equal(p[0], before[0]) and not state.exp_avg[:512].any() and not torch.equal(p[1], before[1])
    assert state.step.tolist() == ([0, 1, 1] if each else [1])
    _step(p, [None] * 3, state)
    assert state.step.tolist() == ([0, 1, 1] if each else [1])
    _step(p, _tensors(sizes, seed=2), state)
    assert state.step.tolist() == ([1, 2, 2] if each else [2])
    # of its first step by its own counter, m and v are g and g^2; by the common one, its second step's corrections apply:
    # 0.1 / (1 - 0.9^2) and 0.01 / (1 - 0.99^2) of them
    size = KW["lr"] if each else KW["lr"] * (0.1 / 0.19) / math.sqrt(0.01 / 0.0199)
    assert (((p[0] - before[0]).abs() - size).abs() < 1e-5).all()


def test_other_orders_of_memory():
    p, g = _tensors([(6, 50)])[0], _tensors([(6, 50)], seed=1)[0]
    q = p.t().contiguous().t()
    a, b = adamw_state([p]), adamw_state([q])
    for grad in (g, g.t().contiguous().t(), torch.stack([g, g], dim=-1)[..., 0]):
        _step([p], [grad], a)
        _step([q], [grad], b)
    assert torch.equal(p, q) and torch.equal(a.exp_avg[:300].view(6, 50), b.exp_avg[:300].view(50, 6).t())


def test_the_rate_as_a_tensor():
    p, q = _tensors([(9,)]), _tensors([(9,)])
    a, b = adamw_state(p), adamw_state(q)
    g = _tensors([(9,)], seed=1)
    _step(p, g, a, lr=torch.tensor(0.25))
    _step(q, g, b, lr=0.25)
    assert torch.equal(p[0], q[0])


def test_norm_of_what_32_bits_do_not_hold():
    assert float(grad_norm([torch.full((4,), 1e30)])) == pytest.approx(2e30, rel=1e-6)
    assert float(grad_norm([torch.full((4,), 1e-30), None])) == pytest.approx(2e-30, rel=1e-6)
    assert float(grad_norm([])) == float(grad_norm([None])) == 0.0
    assert grad_norm([torch.tensor([1.0, math.nan])]).isnan()


def test_old_graphs_notice_the_step():
    p = torch.ones(4, requires_grad=True)
    y = (p * p).sum()
    state = adamw_state([p])
    _step([p], [torch.ones(4)], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals():
    p, g = _tensors([(300,)]), _tensors([(300,)], seed=1)
    s = adamw_state(p)

    def refused(match, params=p, grads=g, state=s, **kw):
        before = [x.clone() for x in params]
        with pytest.raises(RuntimeError, match=match):
            _step(params, grads, state, **kw)
        assert all(torch.equal(x, y) for x, y in zip(params, before))

    refused("1 parameters and 2 gradients", grads=g + g)
    refused("like its parameter", grads=[g[0].double()])
    refused("like its parameter", grads=[g[0][:7]])
    refused("sparse", grads=[g[0].to_sparse()])
    refused("occurs twice", params=p + p, grads=g + g, state=adamw_state(p + p))
    refused("one type", params=[p[0], p[0].bfloat16()], grads=[None, None])
    refused("one behind the other", params=[torch.zeros(9, 2)[:, 0]], grads=[torch.zeros(9)], state=adamw_state([torch.zeros(9)]))
    refused("not supported", params=[p[0].double()], grads=[g[0].double()])
    refused("exp_avg should be", state=s._replace(exp_avg=s.exp_avg[:256]))
    refused("exp_avg_sq should be", state=s._replace(exp_avg_sq=s.exp_avg_sq.double()))
    refused("step should be", state=s._replace(step=s.step.int()))
    refused("step should be", state=s._replace(step=torch.zeros(2, dtype=torch.int64)))
    refused("come with their exponents", state=adamw_state(p, 8)._replace(exp_avg_scale=None))
    refused("uint8 of 2", state=adamw_state(p, 8)._replace(exp_avg_scale=torch.zeros(1, dtype=torch.uint8)))
    refused("have no rest", state=s._replace(rest=torch.zeros(512, dtype=torch.int16)))
    refused("max_grad_norm needs", max_grad_norm=1.0)
    refused("grad_norm should be one", max_grad_norm=1.0, grad_norm=torch.tensor(1.0, dtype=torch.float64))
    refused("should lie in", betas=(1.0, 0.9))
    refused("should lie in", lr=-1.0)
    refused("should lie in", eps=-1.0)
    refused("lr should be", lr=torch.tensor([1.0, 2.0]))
    for kw, match in ((dict(bits=4), "32 or 8"), (dict(rest="low"), "bf16"), (dict(rest="copy"), "16-bit"), (dict(rest="all"), "'copy'")):
        with pytest.raises(RuntimeError, match=match):
            adamw_state(p, **kw)
    with pytest.raises(RuntimeError, match="no parameters"):
        adamw_state([])
    with pytest.raises(RuntimeError, match="one type on one device"):
        grad_norm([g[0], g[0].bfloat16()])
    with pytest.raises(RuntimeError, match="sparse"):
        grad_norm([g[0].to_sparse()])
    with pytest.raises(RuntimeError, match="not supported"):
        grad_norm([torch.zeros(3, dtype=torch.int32)])
    adamw_step([], [], s.exp_avg, s.exp_avg_sq, s.step, lr=1.0)
    assert isinstance(s, AdamWState)
