"""AdamW over many tensors and the norm of all gradients on the GPU, against the definition in 64 bits and, bit by bit, against the
same arithmetic on the CPU."""
import math

import pytest
import torch

import adamw_oracle as oracle
from ipex_llm_b200.ops import adamw

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
KW = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
RAGGED = [(1,), (7,), (255,), (256,), (257,), (0,), (33, 61), (2048,), (2049,), (5000,), (3, 5, 700)]


def _tensors(sizes, dtype, seed=0, std=1.0, offset=0):
    """On the GPU; ``offset``: elements from a 16-byte boundary."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for s in sizes:
        x = (torch.randn(s, generator=g) * std).to(dtype)
        room = torch.empty(x.numel() + offset, dtype=dtype, device="cuda")[offset:]
        out.append(room.view(s).copy_(x))
    return out


def _step(params, grads, state, **kw):
    adamw.adamw_step(params, grads, state.exp_avg, state.exp_avg_sq, state.step, exp_avg_scale=state.exp_avg_scale,
                     exp_avg_sq_scale=state.exp_avg_sq_scale, rest=state.rest, **{**KW, **kw})


def _cpu(x):
    return type(x)(*(_cpu(y) for y in x)) if isinstance(x, tuple) else [_cpu(y) for y in x] if isinstance(x, list) else \
        None if x is None else x.detach().cpu().clone()


def _bits(x):
    """Compared as bits, NaN by its place alone."""
    if not x.is_floating_point():
        return x.cpu()
    x = x.cpu()
    one = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[x.element_size()]
    nan = x.float().isnan()
    return torch.where(nan, torch.full((), -1 if one != torch.uint8 else 127, dtype=one), x.view(one)), nan


def _same(got, want, what):
    if got is None and want is None:
        return
    a, b = _bits(got), _bits(want)
    for x, y in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
        assert torch.equal(x, y), (what, int((x != y).sum()), x.numel())


def _rest_of(dtype):
    return {torch.bfloat16: [None, "low", "copy"], torch.float16: [None, "copy"], torch.float32: [None]}[dtype]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,rest", [(d, r) for d in DTYPES for r in _rest_of(d)])
def test_steps_are_those_of_the_cpu(dtype, rest, bits, offset):
    params = _tensors(RAGGED, dtype, offset=offset)
    state = adamw.adamw_state(params, bits, rest)
    here, kept = _cpu(params), _cpu(state)
    for t in range(4):
        grads = _tensors(RAGGED, dtype, seed=t + 1, std=0.1 ** t, offset=offset)
        norm = adamw.grad_norm(grads)
        assert abs(float(norm) - oracle.norm(grads)) <= oracle.norm_tol(oracle.norm(grads))
        max_norm = 0.0 if t == 0 else 1.0
        _step(params, grads, state, grad_norm=norm, max_grad_norm=max_norm, seed=5)
        _step(here, _cpu(grads), kept, grad_norm=norm.cpu(), max_grad_norm=max_norm, seed=5)
        for i, (p, q) in enumerate(zip(params, here)):
            _same(p, q, (t, i))
        for name, a, b in zip(state._fields, state, kept):
            _same(a, b, (t, name))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [0, 1, 999])
def test_a_step_by_its_definition(dtype, t):
    sizes = [(3, 1031), (40000,)]
    params, grads = _tensors(sizes, dtype), _tensors(sizes, dtype, seed=1, std=0.01)
    state = adamw.adamw_state(params)
    state.step.fill_(t)
    g = torch.Generator(device="cuda").manual_seed(3)
    state.exp_avg.copy_(torch.randn(state.exp_avg.shape, generator=g, device="cuda") * 0.01)
    state.exp_avg_sq.copy_(torch.rand(state.exp_avg.shape, generator=g, device="cuda") * 1e-4)
    at, want = 0, []
    for p, d in zip(params, grads):
        m, v = (x[at:at + p.numel()].view(p.shape) for x in (state.exp_avg, state.exp_avg_sq))
        want.append(oracle.step(p, d, m, v, t + 1, KW["lr"], KW["betas"], KW["eps"], KW["weight_decay"]))
        at += adamw.flat_size([p.numel()])
    _step(params, grads, state)
    at = 0
    for p, ((wp, tp), (wm, tm), (wv, tv)) in zip(params, want):
        m, v = (x[at:at + p.numel()].view(p.shape) for x in (state.exp_avg, state.exp_avg_sq))
        for got, value, tol in ((p, wp, oracle.with_rounding(tp, wp, dtype)), (m, wm, tm), (v, wv, tv)):
            assert ((got.double().cpu() - value).abs() <= tol).all()
        at += adamw.flat_size([p.numel()])


@pytest.mark.parametrize("count", [31, 32, 33, 640, 641, 1500])
@pytest.mark.parametrize("each", [False, True])
def test_many_tensors(count, each):
    """More tensors than a launch takes, some without a gradient."""
    sizes = [(1 + (37 * i) % 700,) for i in range(count)]
    params, grads = _tensors(sizes, torch.bfloat16), _tensors(sizes, torch.bfloat16, seed=1)
    grads = [None if i % 7 == 3 or i == 0 else g for i, g in enumerate(grads)]
    state = adamw.adamw_state(params, 8, "low", each=each)
    here, kept = _cpu(params), _cpu(state)
    for _ in range(2):
        _step(params, grads, state)
        _step(here, _cpu(grads), kept)
    assert torch.equal(torch.cat(_cpu(params)).view(torch.int16), torch.cat(here).view(torch.int16))
    for name, a, b in zip(state._fields, state, kept):
        _same(a, b, name)
    norm = adamw.grad_norm(grads)
    assert abs(float(norm) - oracle.norm(grads)) <= oracle.norm_tol(oracle.norm(grads))
    assert torch.equal(norm, adamw.grad_norm(grads))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite(bits, value):
    params, grads = _tensors([(600,)], torch.bfloat16), _tensors([(600,)], torch.bfloat16, seed=1)
    grads[0][3] = value
    state = adamw.adamw_state(params, bits, "low")
    here, kept = _cpu(params), _cpu(state)
    for _ in range(2):
        _step(params, grads, state)
        _step(here, _cpu(grads), kept)
    _same(params[0], here[0], "parameters")
    assert params[0].isnan().sum() == 1
    for name, a, b in zip(state._fields, state, kept):
        _same(a, b, name)
    norm = adamw.grad_norm(grads)
    assert (norm.isnan() if math.isnan(value) else norm == math.inf)


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e30), (torch.bfloat16, 1e30), (torch.float32, 1e-30), (torch.bfloat16, 1e-30),
                                        (torch.float16, 60000.0), (torch.float16, 6e-8)])
def test_norms_of_what_32_bits_do_not_hold(dtype, size):
    grads = [torch.full((n,), size, dtype=dtype, device="cuda") for n in (1, 7, 5000)]
    norm = adamw.grad_norm(grads)
    assert abs(float(norm) - oracle.norm(grads)) <= oracle.norm_tol(oracle.norm(grads))


def test_norm_of_views():
    x = torch.randn(40, 50, device="cuda")
    grads = [x[:, 3], x[1:7, 5:9], x.t(), x[0].expand(3, 50)]
    norm = adamw.grad_norm(grads)
    assert abs(float(norm) - oracle.norm(grads)) <= oracle.norm_tol(oracle.norm(grads))
    assert float(adamw.grad_norm([x[:0], None])) == 0.0 and float(adamw.grad_norm([None])) == 0.0


@pytest.mark.parametrize("eps,exponents", [(1e-8, (-149, 60)), (1e-8, (-149, 127)), (2.0 ** -38, (-149, 60)), (1e-12, (-149, 100)),
                                           (0.0, (-100, 60)), (1.0, (-20, 20))])
def test_roots_and_quotients_are_the_nearest_numbers(eps, exponents):
    """Moments of every size, none, and not finite: what the kernel takes for roots and divisions against the library's, bit by bit.
    Gradients of 0 and betas of a half leave half of each moment; parameters of 0 show the change."""
    n = 1 << 22
    g = torch.Generator(device="cuda").manual_seed(int(eps * 1e9) + exponents[1])
    size = lambda lo, hi: torch.exp2(torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo)      # noqa: E731
    v = size(*exponents)
    m = size(-60, min(exponents[1], 58)) * torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v[:1000], m[500:1500] = 0.0, 0.0
    if exponents[1] > 100:
        v[2000], v[3000], m[4000], m[5000] = math.inf, math.nan, math.inf, math.nan
    p, zero = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    state = adamw.adamw_state([p])
    state.exp_avg.copy_(m)
    state.exp_avg_sq.copy_(v)
    state.step.fill_(2)
    _step([p], [zero], state, betas=(0.5, 0.5), eps=eps, weight_decay=0.0)
    rate = torch.tensor(KW["lr"] / (1 - 0.5 ** 3), dtype=torch.float64).float().cuda()
    root = torch.tensor(1 / math.sqrt(1 - 0.5 ** 3), dtype=torch.float64).float().cuda()
    m1, v1 = m * 0.5, v * 0.5
    want = zero - (m1 * rate) / (v1.sqrt() * root + eps)
    _same(p, want, "change")
    _same(state.exp_avg, m1, "m")
    _same(state.exp_avg_sq, v1, "v")


def test_captured_steps_count_on():
    """Replays take the step counter, the rate and the gradients as they are then; two graphs of the same parameters, and an eager
    step between them, share nothing but the state."""
    params = _tensors(RAGGED, torch.bfloat16)
    state, lr = adamw.adamw_state(params, 8, "low"), torch.tensor(1e-2, device="cuda")
    grads = _tensors(RAGGED, torch.bfloat16, seed=1)
    here, kept = _cpu(params), _cpu(state)

    def go():
        _step(params, grads, state, lr=lr, grad_norm=adamw.grad_norm(grads), max_grad_norm=1.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go()
        graphs.append(graph)
    rates = [1e-2]
    for k in range(4):
        lr.fill_(1e-2 * (k + 2))
        for i, g in enumerate(grads):
            g.copy_(_tensors([RAGGED[i]], torch.bfloat16, seed=10 * k + i)[0])
        rates.append(float(lr))
        graphs[k % 2].replay() if k != 2 else go()
    torch.cuda.synchronize()
    seen = [_tensors(RAGGED, torch.bfloat16, seed=1)] + [[_tensors([RAGGED[i]], torch.bfloat16, seed=10 * k + i)[0]
                                                          for i in range(len(RAGGED))] for k in range(4)]
    for rate, g in zip(rates, seen):
        _step(here, _cpu(g), kept, lr=torch.tensor(rate), grad_norm=adamw.grad_norm(g).cpu(), max_grad_norm=1.0)
    assert int(state.step) == 5
    for p, q in zip(params, here):
        _same(p, q, "parameters")
    for name, a, b in zip(state._fields, state, kept):
        _same(a, b, name)


def test_streams_and_neighbours():
    """On another stream; what lies around the parameters, and other parts of the same storage, stay as they were."""
    room = torch.full((3000,), 7.0, device="cuda")
    params, grads = [room[5:1006], room[1500:1756]], [torch.ones(1001, device="cuda"), torch.ones(256, device="cuda")]
    state = adamw.adamw_state(params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            _step(params, grads, state)
    torch.cuda.current_stream().wait_stream(side)
    changed = room != 7.0
    assert changed.sum() == 1257 and changed[5:1006].all() and changed[1500:1756].all()


def test_places_past_32_bits_of_bytes():
    """Moments that begin past 2^32 bytes, and an element count whose bytes pass 2^32."""
    big = (1 << 30) + 300
    params = [torch.zeros(big, dtype=torch.bfloat16, device="cuda"), torch.ones(700, dtype=torch.bfloat16, device="cuda")]
    grads = [torch.zeros(big, dtype=torch.bfloat16, device="cuda"), torch.full((700,), 0.5, dtype=torch.bfloat16, device="cuda")]
    grads[0][-1] = 1.0
    state = adamw.adamw_state(params)
    _step(params, grads, state, weight_decay=0.0)
    at = adamw.flat_size([big])
    assert float(state.exp_avg[big - 1]) == pytest.approx(0.1, rel=1e-6) and (state.exp_avg[at:at + 700] == state.exp_avg[at]).all()
    assert float(state.exp_avg[at]) == pytest.approx(0.05, rel=1e-6) and int((state.exp_avg != 0).sum()) == 701
    assert int((params[0] != 0).sum()) == 1 and float(params[0][-1]) < 0
    assert float(adamw.grad_norm(grads)) == pytest.approx(math.sqrt(1 + 700 * 0.25), rel=1e-6)


def test_refusals_leave_everything():
    p, g = _tensors([(300,)], torch.float32), _tensors([(300,)], torch.float32, seed=1)
    state, before = adamw.adamw_state(p), p[0].clone()
    for kw, match in ((dict(grads=[g[0].cpu()]), "like its parameter"), (dict(state=_cpu(state)), "exp_avg should be"),
                      (dict(state=state._replace(step=state.step.cpu())), "step should be"),
                      (dict(max_grad_norm=1.0, grad_norm=torch.tensor(1.0)), "grad_norm should be one"),
                      (dict(lr=torch.tensor(0.1)), "lr should be"),
                      (dict(state=state._replace(exp_avg=torch.zeros(513, device="cuda")[1:])), "exp_avg should be")):
        kw = dict(dict(params=p, grads=g, state=state), **kw)
        with pytest.raises(RuntimeError, match=match):
            _step(**kw)
    assert torch.equal(p[0], before) and int(state.step) == 0
