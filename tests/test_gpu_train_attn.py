"""Attention with a gradient on the GPU, against its definition in 64 bits."""
import math

import pytest
import torch

import train_attn_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _inputs(B, Hq, Hkv, Sq, Skv, D, dtype, seed, grad_std=1.0 / 16):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def heads(n, s, std):
        return (torch.randn(B, s, n, D, generator=g, device="cuda") * std).to(dtype).transpose(1, 2)
    return heads(Hq, Sq, 1.5), heads(Hkv, Skv, 1.0), heads(Hkv, Skv, 1.0), heads(Hq, Sq, grad_std)


def _run(q, k, v, g, **kw):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.train_attn import attention
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, **kw)
    grads = torch.autograd.grad(out, (q, k, v), g)
    cuda_ops.check_error_flag(q.device)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)))


def _check(q, k, v, g, scale=None, causal=True, window=0, key_mask=None):
    got = _run(q, k, v, g, scale=scale, causal=causal, window=window, key_mask=key_mask)
    want = oracle.attention(q, k, v, g, scale or q.shape[-1] ** -0.5, causal, window, key_mask)
    for name, (exact, tol) in want.items():
        t = got[name]
        assert t.shape == exact.shape and t.dtype == q.dtype, name
        off = ((t.double() - exact).abs() / tol).nan_to_num(nan=math.inf)
        assert float(off.max()) <= 1.0, (name, float(off.max()), (off > 1).sum().item(), off.argmax().item())
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [128, 1, 2, 63, 127, 129, 200, 256, 257, 384, 700])
def test_causal_by_length(dtype, D, S):
    _check(*_inputs(2, 4, 2, S, S, D, dtype, S + D))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [8, 24, 32, 72, 80, 96, 112, 120])
def test_head_sizes(dtype, D):
    _check(*_inputs(1, 3, 3, 150, 150, D, dtype, D))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 1), (6, 2), (5, 5), (32, 4)])
def test_shared_key_heads(Hq, Hkv):
    _check(*_inputs(2, Hq, Hkv, 300, 300, 64, torch.bfloat16, Hq))


@pytest.mark.parametrize("Sq,Skv", [(1, 1000), (77, 1101), (128, 129), (300, 128), (200, 1), (130, 70), (513, 1024)])
@pytest.mark.parametrize("causal", [True, False])
def test_queries_and_keys_of_different_lengths(Sq, Skv, causal):
    _check(*_inputs(2, 4, 2, Sq, Skv, 128, torch.bfloat16, Sq), causal=causal)


@pytest.mark.parametrize("window", [1, 2, 64, 128, 129, 200, 1000])
@pytest.mark.parametrize("Sq,Skv", [(515, 515), (130, 600)])
def test_windows(window, Sq, Skv):
    _check(*_inputs(1, 4, 2, Sq, Skv, 64, torch.float16, window), window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("side", ["right", "left", "holes", "one sequence"])
def test_padded_batches(dtype, causal, side):
    q, k, v, g = _inputs(3, 4, 2, 333, 333, 80, dtype, 7)
    at = torch.arange(333, device="cuda").view(1, -1)
    real = torch.tensor([[200], [333], [1]], device="cuda")
    mask = {"right": at < real, "left": at >= 333 - real, "holes": (at * 7919 + real) % 5 < 3,
            "one sequence": (at >= 0) & (real > 1)}[side]
    # what hidden rows hold takes no part
    k.transpose(1, 2)[~mask] = math.nan
    v.transpose(1, 2)[~mask] = math.inf
    got = _check(q, k, v, g, causal=causal, key_mask=mask)
    hidden = ~mask
    assert bool((got["dk"].transpose(1, 2)[hidden] == 0).all()) and bool((got["dv"].transpose(1, 2)[hidden] == 0).all())
    other = _run(q, k, v, g, causal=causal, key_mask=mask.to(torch.int64))          # a tokenizer's mask
    assert all(torch.equal(got[n], other[n]) for n in got)


def test_padding_and_window():
    q, k, v, g = _inputs(2, 4, 4, 400, 400, 64, torch.bfloat16, 8)
    at = torch.arange(400, device="cuda").view(1, -1)
    _check(q, k, v, g, window=100, key_mask=at < torch.tensor([[150], [399]], device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grad_std", [1e-6, 1.0, 200.0])
def test_small_and_large_gradients(dtype, grad_std):
    """fp16 would lose dS to subnormals or past its largest number if it were stored as it is."""
    _check(*_inputs(1, 2, 2, 600, 600, 128, dtype, 5, grad_std))


def test_peaked_scores():
    """Scores far apart: references move in many blocks, most probabilities vanish."""
    q, k, v, g = _inputs(1, 2, 1, 700, 700, 64, torch.float16, 6)
    _check(q * 8, k * torch.linspace(0.1, 8, 700, device="cuda").half().view(1, 1, -1, 1), v, g)
    _check(q, k, v, g, scale=3.0)
    _check(q, k, v, g, scale=1e-4)
    _check(q, k, v, g, scale=100.0)


def test_layouts():
    B, H, S, D = 2, 4, 260, 64
    g0 = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(B, S, 3 * H, D, generator=g0, device="cuda").bfloat16()
    q, k, v = (qkv[:, :, i * H:(i + 1) * H].transpose(1, 2) for i in range(3))
    g = torch.randn(B, H, S, D, generator=g0, device="cuda").bfloat16()                  # head-major
    want = _check(q, k, v, g)
    wide = torch.randn(B, H, S, D + 3, generator=g0, device="cuda").bfloat16()
    for name, f in {"head-major": lambda t: t.contiguous(),
                    "tokens first": lambda t: t.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3),
                    "rows apart": lambda t: wide.clone()[..., 1:D + 1].copy_(t),
                    "columns first": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)}.items():
        got = _run(f(q), f(k), f(v), f(g))
        assert all(torch.equal(got[n], want[n]) for n in got), name
    one = _run(q, k[:, :1].expand(-1, H, -1, -1), v[:, :1].expand(-1, H, -1, -1), g[:1, :1, :1, :1].expand(B, H, S, D))
    two = _run(q, k[:, :1], v[:, :1], g[:1, :1, :1, :1].expand(B, H, S, D).contiguous())
    # expanded heads get a gradient each, shared ones their sum: of four rounded numbers and rounded once more
    assert torch.equal(one["out"], two["out"]) and torch.equal(one["dq"], two["dq"])
    for n in ("dk", "dv"):
        total, size = one[n].double().sum(1, keepdim=True), one[n].double().abs().sum(1, keepdim=True)
        assert bool(((total - two[n].double()).abs() <= 2.0 ** -7 * size + 1e-30).all())


def test_the_same_every_time_and_from_a_graph():
    from ipex_llm_b200.ops.train_attn import attention
    q, k, v, g = _inputs(2, 8, 2, 600, 600, 128, torch.float16, 9)
    at = torch.arange(600, device="cuda").view(1, -1)
    mask = at < torch.tensor([[600], [411]], device="cuda")
    first = _run(q, k, v, g, key_mask=mask)
    for _ in range(3):
        again = _run(q, k, v, g, key_mask=mask)
        assert all(torch.equal(first[n], again[n]) for n in first)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = attention(*leaves, key_mask=mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.synchronize()
    for t in got:
        t.fill_(7.0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, first.values()))


def test_two_at_once():
    """Two streams, each with calls of its own: workspaces are not shared."""
    a, b = _inputs(2, 8, 8, 512, 512, 64, torch.bfloat16, 1), _inputs(1, 4, 1, 900, 900, 128, torch.float16, 2)
    want = [_run(*a), _run(*b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(4):
        for i, (s, case) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i] = _run(*case)
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(x[n], y[n]) for n in x)


def test_empty_and_without_gradient():
    from ipex_llm_b200.ops.train_attn import attention
    q, k, v, g = _inputs(1, 2, 2, 40, 40, 64, torch.bfloat16, 1)
    with torch.no_grad():
        out = attention(q, k, v)
    assert torch.equal(out, _run(q, k, v, g)["out"]) and out.transpose(1, 2).is_contiguous()
    got = _run(q, k[:, :, :0], v[:, :, :0], g, causal=False)
    assert bool((got["out"] == 0).all()) and bool((got["dq"] == 0).all()) and got["dk"].shape == (1, 2, 0, 64)
    got = _run(q[:, :, :0], k, v, g[:, :, :0])
    assert got["out"].numel() == 0 and bool((got["dk"] == 0).all())
    # only some of the inputs learn
    leaf = k.detach().requires_grad_()
    dk, = torch.autograd.grad(attention(q, leaf, v), (leaf,), g)
    assert torch.equal(dk, _run(q, k, v, g)["dk"])


def test_what_the_gpu_refuses():
    from ipex_llm_b200.ops.train_attn import attention
    q, k, v, _ = _inputs(1, 2, 2, 8, 8, 64, torch.bfloat16, 1)
    for bad in (lambda: attention(q.float(), k.float(), v.float()), lambda: attention(q, k.half(), v),
                lambda: attention(q[..., :60], k[..., :60], v[..., :60]), lambda: attention(q, k.cpu(), v),
                lambda: attention(*(torch.cat([t] * 3, -1) for t in (q, k, v))),
                lambda: attention(q, k, v, key_mask=torch.ones(1, 8, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            bad()


def test_long_sequences():
    q, k, v, g = _inputs(1, 2, 1, 4000, 4100, 128, torch.bfloat16, 11)
    _check(q, k, v, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes,kw", [((4, 8, 4, 17, 17, 64), {}), ((4, 8, 4, 5, 5, 128), {}), ((2, 6, 2, 200, 200, 128), {}),
                                      ((4, 8, 8, 40, 33, 64), dict(causal=False)), ((2, 8, 2, 300, 300, 72), dict(window=9)),
                                      ((3, 4, 4, 400, 400, 64), dict(real=(31, 20, 9)))])
def test_few_keys_are_rounded_once(dtype, sizes, kw):
    """Rows of few keys have the largest gradients: what their probabilities' rounding takes is kept.  Rounding x = m 2^e, m in
    [1, 2), errs by a number spread evenly over half a unit to either side, so the squares of the errors come to h^2 / 3 of the sum
    of 4^e, h half a step: with m^2 = 2.2 on average 0.39 h of the norm, 0.43 h as far as m leans to small values, and some 2 %
    either way with the thousands of numbers here.  A second rounding of that size makes 0.6 h of it."""
    kw = dict(kw)
    q, k, v, g = _inputs(*sizes, dtype, 21)
    real = kw.pop("real", None)
    if real is not None:                          # padded on the left
        at = torch.arange(sizes[4], device="cuda").view(1, -1)
        kw["key_mask"] = at >= sizes[4] - torch.tensor(real, device="cuda").view(-1, 1)
    got = _run(q, k, v, g, **kw)
    want = oracle.attention(q, k, v, g, sizes[-1] ** -0.5, kw.get("causal", True), kw.get("window", 0), kw.get("key_mask"))
    for n in ("out", "dq", "dk", "dv"):
        ref = want[n][0]
        assert (got[n].double() - ref).norm() <= 0.5 * torch.finfo(dtype).eps / 2 * ref.norm(), n


def test_more_heads_than_a_launch_takes():
    from ipex_llm_b200.ops.train_attn import attention
    q = torch.zeros(1, 32768, 1, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="heads"):
        attention(q, q, q)


def test_offsets_past_32_bits():
    """2.4e9 numbers in q, out and their gradients: the last rows of all heads, whose windows lie among the last rows."""
    S, H, D, n = 300_000, 64, 128, 100
    g = torch.Generator(device="cuda").manual_seed(5)
    q, grad = (torch.empty(1, S, H, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g).transpose(1, 2) for _ in range(2))
    k, v = (torch.empty(1, S, 1, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g).transpose(1, 2) for _ in range(2))
    got = _run(q, k, v, grad, window=64)
    tail = slice(S - n - 136, S)
    want = oracle.attention(*(t[:, :, tail] for t in (q, k, v, grad)), D ** -0.5, True, 64, None)
    for name, (exact, tol) in want.items():
        off = (got[name][:, :, -n:].double() - exact[:, :, -n:]).abs() / tol[:, :, -n:]
        assert float(off.nan_to_num(nan=math.inf).max()) <= 1.0, name


@pytest.mark.parametrize("Sq,Skv,window", [(100, 1500, 30), (1500, 300, 0), (900, 700, 200)])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_that_nothing_sees(Sq, Skv, window, D):
    """Between tiles with work: blocks of keys before all windows, and blocks of queries before the first key."""
    q, k, v, g = _inputs(3, 16, 8, Sq, Skv, D, torch.bfloat16, 17)
    got = _check(q, k, v, g, window=window)
    if Sq < Skv:
        assert not got["dk"][:, :, : Skv - Sq - window].any() and not got["dv"][:, :, : Skv - Sq - window].any()
    else:
        assert not got["out"][:, :, : Sq - Skv].any() and not got["dq"][:, :, : Sq - Skv].any()
