"""The state of the optimizer over many tensors: what is pruned, saved and loaded, on the CPU."""
import pytest
import torch

from ipex_llm_b200.ops.adamw import flat_size, moments
from ipex_llm_b200.train import MultiTensorAdamW


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _params(sizes, dtype=torch.float32, seed=0):
    g = _gen(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.5).to(dtype)) for s in sizes]


def _set_grads(params, seed):
    g = _gen(seed)
    for p in params:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype)


def _real(bucket):
    """Both moments of the parameters' own elements, without what fills each up to 256."""
    s, out, at = bucket["state"], [], 0
    wide = moments(s.exp_avg, s.exp_avg_sq, s.exp_avg_scale, s.exp_avg_sq_scale)
    for p in bucket["params"]:
        out.append([x[at:at + p.numel()].clone() for x in wide])
        at += flat_size([p.numel()])
    return [torch.cat(x) for x in zip(*out)]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes", [[40] * 30, [231, 300, 1], [256, 512], [(3, 7), 0, 1000]], ids=str)
@pytest.mark.parametrize("ratio", [0.0, 0.1, 0.8, 1.0])
def test_pruned_moments_are_the_smallest_real_ones(bits, sizes, ratio):
    params = _params(sizes)
    opt = MultiTensorAdamW(params, lr=1e-3, bits=bits)
    for t in range(2):
        _set_grads(params, t)
        opt.step()
    (bucket,) = opt.buckets()
    before = _real(bucket)
    opt.prune_moments(ratio)
    for x, y in zip(before, _real(bucket)):
        k = int(ratio * x.numel())
        limit = x.abs().sort().values[k - 1] if k else -1.0
        assert torch.equal(y, torch.where(x.abs() > limit, x, 0.0))          # ties with the last one go, too
        if bits == 32:
            assert int((y != 0).sum()) == x.numel() - k


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_rate_on_the_device_stays_there(device, tmp_path):
    """Steps that are captured read the rate's tensor: loading a state writes into it."""
    params = [torch.nn.Parameter(p.detach().to(device)) for p in _params([300, 7])]
    rate = torch.tensor(0.25, device=device)
    opt = MultiTensorAdamW([{"params": params[:1]}, {"params": params[1:], "lr": 0.125}], lr=rate)
    _set = lambda t: [setattr(p, "grad", torch.full_like(p, float(t))) for p in params]      # noqa: E731
    _set(1)
    opt.step()
    torch.save(opt.state_dict(), tmp_path / "o.pt")
    saved = torch.load(tmp_path / "o.pt", map_location="cpu", weights_only=False)
    rate.fill_(9.0)
    opt.param_groups[1]["lr"] = 9.0
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is rate and float(rate) == 0.25 and opt.param_groups[1]["lr"] == 0.125
    assert rate.device.type == device
    opt.step()                                                    # takes the rate where it is
    # a rate that was saved from a tensor, for an optimizer with a number, and the other way round
    other = MultiTensorAdamW([{"params": params[:1]}, {"params": params[1:], "lr": torch.tensor(3.0, device=device)}], lr=1.0)
    other.load_state_dict(saved)
    assert other.param_groups[0]["lr"] == 0.25 and isinstance(other.param_groups[0]["lr"], float)
    assert float(other.param_groups[1]["lr"]) == 0.125 and other.param_groups[1]["lr"].device.type == device
    other.step()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_that_was_taken_does_not_move(bits):
    """Of parameters on the CPU, too, and a rate in a tensor with it: an earlier state can be gone back to."""
    params, rate = _params([300, 7], torch.bfloat16), torch.tensor(0.25)
    opt = MultiTensorAdamW(params, lr=rate, bits=bits)
    _set_grads(params, 0)
    opt.step()
    held = [p.detach().clone() for p in params]
    taken = opt.state_dict()

    def go_on():
        out = []
        for t in range(1, 3):
            _set_grads(params, t)
            opt.step()
            out += [p.detach().clone() for p in params]
            rate.mul_(0.5)
        return out
    first = go_on()
    with torch.no_grad():
        for p, q in zip(params, held):
            p.copy_(q)
    opt.load_state_dict(taken)
    assert float(rate) == 0.25
    assert all(torch.equal(p, q) for p, q in zip(first, go_on()))


def test_a_resumed_state_rounds_as_the_saved_one():
    """8-bit moments are rounded by a hash of the seed: it comes with the state."""
    a, b = _params([300, 7]), _params([300, 7])
    one, other = MultiTensorAdamW(a, lr=1e-2, bits=8, seed=3), MultiTensorAdamW(b, lr=1e-2, bits=8, seed=4)
    _set_grads(a, 0)
    one.step()
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    other.load_state_dict(one.state_dict())
    assert other.seed == 3
    for t in range(1, 4):
        _set_grads(a, t)
        _set_grads(b, t)
        one.step()
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    older = one.state_dict()
    del older["seed"]                                             # as states were saved before
    other.load_state_dict(older)
    assert other.seed == 3


def test_a_state_of_other_parameters_is_refused():
    """Also where all of them take as much room, or fall into as many buckets."""
    def of(*groups):
        params = [_params(sizes, dtype) for sizes, dtype in groups]
        opt = MultiTensorAdamW([{"params": p} for p in params], lr=1e-3)
        _set_grads([p for g in params for p in g], 1)
        opt.step()
        return opt
    f32, bf16 = torch.float32, torch.bfloat16
    saved = of(([300, 7], f32))
    for other in (of(([7, 300], f32)), of(([(2, 300), 7], f32)), of(([301, 7], f32))):
        before = [p.detach().clone() for p in other.param_groups[0]["params"]]
        kept = [t.clone() for t in other.buckets()[0]["state"] if t is not None]
        with pytest.raises(RuntimeError, match="other parameters"):
            other.load_state_dict(saved.state_dict())
        assert all(torch.equal(a, b) for a, b in zip(before, other.param_groups[0]["params"]))
        assert all(torch.equal(a, b) for a, b in zip(kept, (t for t in other.buckets()[0]["state"] if t is not None)))
    two = of(([300], f32), ([300], bf16))
    both = MultiTensorAdamW([*_params([300], f32), *_params([300], bf16)], lr=1e-3)
    with pytest.raises(RuntimeError, match="other parameters"):
        both.load_state_dict(two.state_dict())
    older = saved.state_dict()
    del older["sizes"]                                            # as states were saved before
    of(([300, 7], f32)).load_state_dict(older)
