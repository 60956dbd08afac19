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
