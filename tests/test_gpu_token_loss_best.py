"""The best tokens of rows where a few threads hold nearly all large logits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

READERS = 224              # threads of a CTA that read a row
CANDIDATES = 1024          # more than these that reach the bound, and a slice is scanned once for each rank


def _row(dtype, V, threads):
    """Large numbers in the vectors of the first `threads` threads, all of them above all others."""
    vec = 4 if dtype == torch.float32 else 8
    at = torch.arange(V, device="cuda")
    of = at // vec % READERS < threads
    # few values (in bf16 from 5 to 7 in steps of 2^-5, so that many are equal): the lower index comes first
    return torch.where(of, 5.0 + (at * 7919 % 64) / 32.0, (at * 104729 % 64) / 32.0).to(dtype), of


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 200])
@pytest.mark.parametrize("threads,top", [(31, 32), (31, 1), (3, 32), (20, 24)])
def test_few_threads_hold_the_large_ones(dtype, rows, threads, top):
    from ipex_llm_b200.ops import cuda_ops
    from ipex_llm_b200.ops.token_loss import token_logprobs
    V = 400_000
    row, of = _row(dtype, V, threads)
    assert int(of.sum()) > 8 * CANDIDATES or threads == 3
    x = row.expand(rows, V).contiguous()
    x = torch.stack([x[i].roll(i * 8 * READERS) for i in range(rows)]) if rows > 1 else x
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    r = token_logprobs(x, t, top=top)
    cuda_ops.check_error_flag(x.device)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids, order)
    logp = torch.log_softmax(x.double(), -1).gather(-1, order)
    # a row's sum: below V / 512 + 200 roundings of 32 bits (thread, warp, CTA), logarithms of up to 20
    assert (r.top_logprobs.double() - logp).abs().max() <= (2 * (V / 512 + 200) + 8 * 20) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_of_a_slice_is_nan_or_infinite(dtype):
    """Keys of equal values in thousands: order by index alone."""
    from ipex_llm_b200.ops.token_loss import token_logprobs
    V = 100_000
    for value in (float("nan"), float("inf"), -float("inf")):
        for rows in (1, 150):
            x = torch.full((rows, V), value, dtype=dtype, device="cuda")
            r = token_logprobs(x, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=32)
            assert torch.equal(r.top_ids, torch.arange(32, device="cuda").expand(rows, 32))
