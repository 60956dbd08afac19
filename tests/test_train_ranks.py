"""Finetuning on several ranks by the trainer."""
from test_dist import run_workers


def test_optimizers_by_name_on_two_ranks():
    """One process has its own optimizers over many tensors; ranks average gradients and share the optimizer's state."""
    res = run_workers("trainer_worker.py", 2, [])
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-3000:]
    assert res.stdout.count(": ok") == 2
