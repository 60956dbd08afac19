"""Trainer worker (gloo, CPU): the names of optimizers over many tensors train on several ranks as ``fused_lora_adamw`` does."""
import os
import sys
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

import torch
import torch.distributed as dist


class Tiny(torch.nn.Module):
    def __init__(self):
        super().__init__()
        torch.manual_seed(0)
        self.table, self.out = torch.nn.Embedding(31, 16), torch.nn.Linear(16, 31)

    def forward(self, input_ids, labels=None):
        return (self.out(self.table(input_ids)),)


def main():
    rank = int(os.environ["RANK"])
    dist.init_process_group("gloo")
    from ipex_llm_b200.train import FusedLoraAdamW, Trainer
    from ipex_llm_b200.transformers.qlora import TrainingArguments
    data = [{"input_ids": torch.randint(0, 31, (5 + i % 3,), generator=torch.Generator().manual_seed(i)).tolist()} for i in range(12)]
    got = {}
    for optim in ("fused_lora_adamw", "adamw_8bit", "adamw_multi"):
        args = TrainingArguments(output_dir=os.path.join(tempfile.gettempdir(), f"t{rank}"), per_device_train_batch_size=2, max_steps=3,
                                 logging_steps=1, bf16=False, fused_loss=True, learning_rate=1e-2, optim=optim)
        model = Tiny()
        trainer = Trainer(model, args, train_dataset=data)
        trainer.train()
        assert isinstance(trainer.optimizer, FusedLoraAdamW), optim
        got[optim] = torch.cat([p.detach().flatten() for p in model.parameters()])
        assert torch.equal(got[optim], got["fused_lora_adamw"]), optim
        lo, hi = got[optim].clone(), got[optim].clone()
        dist.all_reduce(lo, op=dist.ReduceOp.MIN)
        dist.all_reduce(hi, op=dist.ReduceOp.MAX)
        assert torch.equal(lo, hi), "ranks diverged"
    dist.barrier()
    dist.destroy_process_group()
    print(f"rank {rank}: ok")


if __name__ == "__main__":
    main()
