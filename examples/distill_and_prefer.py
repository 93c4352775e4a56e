"""Distillation and preference training of an engram, end to end on a small random base:

  1. a teacher (the base with an engram whose output projection is not zero) records the top logits of
     some packed batches (top_logits: ids, values, log-sum-exp);
  2. the same base with a fresh engram learns them (distillation with the rest of the vocabulary as one
     class), starting exactly at the base;
  3. the base without an engram records its log-probabilities of chosen / rejected answers, and the engram is
     trained to prefer the chosen ones (paired log ratios).

    python examples/distill_and_prefer.py [--steps 30] [--seq 512]

Runs on one B200 (the sm_100a kernels) or, slowly, on a CPU (the plain forms). Prints one JSON line.
"""
import argparse
import json
import os
import sys
import tempfile

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def make_trainer(folder, seq, vocab):
    from micro_engram.train.config import load_config
    from micro_engram.train.data import Samples
    from micro_engram.train.loop import Trainer
    from micro_engram_fork_b200.models.gemma import tiny_config

    base = os.path.join(folder, "base")
    os.makedirs(base, exist_ok=True)
    with open(os.path.join(base, "config.json"), "w") as f:
        json.dump({**tiny_config(vocab_size=vocab).to_dict(), "model_type": "gemma4_text"}, f)
    trainer = Trainer(load_config({
        "base_model": base, "base_init": "random", "datasets": [{"path": "unused.jsonl", "type": "completion"}],
        "output_dir": os.path.join(folder, "out"), "sequence_len": seq, "gradient_accumulation_steps": 1, "max_steps": 1000,
        "learning_rate": 2e-2, "lr_scheduler": "constant", "micro_engram_table_sizes": {2: 4096, 3: 8192},
        "micro_engram_dim": 64, "micro_engram_heads": 2, "micro_engram_gate": "scalar_sqrt",
        "micro_engram_optimizer": "rowwise_adam", "micro_engram_stats_steps": 0, "gradient_checkpointing": False,
        "seed": 7}))
    trainer.build(samples=Samples.from_list([(np.arange(8, 8 + seq, dtype=np.int32), None)] * 4), tokenizer=None)
    return trainer


def packed(lengths, vocab, seq, gen, device):
    """One packed row of random documents: input_ids, position_ids, next-token labels."""
    ids = torch.randint(8, vocab, (1, seq), generator=gen)
    pos = torch.cat([torch.arange(n) for n in lengths] + [torch.arange(seq - sum(lengths))]).view(1, seq)
    labels = torch.full_like(ids, -100)
    labels[0, :-1] = torch.where(pos[0, 1:] == 0, -100, ids[0, 1:])
    labels[0, sum(lengths):] = -100
    return {k: v.to(device) for k, v in (("input_ids", ids), ("position_ids", pos), ("labels", labels))}


def set_output(trainer, std, seed=0):
    """The engram's output projection: 0 is exactly the base."""
    gen = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for slot in trainer.slots:
            w = slot.engram.value.weight
            w.copy_(torch.randn(w.shape, generator=gen) * std)


def main(steps=30, seq=512, vocab=4096, k=32):
    from micro_engram.train.objectives import Distillation, Preference, record_reference, record_teacher

    with tempfile.TemporaryDirectory() as folder:
        trainer = make_trainer(folder, seq, vocab)
        gen = torch.Generator().manual_seed(1)
        third = seq // 3
        batches = [packed([third, third], vocab, seq, gen, trainer.device) for _ in range(2)]

        set_output(trainer, 1.0)
        recorded = [record_teacher(trainer, b, k) for b in batches]
        set_output(trainer, 0.0)
        trainer.objective = Distillation(with_rest=True)
        distill = [trainer.train_step(None, batches=recorded)["loss"] for _ in range(steps)]

        set_output(trainer, 0.0)
        lengths = [third, seq // 4, seq // 5, seq // 6]  # chosen, rejected, chosen, rejected
        pairs = packed(lengths, vocab, seq, gen, trainer.device)
        pairs["cu_seqlens"] = torch.tensor([0] + lengths, device=trainer.device).cumsum(0)
        pairs = record_reference(trainer, pairs)
        trainer.objective = Preference(beta=0.1)
        prefer = [trainer.train_step(None, batches=[pairs])["loss"] for _ in range(steps)]
        rewards = trainer.objective.rewards.tolist()
    out = {"device": str(trainer.device), "distill_loss": [distill[0], distill[-1]],
           "preference_loss": [prefer[0], prefer[-1]], "margins": [c - r for c, r in rewards]}
    import torch.distributed as dist

    if dist.is_initialized():
        dist.destroy_process_group()
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--seq", type=int, default=512)
    args = ap.parse_args()
    print(json.dumps(main(args.steps, args.seq)))
