"""What a training step minimises: next-token cross entropy (the default), distillation from a teacher's
recorded top logits, or a preference loss over packed chosen / rejected sequences.

An objective is given to the trainer before its steps (``trainer.objective = Distillation()``); it gets the
final hidden states of a micro-batch and the batch's tensors, and returns the sum of its terms. ``fields`` names what it
needs of a batch beside input_ids and position_ids:

  NextToken     labels
  Distillation  teacher_ids, teacher_logits [tokens, k] (and teacher_lse [tokens] with the temperature that it is of,
                teacher_temperature): record_teacher()
  Preference    ref_logps [tokens] (record_reference()) and cu_seqlens [2 pairs + 1]; one micro-batch
                holds whole pairs

The data set's batches have labels alone, so the last two run through ``trainer.train_step(None, batches=[...])`` on
batches that the caller records; ``trainer.train()``, which draws its batches from the data set, refuses them.

Teacher and reference are models of the same vocabulary. A natural reference policy is the frozen base
without its engram; natural teachers are the bf16 base of an NF4 run and a larger model. The last two
need the whole head on the GPU, as a trainer on one GPU has it (VocabShard with world 1).
"""
import torch

from micro_engram_fork_b200.ops import objectives as ops

from .head import IGNORE


def _flat(batch, key):
    return batch[key].reshape(-1)


def trained_tokens(batch):
    return (batch["labels"] != IGNORE).sum()


class NextToken:
    """Summed cross entropy of the trained tokens."""
    fields = ("labels",)

    def terms(self, batch):
        """How many terms the sum has (the step minimises their mean): here the trained tokens."""
        return trained_tokens(batch)

    def __call__(self, vocab, hidden, batch):
        return vocab.loss_sum(hidden, _flat(batch, "labels"))[0]


class Distillation(NextToken):
    """Summed divergence from the teacher over the trained tokens; with_rest: the teacher's mass outside its
    entries is a class of its own (teacher_lse, recorded at the same temperature: a batch that says another one, in
    teacher_temperature, is refused)."""

    def __init__(self, temperature=1.0, with_rest=False):
        self.temperature, self.with_rest = float(temperature), with_rest
        self.fields = ("labels", "teacher_ids", "teacher_logits") + (("teacher_lse",) if with_rest else ())

    def __call__(self, vocab, hidden, batch):
        lse = None
        if self.with_rest:
            lse = _flat(batch, "teacher_lse")
            recorded = float(batch.get("teacher_temperature", self.temperature))
            if recorded != self.temperature:
                raise ValueError(f"teacher_lse was recorded at temperature {recorded:g}, the distillation with the rest "
                                 f"is at {self.temperature:g}: record_teacher(..., temperature={self.temperature:g})")
        k = batch["teacher_ids"].shape[-1]
        weights = (_flat(batch, "labels") != IGNORE).float()
        return vocab.distill(hidden, batch["teacher_ids"].reshape(-1, k), batch["teacher_logits"].reshape(-1, k), lse,
                             weights, self.temperature).sum()


class Preference:
    """Summed loss of the micro-batch's pairs; `rewards` [pairs, 2] of the last call."""
    fields = ("labels", "ref_logps", "cu_seqlens")

    def __init__(self, beta=0.1, label_smoothing=0.0, kind="sigmoid"):
        self.args = (beta, label_smoothing, kind)
        self.rewards = None

    def terms(self, batch):
        cu = batch["cu_seqlens"]
        return torch.full((), cu.numel() // 2, dtype=torch.int64, device=cu.device)

    def __call__(self, vocab, hidden, batch):
        logps = vocab.token_logprobs(hidden, _flat(batch, "labels"))
        loss, self.rewards = ops.preference_loss(logps, _flat(batch, "ref_logps"), batch["cu_seqlens"], *self.args)
        return loss.sum()


def record_teacher(trainer, batch, k, temperature=1.0):
    """The batch with this trainer's model's top logits on it: teacher_ids, teacher_logits, teacher_lse and
    teacher_temperature (one number, on the host)."""
    with torch.no_grad():
        values, ids, lse = trainer.vocab.top_logits(trainer.hidden(batch), k, temperature)
    return {**batch, "teacher_ids": ids, "teacher_logits": values, "teacher_lse": lse,
            "teacher_temperature": torch.tensor(float(temperature), dtype=torch.float64)}


def record_reference(trainer, batch):
    """The batch with this trainer's model's token log-probabilities on it: ref_logps."""
    with torch.no_grad():
        return {**batch, "ref_logps": trainer.vocab.token_logprobs(trainer.hidden(batch), _flat(batch, "labels"))}
