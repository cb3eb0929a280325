"""Distillation of one LM into another of the same vocabulary, on the device.

A teacher's runtime records the top logits of every position; the student's
runtime trains on them (hx_lm_distill_forward_backward_device and the prepared
optimizer) and generates with its tokens sampled on the device.  Tokens, records
and gradients stay in device memory; only losses and generated ids come back.

    python -m hexatrain_b200.distillation --steps 200

trains a small student from a wider teacher that is itself trained first, on
seeded Zipf tokens of a repeating pattern, and samples a continuation.
"""
from __future__ import annotations

import argparse

import numpy as np

from . import data
from .parallel import _device_view
from .runtime import LmConfig, OptimizerConfig, Runtime


class Distiller:
    """A teacher and a student runtime with prepared and uploaded LMs of one
    vocabulary, sequence length and batch, driven on torch's current stream."""

    def __init__(self, teacher: Runtime, student: Runtime, k: int = 32, temperature: float = 2.0,
                 kd_weight: float = 0.5, ce_weight: float = 0.5, tail: bool = True):
        import torch
        t, s = teacher._lm_cfg, student._lm_cfg
        if t is None or s is None:
            raise ValueError("distillation: prepare both LMs first")
        if (t.vocabulary_size, t.tokens, teacher._lm_batch) != (s.vocabulary_size, s.tokens, student._lm_batch):
            raise ValueError("distillation: teacher and student differ in vocabulary, sequence length or batch")
        if not 1 <= k <= min(256, s.vocabulary_size):
            raise ValueError("distillation: record length must be in [1, min(256, vocabulary)]")
        self.teacher, self.student = teacher, student
        self.k, self.temperature, self.kd_weight, self.ce_weight = k, temperature, kd_weight, ce_weight
        self.batch, rows = student._lm_batch, student._lm_batch * s.tokens
        self.tokens = torch.empty(self.batch, s.tokens + 1, device="cuda", dtype=torch.int32)
        self.values = torch.empty(rows, k, device="cuda")
        self.indices = torch.empty(rows, k, device="cuda", dtype=torch.int32)
        self.lse = torch.empty(rows, device="cuda") if tail else None
        self._torch = torch

    def _check(self, ok: bool, rt: Runtime):
        if not ok:
            raise RuntimeError(rt.last_error)

    def step(self, tokens, step: int) -> None:
        """One training step of the student on tokens [batch, T+1]; `step` is
        1-based.  Asynchronous: loss() reads the result."""
        torch = self._torch
        stream = torch.cuda.current_stream().cuda_stream or 1  # 1: the legacy default stream
        for rt in (self.teacher, self.student):
            self._check(rt.set_stream(stream), rt)
        self.tokens.copy_(torch.from_numpy(np.ascontiguousarray(tokens, np.uint32).view(np.int32)))
        lse = 0 if self.lse is None else self.lse.data_ptr()
        self._check(self.teacher.lm_top_logits_device(self.tokens.data_ptr(), self.k, self.values.data_ptr(),
                                                      self.indices.data_ptr(), lse, self.temperature), self.teacher)
        self._check(self.student.lm_distill_forward_backward_device(
            self.tokens.data_ptr(), 1.0 / self.batch, self.k, self.values.data_ptr(), self.indices.data_ptr(), lse,
            self.temperature, self.kd_weight, self.ce_weight), self.student)
        self._check(self.student.lm_optimizer_step_device(step), self.student)

    def loss(self) -> float:
        """The mean loss of the last step (waits for it).  Raises what either runtime
        found wrong since the last time, a token id beyond the vocabulary among it."""
        p, n = self.student.lm_grad_buffer()
        done = [(rt.synchronize(), rt) for rt in (self.teacher, self.student)]
        for ok, rt in done:
            self._check(ok, rt)
        return float(_device_view(p, n)[-1])


def pattern_tokens(seed: int, batch: int, tokens: int, vocab: int) -> np.ndarray:
    """Zipf tokens in which every odd position repeats the one before, shifted:
    something to learn."""
    ids = data.lm_tokens(seed, batch, tokens, vocab).astype(np.int64)
    ids[:, 1::2] = (ids[:, 0:ids.shape[1] - 1:2][:, :ids[:, 1::2].shape[1]] * 3 + 1) % vocab
    return ids.astype(np.uint32)


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--vocab", type=int, default=1024)
    ap.add_argument("--seed", type=int, default=20260710)
    a = ap.parse_args(argv)
    wide = LmConfig(a.vocab, 64, 128, 256, 2, 4, learned_position=True)
    small = LmConfig(a.vocab, 64, 64, 64, 2, 4, learned_position=True)
    teacher, student = Runtime(), Runtime()
    for rt, cfg, seed in ((teacher, wide, a.seed), (student, small, a.seed + 1)):
        if not (rt.initialize(0) and rt.prepare_lm(cfg, a.batch) and rt.lm_set_optimizer(OptimizerConfig()) and
                rt.lm_state_upload(cfg.init_normal(seed, 0.02))):
            raise RuntimeError(rt.last_error)
    taught = 0.0
    for step in range(1, a.steps + 1):
        ok, taught = teacher.lm_train_step(pattern_tokens(a.seed + step, a.batch, 64, a.vocab), step)
        if not ok:
            raise RuntimeError(teacher.last_error)
    d = Distiller(teacher, student)
    losses = []
    for step in range(1, a.steps + 1):
        d.step(pattern_tokens(a.seed + 1000000 + step, a.batch, 64, a.vocab), step)
        if step == 1 or step == a.steps:
            losses.append(d.loss())
    prompts = pattern_tokens(a.seed + 7, a.batch, 63, a.vocab)[:, :9]
    ids, log_probs = student.lm_generate_device(prompts, 8, temperature=0.8, top_k=40, top_p=0.95, seed=a.seed)
    if ids is None:
        raise RuntimeError(student.last_error)
    report = dict(teacher_loss=taught, first_loss=losses[0], last_loss=losses[-1], generated=ids, log_probs=log_probs)
    print(f"teacher loss {taught:.4f}; student loss {losses[0]:.4f} -> {losses[-1]:.4f}; stream 0: "
          f"{prompts[0].tolist()} -> {ids[0].tolist()}")
    teacher.close()
    student.close()
    return report


if __name__ == "__main__":
    main()
