"""Distillation through the trainer: a teacher's top log probabilities feed
the student's loss, against the same written out in plain torch."""

import pytest
import torch

from simumax_amd.core.config import ModelConfig
from simumax_amd.train.model import LlamaForTraining
from simumax_amd.train.trainer import (TrainConfig, build_trainer,
                                       distill_step, make_synthetic_batch)


def _config(head_size=16, hidden=64):
    return ModelConfig(hidden_size=hidden, head_num=4, kv_head_num=2,
                       head_size=head_size, intermediate_size=128,
                       layer_num=2, vocab_size=384, use_swiglu=True,
                       model_type="dense")


def _plain_loss(logits, top_lp, top_ids, T, tail):
    lp = torch.log_softmax(logits.double() / T, -1)
    q = top_lp.double().exp()
    if tail == "renormalize":
        q = q / q.sum(-1, keepdim=True)
    loss = (q * (q.log() - lp.gather(-1, top_ids))).sum(-1)
    if tail == "bucket":
        q_rest = (1 - q.sum(-1)).clamp(min=0)
        p_rest = lp.exp().scatter(-1, top_ids, 0.0).sum(-1)
        loss = loss + torch.xlogy(q_rest, q_rest / p_rest)
    return loss.mean()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_loss_and_gradients(tail):
    T, topk = 1.3, 12
    cfg = _config()
    torch.manual_seed(0)
    teacher = LlamaForTraining(cfg, 16, dtype=torch.float32)
    student = LlamaForTraining(cfg, 16, dtype=torch.float32)
    with torch.no_grad():
        for m in (teacher, student):
            m.lm_head.weight.mul_(20)      # distributions that differ
    toks = torch.randint(0, cfg.vocab_size, (2, 16))
    with torch.no_grad():
        top = teacher.token_logprobs(toks, topk=topk, temperature=T)
        ref = torch.log_softmax(teacher.logits(toks).double() / T, -1)
    # the teacher's logits are 32-bit; their log probabilities are rounded
    # once more, half a step of a number below 16
    assert (top.top_logprobs - ref.topk(topk).values).abs().max() <= 2 ** -20
    loss = student.distillation_loss(toks, top.top_logprobs, top.top_ids, T,
                                     tail)
    loss.backward()
    got = {n: p.grad.clone() for n, p in student.named_parameters()}
    student.zero_grad(set_to_none=True)
    plain = _plain_loss(student.logits(toks), top.top_logprobs, top.top_ids,
                        T, tail)
    plain.backward()
    # the loss is one 32-bit rounding per row and the mean's, of terms < 32
    assert abs(loss.item() - plain.item()) <= 32 * 4 * 2 ** -24 * 32
    for n, p in student.named_parameters():
        # both go through the same 32-bit model: sums of at most 512 terms
        # in each of its 20 products, a half step each
        room = 20 * 512 * 2 ** -24 * p.grad.abs().max()
        assert (got[n] - p.grad).abs().max() <= room, n


def test_positions_without_a_teacher_do_not_count():
    cfg = _config()
    torch.manual_seed(1)
    student = LlamaForTraining(cfg, 8, dtype=torch.float32)
    toks = torch.randint(0, cfg.vocab_size, (1, 8))
    targets = torch.randint(0, cfg.vocab_size, (1, 8))
    targets[0, 5:] = -100
    top = student.token_logprobs(toks, targets, topk=4)
    lp, ids = top.top_logprobs.detach() - 0.5, top.top_ids
    assert (ids[0, 5:] == -1).all()
    whole = student.distillation_loss(toks, lp, ids)
    part = student.distillation_loss(toks[:, :5], lp[:, :5], ids[:, :5])
    assert abs(whole.item() - part.item()) <= 1e-5 * abs(part.item())


def test_sharded_vocabulary_is_refused():
    cfg = _config()
    m = LlamaForTraining(cfg, 8, dtype=torch.float32, tp_size=2)
    with pytest.raises(NotImplementedError):
        m.token_logprobs(torch.zeros(1, 8, dtype=torch.int64))


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_distill_step(device):
    if device != "cpu" and not torch.cuda.is_available():
        pytest.skip("no GPU")
    cfg = _config(head_size=128, hidden=512)
    tc = TrainConfig(seq_len=64, micro_batch_size=2, micro_batch_num=2)
    teacher, _, tr = build_trainer(cfg, tc, device)
    student, opt, red = build_trainer(cfg, tc, device)
    with torch.no_grad():
        # another model than the teacher
        for p in student.parameters():
            p.add_(0.05 * torch.randn_like(p))
    toks, _ = make_synthetic_batch(cfg.vocab_size, 2, 2, 64, device)
    before = [p.detach().clone() for p in student.parameters()]
    for tail in ("renormalize", "bucket"):
        loss = distill_step(student, teacher, opt, red, toks, 2, topk=16,
                            tail=tail)
        assert 0 < loss < float("inf")
    assert all(torch.isfinite(p).all() for p in student.parameters())
    assert any((a != b).any() for a, b in zip(before, student.parameters()))
    red.remove_hooks()
    tr.remove_hooks()
