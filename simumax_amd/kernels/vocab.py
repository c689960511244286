"""Post-training operators over a language model's logits: log probabilities
of given tokens (with entropies and top alternatives) and distillation from a
teacher's top log probabilities, each with its gradient.

They stand beside ``ops.fused_cross_entropy`` and follow its policy: on a GPU
the HIP kernels (csrc/vocab.hip) run, or the call raises; on the CPU plain
torch in 64 bits does. ``ops`` exports both functions.

Both take logits [..., V] in bf16, fp16 or fp32, with any V and any row
strides: a view such as ``logits[:, :-1]`` is read in place (more than two
strides over the rows, or a stride within a row, cost a copy). Statistics,
losses and log probabilities are 32-bit; the gradient has the logits' type.
No call synchronises with the host, and the same input gives the same bits.
The autograd functions here run on the CPU and while ``insitu`` records; else
the extension's own do the same without Python in the backward pass.

What a row gives where its mask leaves little or nothing:

* logits at -inf have probability 0 and add nothing to the entropy;
* a row without a finite logit has no distribution: log probabilities -inf,
  entropy 0, a divergence of +inf, and a gradient of zero;
* a row that holds NaN or +inf gives NaN, and -1 for the ids of its top
  alternatives;
* an id outside [0, V) that does not mark an entry as absent gives NaN for
  its row (on a GPU it cannot be reported without a synchronisation).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import insitu

MAX_TOPK = 256       # VOCAB_MAX_K in csrc/vocab.h
MAX_TOP_V = 524288   # VOCAB_MAX_TOP_V there
NO_MASS = 1e-300     # VOCAB_NO_MASS in csrc/vocab.hip
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]      # [...] fp32, None without tokens
    entropy: torch.Tensor                 # [...] fp32, in nats
    top_logprobs: Optional[torch.Tensor]  # [..., topk] fp32, descending
    top_ids: Optional[torch.Tensor]       # [..., topk] int64


_ops = None  # imports this module: it is looked up at the first call


def _hip(t):
    global _ops
    if not t.is_cuda:
        return None
    if _ops is None:
        from . import ops as _ops
    return _ops.ext()  # raises if missing


def _record(name, nbytes):
    return insitu.start(name, str(nbytes)) if insitu.ENABLED else (
        lambda: None)


def _check_logits(logits, temperature):
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be bf16, fp16 or fp32, "
                        f"not {logits.dtype}")
    shape = logits.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"logits must be [..., V] with V >= 1, "
                         f"not {tuple(shape)}")
    # its reciprocal times log2(e) has to be a normal number of 32 bits
    if not 1e-30 <= float(temperature) <= 1e30:
        raise ValueError(f"temperature must be in [1e-30, 1e30], "
                         f"not {temperature}")
    return shape


def _check_ids(name, ids, shape, device):
    if ids.dtype != torch.int64:
        raise TypeError(f"{name} must be int64, not {ids.dtype}")
    if ids.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, "
                         f"not {tuple(ids.shape)}")
    if ids.device != device:
        raise ValueError(f"{name} is on {ids.device}, the logits on {device}")


# --------------------------------------------------------------------------
# Log probabilities of given tokens, entropies, top alternatives
# --------------------------------------------------------------------------
def _softmax_torch(logits, temperature):
    """Rows in 64 bits: z, its largest value (0 where there is none), the sum
    of exponentials, probabilities, and which rows have none or are bad."""
    z = logits.double() / temperature
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    e = (z - top).exp()
    s = e.sum(-1, keepdim=True)
    none, bad = s == 0, ~(s < float("inf"))
    p = torch.where(none, 0.0, e / s)
    return z - top, s, p, none, bad


def _token_logprobs_torch(logits, tokens, topk, temperature, ignore_index):
    z, s, p, none, bad = _softmax_torch(logits, temperature)
    V = logits.shape[-1]
    lp = torch.where(none, float("-inf"), z - s.log())
    lp = torch.where(bad, float("nan"), lp)
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1, keepdim=True)
    ent = torch.where(bad, float("nan"), ent).squeeze(-1)
    # stable descending sort: the lowest index wins a tie
    ids = torch.where(bad, -1, logits.float().sort(
        dim=-1, descending=True, stable=True).indices[..., :topk])
    top = lp.gather(-1, ids.clamp(min=0))
    logprobs = torch.empty(0)
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < V)
        at = torch.where(inside, tokens, 0)[..., None]
        logprobs = torch.where(inside, lp.gather(-1, at).squeeze(-1),
                               float("nan"))
        left_out = tokens == ignore_index
        logprobs = torch.where(left_out, 0.0, logprobs).float()
        ent = torch.where(left_out, 0.0, ent)
        top = torch.where(left_out[..., None], 0.0, top)
        ids = torch.where(left_out[..., None], -1, ids)
    return logprobs, ent.float(), top.float(), ids


def _token_logprobs_grad_torch(logits, tokens, top_ids, d_logprobs, d_entropy,
                               d_top, temperature, ignore_index):
    z, s, p, none, bad = _softmax_torch(logits, temperature)
    V = logits.shape[-1]
    lp = torch.where(p > 0, z - s.log(), 0.0)
    lp = torch.where(bad, float("nan"), lp)
    d = torch.zeros_like(p)
    if d_logprobs is not None:
        inside = (tokens >= 0) & (tokens < V)
        g = torch.where(inside, d_logprobs.double(), float("nan"))[..., None]
        d = d - p * g
        d.scatter_add_(-1, torch.where(inside, tokens, 0)[..., None], g)
    if d_entropy is not None:
        ent = -(p * lp).sum(-1, keepdim=True)
        d = d - d_entropy.double()[..., None] * p * (lp + ent)
    if d_top is not None:
        g = d_top.double()
        d = d - p * g.sum(-1, keepdim=True)
        d.scatter_add_(-1, top_ids.clamp(min=0), g)
    d = torch.where(none, 0.0, d / temperature)
    if tokens is not None:
        d = torch.where((tokens == ignore_index)[..., None], 0.0, d)
    return d.to(logits.dtype)


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, topk, temperature, ignore_index):
        ctx.set_materialize_grads(False)
        ctx.args = (temperature, ignore_index)
        e = _hip(logits)
        if e is None:
            lp, ent, top, ids = _token_logprobs_torch(
                logits, tokens, topk, temperature, ignore_index)
            stat = None
        else:
            stop = _record("bw_token_logprobs",
                           logits.numel() * logits.element_size())
            lp, ent, top, ids, stat = e.token_logprobs_fwd(
                logits, tokens, topk, temperature, ignore_index)
            stop()
        ctx.save_for_backward(logits, tokens, ids, stat)
        ctx.mark_non_differentiable(ids)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, d_lp, d_ent, d_top, _):
        logits, tokens, ids, stat = ctx.saved_tensors
        if tokens is None:
            d_lp = None
        if ids.shape[-1] == 0:
            d_top = None
        if stat is None:
            return _token_logprobs_grad_torch(
                logits, tokens, ids, d_lp, d_ent, d_top,
                *ctx.args), None, None, None, None
        grads = [None if g is None else g.contiguous()
                 for g in (d_lp, d_ent, d_top)]
        stop = _record("bw_token_logprobs_bwd",
                       2 * logits.numel() * logits.element_size())
        d = _hip(logits).token_logprobs_bwd(logits, tokens, ids, stat,
                                            *grads, *ctx.args)
        stop()
        return d, None, None, None, None


def token_logprobs(logits, tokens=None, topk=0, temperature=1.0,
                   ignore_index=-100):
    """Log probabilities of ``tokens`` under softmax(logits / temperature),
    with each row's entropy and its ``topk`` most probable tokens.

    logits [..., V]; tokens [...] int64, or None where only the entropies and
    alternatives are wanted. A row whose token is ``ignore_index`` is left
    out whole: zeros, ids of -1, no gradient, and it is not read. Of equal
    logits the one of lowest index comes first. ``topk`` <= 256, and where it
    is not 0, V <= 524288.

    Returns ``TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)``, of
    which the first three are differentiable; what was not asked for is
    None."""
    shape = _check_logits(logits, temperature)
    V = shape[-1]
    if not 0 <= topk <= min(MAX_TOPK, V):
        raise ValueError(f"topk must be in [0, {min(MAX_TOPK, V)}] for a "
                         f"vocabulary of {V}, not {topk}")
    if topk and V > MAX_TOP_V:
        raise ValueError(f"top alternatives of a vocabulary of {V}: at most "
                         f"{MAX_TOP_V}")
    if tokens is not None:
        _check_ids("tokens", tokens, shape[:-1], logits.device)
        tokens = tokens.contiguous()
    args = (logits, tokens, int(topk), float(temperature), int(ignore_index))
    if logits.is_cuda and not insitu.ENABLED:
        lp, ent, top, ids = _hip(logits).token_logprobs(*args)
    else:
        lp, ent, top, ids = _TokenLogprobsFn.apply(*args)
    return TokenLogprobs(lp if tokens is not None else None, ent,
                         top if topk else None, ids if topk else None)


# --------------------------------------------------------------------------
# Distillation from a teacher's top log probabilities
# --------------------------------------------------------------------------
def _teacher_torch(teacher_logprobs, teacher_ids, V, bucket):
    held = teacher_ids >= 0
    wrong = (teacher_ids >= V).any(-1, keepdim=True)
    ids = teacher_ids.clamp(0, V - 1)
    l = teacher_logprobs.double()
    q = torch.where(held, l.exp(), 0.0)
    total = q.sum(-1, keepdim=True)
    rest = torch.zeros_like(total)
    if bucket:
        rest = torch.where(total < 1, 1 - total, 0.0)
    else:
        vain = total <= NO_MASS
        q = torch.where(vain, 0.0, q / total)
        l = l - torch.where(vain, 0.0, total.log())
    left_out = ~held.any(-1, keepdim=True)
    if not bucket:
        left_out = left_out | vain
    return held, wrong, ids, l, q, rest, left_out


def _topk_distillation_torch(logits, teacher_logprobs, teacher_ids,
                             temperature, bucket, dloss=None):
    """Losses, or, given theirs, the logits' gradients."""
    V = logits.shape[-1]
    z, s, p, none, bad = _softmax_torch(logits, temperature)
    held, wrong, ids, l, q, q_rest, left_out = _teacher_torch(
        teacher_logprobs, teacher_ids, V, bucket)
    inf = float("inf")
    lp = torch.where(none, -inf, z - s.log()).gather(-1, ids)
    loss = torch.where(q == 0, 0.0, q * (l - lp)).sum(-1, keepdim=True)
    inside = torch.zeros_like(p).scatter_add_(-1, ids, held.double()) > 0
    ratio = torch.zeros_like(loss)
    if bucket:
        p_rest = torch.where(inside, 0.0, p).sum(-1, keepdim=True)
        open_ = (q_rest > 0) & (p_rest > NO_MASS)
        ratio = torch.where(open_, q_rest / p_rest, 0.0)
        loss = loss + torch.where(open_, q_rest * ratio.log(), 0.0)
        loss = torch.where((p_rest <= NO_MASS) & (q_rest > 2.0 ** -20), inf,
                           loss)
    nan = bad | wrong
    if dloss is None:
        loss = torch.where(nan, float("nan"), loss)
        return torch.where(left_out, 0.0, loss).squeeze(-1).float()
    mass = q.sum(-1, keepdim=True) + q_rest
    d = p * torch.where(inside, mass, mass - ratio)
    d = d.scatter_add(-1, ids, -q)
    # the rows without a gradient last: they have none of a NaN either
    d = d * dloss.double()[..., None] / temperature
    d = torch.where(none, 0.0, d)
    d = torch.where(nan, float("nan"), d)
    return torch.where(left_out, 0.0, d).to(logits.dtype)


class _TopkDistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logprobs, teacher_ids, temperature,
                bucket):
        ctx.args = (temperature, bucket)
        e = _hip(logits)
        if e is None:
            loss = _topk_distillation_torch(
                logits, teacher_logprobs, teacher_ids, temperature, bucket)
            ctx.save_for_backward(logits, teacher_logprobs, teacher_ids, None)
            return loss
        stop = _record("bw_topk_distillation",
                       logits.numel() * logits.element_size())
        loss, entry, stat = e.topk_distillation_fwd(
            logits, teacher_logprobs, teacher_ids, temperature, bucket)
        stop()
        ctx.save_for_backward(logits, None, entry, stat)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        logits, teacher, entry, stat = ctx.saved_tensors
        temperature, bucket = ctx.args
        if stat is None:
            return _topk_distillation_torch(
                logits, teacher, entry, temperature, bucket,
                dloss), None, None, None, None
        stop = _record("bw_topk_distillation_bwd",
                       2 * logits.numel() * logits.element_size())
        d = _hip(logits).topk_distillation_bwd(dloss.contiguous(), logits,
                                               entry, stat, temperature)
        stop()
        return d, None, None, None, None


def topk_distillation(logits, teacher_logprobs, teacher_ids, temperature=1.0,
                      tail="renormalize"):
    """Divergence KL(teacher || student) of softmax(logits / temperature)
    from a teacher known by its top log probabilities, per row in fp32.

    logits [..., V]; teacher_logprobs [..., K] at the same temperature, in
    any float type, and teacher_ids [..., K] int64, as ``token_logprobs``
    gives them (K <= 256); an id below 0 marks an absent entry, a row without
    entries has loss 0 and no gradient, as has one whose entries are to
    be scaled and have a mass of no more than 1e-300. With l_k and i_k a row's
    entries and p the student's probabilities:

    * ``tail="renormalize"``: the teacher's entries are scaled to sum to 1,
      q = softmax(l), and the loss is sum_k q_k (ln q_k - ln p[i_k]);
    * ``tail="bucket"``: q_k = exp(l_k), and what is left of the teacher,
      q_r = max(0, 1 - sum q), is compared with what the student gives to all
      tokens that are not listed, p_r: the loss gains q_r (ln q_r - ln p_r).
      Where nothing is left of the student (p_r up to 1e-300), q_r up to 2^-20
      (the rounding of 32-bit log probabilities) counts as none, and more as
      +inf.

    Only the logits receive a gradient. The loss is not scaled by
    temperature^2."""
    shape = _check_logits(logits, temperature)
    if tail not in ("renormalize", "bucket"):
        raise ValueError(f"tail must be 'renormalize' or 'bucket', "
                         f"not {tail!r}")
    if teacher_ids.dim() != logits.dim():
        raise ValueError(f"teacher_ids must be [..., K] beside logits of "
                         f"{tuple(logits.shape)}, not "
                         f"{tuple(teacher_ids.shape)}")
    K = teacher_ids.shape[-1]
    if not 1 <= K <= MAX_TOPK:
        raise ValueError(f"a row takes 1 to {MAX_TOPK} teacher entries, "
                         f"not {K}")
    shape = (*shape[:-1], K)
    _check_ids("teacher_ids", teacher_ids, shape, logits.device)
    if not teacher_logprobs.is_floating_point():
        raise TypeError(f"teacher_logprobs must be floating point, "
                        f"not {teacher_logprobs.dtype}")
    if (teacher_logprobs.shape != shape
            or teacher_logprobs.device != logits.device):
        raise ValueError(f"teacher_logprobs must be {shape} on "
                         f"{logits.device}, not "
                         f"{tuple(teacher_logprobs.shape)} on "
                         f"{teacher_logprobs.device}")
    args = (logits, teacher_logprobs.detach().float().contiguous(),
            teacher_ids.contiguous(), float(temperature), tail == "bucket")
    if logits.is_cuda and not insitu.ENABLED:
        return _hip(logits).topk_distillation(*args)
    return _TopkDistillationFn.apply(*args)
