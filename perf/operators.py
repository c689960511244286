"""What the vocabulary operators of post-training are measured on.

Two operators over the rows of a language model's logits:

* ``token_logprobs``: log probabilities of given tokens, with each row's
  entropy and its top alternatives, and the gradient of the logits;
* ``topk_distillation``: the divergence of a student's distribution from a
  teacher's top log probabilities, and the gradient of the logits.

``run`` computes them in plain torch operations, or, where ``own`` is true,
through the framework's entry points. ``exact`` gives the same outputs in 64
bits, block by block of rows, from the definitions.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}
IGNORE = -100


def _case(name, op, batch, seq, vocab, dtype, topk, temperature=1.0,
          grad=False, shift=False, masked=0.0, padded=0.0, tail=""):
    """batch x seq rows of `vocab` logits; `topk`: alternatives returned, or
    entries of the teacher; `shift`: the rows are a view that leaves out the
    last position of every sequence; `masked`: share of the vocabulary at
    -inf; `padded`: share of rows behind the end of their sequence."""
    return dict(name=name, op=op, batch=batch, seq=seq, vocab=vocab,
                dtype=dtype, topk=topk, temperature=temperature, grad=grad,
                shift=shift, masked=masked, padded=padded, tail=tail)


def listed():
    return [
        # one sampled token of one sequence, with its 20 alternatives
        _case("lp_one", "logprobs", 1, 1, 128257, "bf16", 20),
        # a step of 64 sequences under a grammar that bars most tokens
        _case("lp_step", "logprobs", 64, 1, 151936, "bf16", 20,
              temperature=0.7, masked=0.9),
        # a teacher's pass over one sequence, its top 64 kept for a student
        _case("lp_teacher", "logprobs", 1, 4096, 128257, "bf16", 64),
        # the same from 32-bit logits, 128 kept
        _case("lp_teacher_fp32", "logprobs", 1, 512, 102400, "fp32", 128,
              shift=True),
        # a policy's log probabilities with an entropy bonus, both directions
        _case("lp_policy", "logprobs", 2, 4096, 128257, "bf16", 0, grad=True,
              shift=True),
        # odd rows of an odd vocabulary in fp16, a fifth of them padding
        _case("lp_padded", "logprobs", 1, 1021, 50257, "fp16", 4,
              temperature=0.9, grad=True, padded=0.2),
        # a micro batch of a few tokens
        _case("di_small", "distill", 1, 16, 32000, "bf16", 8, grad=True,
              tail="renormalize"),
        # one training sequence from the teacher's renormalised top 64
        _case("di_sequence", "distill", 1, 4096, 128384, "bf16", 64,
              grad=True, tail="renormalize"),
        # fp16 logits, a softened distribution, the last position left out
        _case("di_soft", "distill", 2, 1024, 129280, "fp16", 20,
              temperature=2.0, grad=True, shift=True, tail="renormalize"),
        # 32-bit logits of odd size, the teacher's remaining mass in a bucket
        _case("di_fp32", "distill", 7, 111, 50257, "fp32", 100, grad=True,
              tail="bucket"),
        # an evaluation pass, loss alone
        _case("di_eval", "distill", 1, 4096, 151936, "bf16", 50,
              tail="bucket"),
        # the largest: two sequences, the teacher's top 128 and a bucket
        _case("di_largest", "distill", 2, 4096, 128257, "bf16", 128,
              grad=True, padded=0.05, tail="bucket"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = min(_log_uniform(rng, 1000, 160000), 160000)
    vocab += rng.choice([0, 0, 1, 3])
    # never more logits than the largest listed case
    largest = 8192 * 128257 // (2 if dtype == "fp32" else 1)
    rows = max(1, min(_log_uniform(rng, 1, 16384), largest // vocab))
    batch = rng.choice([1, 1, 2, 5])
    seq = max(1, rows // batch)
    if batch * seq > rows:
        batch = 1
    temperature = rng.choice([1.0, 1.0, 0.6, 1.7])
    shift = rng.random() < 0.3
    if op == "logprobs":
        grad = rng.random() < 0.5
        return _case("", op, batch, seq, vocab, dtype,
                     rng.choice([0, 1, 5, 20, 64, 128, 256]),
                     temperature=temperature, grad=grad, shift=shift,
                     masked=rng.choice([0.0, 0.0, 0.3, 0.95]),
                     padded=rng.choice([0.0, 0.0, 0.25]))
    return _case("", op, batch, seq, vocab, dtype,
                 rng.choice([1, 4, 16, 50, 100, 128, 200, 256]),
                 temperature=temperature, grad=rng.random() < 0.8,
                 shift=shift, padded=rng.choice([0.0, 0.0, 0.25]),
                 tail=rng.choice(["renormalize", "bucket"]))


def _logits(case, gen):
    """Rows as a language model gives them: a broad body, and a few tokens
    per row that stand out by up to a factor of e^12."""
    b, s, v = case["batch"], case["seq"], case["vocab"]
    s_all = s + 1 if case["shift"] else s
    out = torch.empty(b, s_all, v, dtype=DTYPES[case["dtype"]],
                      device="cuda")
    flat = out.view(-1, v)
    for lo in range(0, flat.shape[0], 1024):
        part = flat[lo:lo + 1024]
        x = torch.randn(part.shape, generator=gen, device="cuda") * 2.0
        n = min(40, v)
        ids = torch.randint(0, v, (part.shape[0], n), generator=gen,
                            device="cuda")
        peaks = torch.rand(part.shape[0], n, generator=gen, device="cuda")
        x.scatter_add_(1, ids, 12.0 * peaks ** 2)
        if case["masked"]:
            keep = torch.rand(part.shape, generator=gen, device="cuda")
            x.masked_fill_(keep < case["masked"], float("-inf"))
        part.copy_(x)
    return out[:, :-1] if case["shift"] else out


def _padding(case, gen):
    """[batch, seq] truth: rows behind the end of their sequence."""
    b, s = case["batch"], case["seq"]
    if not case["padded"]:
        return torch.zeros(b, s, dtype=torch.bool, device="cuda")
    share = torch.rand(b, generator=gen, device="cuda") * 2 * case["padded"]
    keep = ((1 - share.clamp(max=1.0)) * s).ceil()
    return torch.arange(s, device="cuda")[None] >= keep[:, None]


def _unit(case):
    """What a row's loss counts: its share of the mean, or, in fp16, where
    that would vanish, what a loss scale makes of it."""
    if case["dtype"] == "fp16":
        return 64.0
    return 1.0 / (case["batch"] * case["seq"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = _logits(case, gen)
    b, s, v = logits.shape
    pad = _padding(case, gen)
    state = dict(case=case, logits=logits.detach())
    if case["op"] == "logprobs":
        # tokens that the row may hold: a barred one is not sampled
        flat = logits.reshape(-1, v)
        tokens = torch.empty(b * s, dtype=torch.int64, device="cuda")
        for lo in range(0, b * s, 1024):
            part = flat[lo:lo + 1024].float()
            noise = torch.rand(part.shape, generator=gen, device="cuda")
            tokens[lo:lo + 1024] = (part - (-noise.log()).log()).argmax(-1)
        tokens = tokens.view(b, s).masked_fill_(pad, IGNORE)
        state["tokens"] = tokens
        if case["grad"]:
            # a policy's advantages, and the weight of its entropy bonus
            unit = _unit(case)
            state["d_logprobs"] = torch.randn(b, s, generator=gen,
                                              device="cuda") * unit
            state["d_entropy"] = torch.rand(b, s, generator=gen,
                                            device="cuda") * 0.1 * unit
    else:
        # the teacher's logits are near the student's; its top entries come
        # as log probabilities at the loss's temperature
        k = case["topk"]
        ids = torch.empty(b * s, k, dtype=torch.int64, device="cuda")
        lps = torch.empty(b * s, k, dtype=torch.float32, device="cuda")
        flat = logits.reshape(-1, v)
        for lo in range(0, b * s, 1024):
            part = flat[lo:lo + 1024].float()
            noise = torch.randn(part.shape, generator=gen, device="cuda")
            t = (part + 0.5 * noise) / case["temperature"]
            top, where = t.topk(k, dim=-1)
            ids[lo:lo + 1024] = where
            lps[lo:lo + 1024] = top - t.logsumexp(-1, keepdim=True)
        ids = ids.view(b, s, k).masked_fill_(pad[:, :, None], -1)
        state["teacher_ids"] = ids
        state["teacher_logprobs"] = lps.view(b, s, k).masked_fill_(
            pad[:, :, None], 0.0)
        if case["grad"]:
            state["d_loss"] = torch.full((b, s), _unit(case), device="cuda")
    if case["grad"]:
        state["logits"].requires_grad_(True)
    return state


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "logprobs":
            return _plain_logprobs(case, state)
        return _plain_distill(case, state)


# --------------------------------------------------------------------------
# through the framework
# --------------------------------------------------------------------------
def _run_own(case, state):
    from simumax_amd.kernels import ops as K

    logits = state["logits"]
    if case["op"] == "logprobs":
        out = K.token_logprobs(logits, state["tokens"], topk=case["topk"],
                               temperature=case["temperature"],
                               ignore_index=IGNORE)
        res = dict(logprobs=out.logprobs, entropy=out.entropy)
        if case["topk"]:
            res["top_logprobs"] = out.top_logprobs
            res["top_ids"] = out.top_ids
        if case["grad"]:
            res["d_logits"], = torch.autograd.grad(
                (out.logprobs, out.entropy), logits,
                (state["d_logprobs"], state["d_entropy"]))
        return {n: t.detach() for n, t in res.items()}
    loss = K.topk_distillation(logits, state["teacher_logprobs"],
                               state["teacher_ids"],
                               temperature=case["temperature"],
                               tail=case["tail"])
    res = dict(loss=loss)
    if case["grad"]:
        res["d_logits"], = torch.autograd.grad(loss, logits, state["d_loss"])
    return {n: t.detach() for n, t in res.items()}


# --------------------------------------------------------------------------
# plain form
# --------------------------------------------------------------------------
def _unique_keys(x):
    """Whole numbers that sort as (value up, index down): no two of a row
    are equal, so the lowest index wins a tie."""
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    index = torch.arange(x.shape[-1], device=x.device)
    return (order << 32) | (0x7FFFFFFF - index)


def _plain_logprobs(case, state):
    logits, tokens = state["logits"], state["tokens"]
    v, t, k = case["vocab"], case["temperature"], case["topk"]
    keep = tokens != IGNORE
    x = logits.float() / t
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    s = e.sum(-1, keepdim=True)
    lp = x - top - s.log()
    p = e / s
    ent = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    safe = torch.where(keep, tokens, 0)
    tok = lp.gather(-1, safe[..., None]).squeeze(-1)
    res = dict(logprobs=torch.where(keep, tok, 0.0),
               entropy=torch.where(keep, ent, 0.0))
    if k:
        best = _unique_keys(logits.float()).topk(k, dim=-1).values
        ids = 0x7FFFFFFF - (best & 0x7FFFFFFF)
        res["top_logprobs"] = torch.where(keep[..., None],
                                          lp.gather(-1, ids), 0.0)
        res["top_ids"] = torch.where(keep[..., None], ids, -1)
    if case["grad"]:
        g, h = state["d_logprobs"][..., None], state["d_entropy"][..., None]
        hot = torch.arange(v, device=x.device) == safe[..., None]
        bonus = torch.where(p > 0, p * (lp + ent[..., None]), 0.0)
        d = (g * (hot.float() - p) - h * bonus) / t
        res["d_logits"] = torch.where(keep[..., None], d,
                                      0.0).to(logits.dtype)
    return res


def _plain_distill(case, state):
    logits = state["logits"]
    ids, tl = state["teacher_ids"], state["teacher_logprobs"]
    t = case["temperature"]
    held = ids >= 0
    safe = torch.where(held, ids, 0)
    x = logits.float() / t
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    s = e.sum(-1, keepdim=True)
    p = e / s
    lp = (x - top - s.log()).gather(-1, safe)
    q = torch.where(held, tl.double().exp(), 0.0)
    inside = torch.zeros(x.shape, dtype=torch.bool, device=x.device)
    b, r, _ = x.shape
    at_b = torch.arange(b, device=x.device)[:, None, None].expand_as(ids)
    at_r = torch.arange(r, device=x.device)[None, :, None].expand_as(ids)
    inside[at_b[held], at_r[held], ids[held]] = True
    if case["tail"] == "renormalize":
        total = q.sum(-1, keepdim=True)
        q = torch.where(total > 0, q / total, 0.0)
        q_rest = torch.zeros_like(total)
        lost = torch.zeros_like(total)
    else:
        q_rest = (1.0 - q.sum(-1, keepdim=True)).clamp(min=0.0)
        rest = torch.where(inside, 0.0, p).sum(-1, keepdim=True).double()
        lost = torch.where(q_rest > 0, q_rest * (q_rest / rest).log(), 0.0)
    loss = torch.where(q > 0, q * (q.log() - lp), 0.0).sum(-1)
    loss = (loss + lost.squeeze(-1)).float()
    res = dict(loss=loss)
    if case["grad"]:
        scale = state["d_loss"][..., None] / t
        mass = (q.sum(-1, keepdim=True) + q_rest).float()
        d = p * mass
        if case["tail"] == "bucket":
            ratio = torch.where(q_rest > 0, q_rest / rest, 0.0).float()
            d = d - torch.where(inside, 0.0, p * ratio)
        d.scatter_add_(-1, safe, -q.float())
        res["d_logits"] = (d * scale).to(logits.dtype)
    return res


# --------------------------------------------------------------------------
# 64 bits, from the definitions
# --------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    v = case["vocab"]
    rows = case["batch"] * case["seq"]
    flat = state["logits"].detach().reshape(rows, v)
    block = max(1, min(rows, (1 << 27) // v))
    parts = {}
    for lo in range(0, rows, block):
        part = {n: t.reshape(rows, *t.shape[2:])[lo:lo + block]
                for n, t in state.items()
                if torch.is_tensor(t) and n != "logits"}
        z = flat[lo:lo + block].double() / case["temperature"]
        one = (_exact_logprobs if case["op"] == "logprobs"
               else _exact_distill)(case, z, part)
        for n, t in one.items():
            parts.setdefault(n, []).append(t)
    lead = (case["batch"], case["seq"])
    return {n: torch.cat(ts).reshape(*lead, *ts[0].shape[1:])
            for n, ts in parts.items()}


def _exact_logprobs(case, z, part):
    tokens = part["tokens"]
    norm = z.logsumexp(-1)
    prob = (z - norm[:, None]).exp()
    mean = (prob * z.clamp(min=-1e300)).sum(-1)
    entropy = norm - mean
    live = (tokens != IGNORE).double()
    at = tokens.clamp(min=0)[:, None]
    res = dict(logprobs=(z.gather(1, at)[:, 0] - norm) * live,
               entropy=entropy * live)
    k = case["topk"]
    if k:
        order = z.sort(dim=-1, descending=True, stable=True)
        dead = tokens == IGNORE
        res["top_logprobs"] = (order.values[:, :k] - norm[:, None]
                               ).masked_fill(dead[:, None], 0.0)
        res["top_ids"] = order.indices[:, :k].clone().masked_fill(
            dead[:, None], -1)
    if case["grad"]:
        g = part["d_logprobs"].double() * live
        h = part["d_entropy"].double() * live
        # dH/dz_j = p_j (E[z] - z_j), d logp/dz_j = [j is the token] - p_j
        d = prob * (h[:, None] * (mean[:, None] - z.clamp(min=-1e300))
                    - g[:, None])
        d.scatter_add_(1, at, g[:, None])
        res["d_logits"] = d / case["temperature"]
    return res


def _exact_distill(case, z, part):
    ids, tl = part["teacher_ids"], part["teacher_logprobs"].double()
    rows, v = z.shape
    # the teacher as a dense row, with one column for the padding
    at = torch.where(ids < 0, v, ids)
    dense = torch.zeros(rows, v + 1, dtype=torch.float64, device=z.device)
    dense.scatter_add_(1, at, tl.exp())
    member = torch.zeros(rows, v + 1, dtype=torch.float64, device=z.device)
    member.scatter_(1, at, 1.0)
    dense, member = dense[:, :v], member[:, :v]
    norm = z.logsumexp(-1, keepdim=True)
    prob = (z - norm).exp()
    held = dense.sum(-1, keepdim=True)
    grad = None
    if case["tail"] == "renormalize":
        dense = dense / held.where(held > 0, torch.ones_like(held))
        mass = (held > 0).double()
        loss = (torch.xlogy(dense, dense) - dense * (z - norm)).sum(-1)
        grad = prob * mass - dense
    else:
        q_rest = (1.0 - held).clamp(min=0.0)
        p_rest = (prob * (1.0 - member)).sum(-1, keepdim=True)
        loss = (torch.xlogy(dense, dense) - dense * (z - norm)).sum(-1)
        loss = loss + (torch.xlogy(q_rest, q_rest)
                       - torch.xlogy(q_rest, p_rest))[:, 0]
        ratio = torch.where(q_rest > 0, q_rest / p_rest,
                            torch.zeros_like(q_rest))
        grad = (prob * (held + q_rest) - dense
                - prob * (1.0 - member) * ratio)
    res = dict(loss=loss)
    if case["grad"]:
        res["d_logits"] = (grad * part["d_loss"].double()[:, None]
                           / case["temperature"])
    return res


def work(case):
    rows = case["batch"] * case["seq"]
    n = rows * case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    k = case["topk"]
    # the logits once and, in training, their gradient once
    nbytes = n * size * (2 if case["grad"] else 1)
    if case["op"] == "logprobs":
        # tokens; log probabilities and entropies; the alternatives; the
        # gradients of the first two
        nbytes += rows * (8 + 8 + 12 * k + (8 if case["grad"] else 0))
    else:
        # the teacher's entries and ids, the loss and its gradient
        nbytes += rows * (12 * k + 4 + (4 if case["grad"] else 0))
    # scale, subtract, exponential, sum (and one more product and sum for
    # the entropy); the gradient's exponential and products
    per = 6 if case["op"] == "logprobs" else 4
    return {"bytes": nbytes, "flops": n * (per + (5 if case["grad"] else 0))}
