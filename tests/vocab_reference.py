"""Plain 64-bit forms of the vocabulary operators, row by row from their
definitions, and how far a 32-bit computation may be from them.

Bounds, with u = 2^-24 (half a step of fp32). A term 2^d, d = (x - m) c <= 0,
is off by at most |d| ln 2 * 2u for the rounded c and d, and 2u for the
exponential itself; a sum of n <= 64 terms in order and a tree of 6 adds 70 u
at most. Terms with large |d| are small, and V of them reach the largest
term's size only where d > -log2 V > -20: a sum of exponentials is off by at
most (2 * 20 * 0.7 + 2 + 70) u < 100 u of itself, and so is its logarithm,
absolutely. The entropy adds a sum of d 2^d, whose terms' relative error is
that of 2^d plus 2u for d and 1u for the product: 105 u.
"""

import math

import torch

U = 2.0 ** -24
SUM = 100 * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def softmax_row(x, temperature):
    """z, log p (-inf where p is 0), p, in 64 bits; None without a finite
    logit, NaN where there is no distribution."""
    z = x.double() / temperature
    if torch.isnan(z).any() or (z == math.inf).any():
        nan = torch.full_like(z, math.nan)
        return nan, nan
    if (z == -math.inf).all():
        return None
    # shifted first: ln V is lost beside a type's lowest value
    z = z - z.max()
    lp = z - z.exp().sum().log()
    return lp, lp.exp()


def logprobs_row(x, token, topk, temperature, ignore=-100, g=0.0, h=0.0,
                 gk=None):
    """(logprob, entropy, top_logprobs, top_ids, gradient, bound on the
    gradient before its last rounding) of one row; token None: none given."""
    if token is not None and token == ignore:
        zero = torch.zeros(x.numel(), dtype=torch.float64)
        return 0.0, 0.0, [0.0] * topk, [-1] * topk, zero, zero
    order = []
    if topk:
        order = x.double().sort(descending=True,
                                stable=True).indices[:topk].tolist()
    return _logprobs_row(x, token, order, temperature, g, h, gk)


def _logprobs_row(x, token, order, temperature, g, h, gk):
    V = x.numel()
    nan = math.nan
    sm = softmax_row(x, temperature)
    zero = torch.zeros(V, dtype=torch.float64)
    if sm is None:
        lp = -math.inf
        if token is not None and not 0 <= token < V:
            lp = nan
        return lp, 0.0, [-math.inf] * len(order), order, zero, zero
    lp, p = sm
    if torch.isnan(lp).any():
        bad = torch.full((V,), nan, dtype=torch.float64)
        return nan, nan, [nan] * len(order), [-1] * len(order), bad, zero
    plogp = torch.where(p > 0, p * lp, 0.0)
    H = -float(plogp.sum())
    at = nan
    if token is not None and 0 <= token < V:
        at = float(lp[token])
    grad, mag = torch.zeros(V, dtype=torch.float64), p * 0
    if token is not None and g:
        if 0 <= token < V:
            grad[token] += g
            mag[token] += abs(g)
        else:
            g = nan
        grad = grad - g * p
        mag = mag + abs(g) * p
    if h:
        grad = grad - h * (plogp + p * H)
        mag = mag + abs(h) * (plogp.abs() + p * H)
    if gk is not None:
        for i, v in zip(order, gk):
            grad[i] += v
            mag[i] += abs(v)
        grad = grad - sum(gk) * p
        mag = mag + sum(abs(v) for v in gk) * p
    # p is off by its exponent's error and the sum's
    err = (2 * 0.7 * (lp.clamp(min=-150).abs() / math.log(2)) + 10) * U + SUM
    return (at, H, [float(lp[i]) for i in order], order, grad / temperature,
            mag * (err + 105 * U) / temperature)


def distill_row(x, teacher, temperature, tail, g=1.0):
    """(loss, bound, gradient, bound) of one row; teacher: [(l, id)]."""
    V = x.numel()
    nan, inf = math.nan, math.inf
    zero = torch.zeros(V, dtype=torch.float64)
    held = [(float(l), int(i)) for l, i in teacher if i >= 0]
    q = [math.exp(l) for l, _ in held]
    total = sum(q)
    if not held or (tail == "renormalize" and total == 0):
        return 0.0, 0.0, zero, zero
    sm = softmax_row(x, temperature)
    bad = torch.full((V,), nan, dtype=torch.float64)
    if any(i >= V for _, i in held) or total != total:
        return nan, 0.0, bad, zero
    if sm is not None and torch.isnan(sm[0]).any():
        return nan, 0.0, bad, zero
    rest = 0.0
    if tail == "renormalize":
        q = [v / total for v in q]
    else:
        rest = max(0.0, 1.0 - total)
    if sm is None:
        lost = any(v > 0 for v in q) or rest > 2.0 ** -20
        return (inf if lost else 0.0), 0.0, zero, zero
    lp, p = sm
    loss, bound = 0.0, 0.0
    dense, inside = zero.clone(), torch.zeros(V, dtype=torch.bool)
    for v, (l, i) in zip(q, held):
        if v > 0:
            lq = math.log(v)
            loss += v * (lq - float(lp[i]))
            bound += v * (abs(lq) + abs(float(lp[i])) + 1) * 4 * U + v * SUM
        dense[i] += v
        inside[i] = True
    ratio = 0.0
    if rest > 0:
        p_rest = float(p[~inside].sum())
        if p_rest > 0:
            loss += rest * math.log(rest / p_rest)
            bound += rest * 2 * SUM
            ratio = rest / p_rest
        elif rest > 2.0 ** -20:
            loss = inf
    mass = sum(q) + rest
    # of two Python numbers torch.where makes 32 bits
    coef = mass - torch.where(inside, 0.0, ratio * torch.ones_like(p))
    grad = (p * coef - dense) * g / temperature
    mag = p * (2 * mass - coef) + dense
    err = (2 * 0.7 * (lp.clamp(min=-150).abs() / math.log(2)) + 20) * U \
        + 3 * SUM
    return (loss, bound + abs(loss) * 2 * U if loss < inf else 0.0, grad,
            mag * err * abs(g) / temperature)


def assert_close(got, want, bound, what, dtype=torch.float32):
    """|got - want| <= bound + half a step of the type at the wanted value,
    and the type's smallest numbers, below which it has no relative step
    (32-bit exponentials below 2^-126 are 0)."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    # what passes the type's range rounds to infinity
    want = torch.where(want.abs() > torch.finfo(dtype).max,
                       want.sign() * math.inf, want)
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu()
    same = ((torch.isnan(got) & torch.isnan(want)) | (got == want))
    step = torch.where(want.abs() < math.inf, want.abs(), 0.0) \
        * half_step(dtype)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps + 2.0 ** -120
    off = torch.where(same, 0.0, (got - want).abs())
    off = torch.nan_to_num(off, nan=math.inf, posinf=math.inf)
    room = bound.nan_to_num(nan=0.0) * (1 + half_step(dtype)) + step + tiny
    worst = (off - room).max().item() if off.numel() else 0.0
    i = (off - room).reshape(-1).argmax().item() if off.numel() else 0
    assert worst <= 0, (
        f"{what}: {got.reshape(-1)[i]} for {want.reshape(-1)[i]}, off by "
        f"{off.reshape(-1)[i]:.3e} with room for "
        f"{room.expand_as(off).reshape(-1)[i]:.3e}, at {i} of {off.numel()}")


def make_logits(rows, V, dtype, gen, spread=2.0):
    """A broad body with some tokens that stand out, and many ties (the
    16-bit types' own)."""
    x = torch.randn(rows, V, generator=gen) * spread
    n = max(1, V // 100)
    at = torch.randint(0, V, (rows, n), generator=gen)
    x.scatter_add_(1, at, 9 * torch.rand(rows, n, generator=gen))
    return x.to(dtype)


def check_logprobs(x, tokens, topk, temperature, out, grads=None, d=None,
                   ignore=-100):
    """x [rows, V] on the CPU; out the operator's TokenLogprobs with rows
    flattened; grads (g [rows], h [rows], gk [rows, topk] or None) and the
    logits' gradient d."""
    rows = x.shape[0]
    g, h, gk = grads if grads is not None else (None, None, None)
    ref = []
    for r in range(rows):
        ref.append(logprobs_row(
            x[r], None if tokens is None else int(tokens[r]), topk,
            temperature, ignore,
            0.0 if g is None else float(g[r]),
            0.0 if h is None else float(h[r]),
            None if gk is None else [float(v) for v in gk[r]]))
    f = dict(dtype=torch.float64)
    if tokens is not None:
        want = torch.tensor([t[0] for t in ref], **f)
        assert_close(out.logprobs, want, SUM + 4 * U, "logprobs")
    else:
        assert out.logprobs is None
    H = torch.tensor([t[1] for t in ref], **f)
    assert_close(out.entropy, H, (2 + H.nan_to_num()) * 210 * U, "entropy")
    if topk:
        ids = torch.tensor([t[3] for t in ref])
        assert torch.equal(out.top_ids.cpu(), ids), "top_ids"
        assert_close(out.top_logprobs, torch.tensor([t[2] for t in ref], **f),
                     SUM + 4 * U, "top_logprobs")
    else:
        assert out.top_ids is None and out.top_logprobs is None
    if d is not None:
        assert d.dtype == x.dtype
        for r in range(rows):
            assert_close(d[r], ref[r][4], ref[r][5], f"gradient of row {r}",
                         x.dtype)


def check_distill(x, tlp, tid, temperature, tail, loss, d=None, g=None):
    rows = x.shape[0]
    ref = [distill_row(x[r], list(zip(tlp[r].tolist(), tid[r].tolist())),
                       temperature, tail,
                       1.0 if g is None else float(g[r]))
           for r in range(rows)]
    f = dict(dtype=torch.float64)
    assert_close(loss, torch.tensor([t[0] for t in ref], **f),
                 torch.tensor([t[1] for t in ref], **f), "loss")
    if d is not None:
        assert d.dtype == x.dtype
        for r in range(rows):
            assert_close(d[r], ref[r][2], ref[r][3], f"gradient of row {r}",
                         x.dtype)


def make_teacher(x, K, temperature, gen, noise=0.5):
    """Top K log probabilities of logits near x."""
    t = (x.float() + noise * torch.randn(x.shape, generator=gen)) / temperature
    top, ids = t.topk(K, dim=-1)
    return top - t.logsumexp(-1, keepdim=True), ids
