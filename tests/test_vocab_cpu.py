"""Vocabulary operators on the CPU: what they compute, what they refuse, and
their gradients against differences."""

import math

import pytest
import torch
import vocab_reference as R

from simumax_amd.kernels import ops as K
from simumax_amd.kernels import vocab as VO

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("rows,V,topk,temperature", [
    (1, 1, 1, 1.0), (3, 7, 7, 0.5), (5, 257, 20, 1.0), (2, 1000, 0, 1.7)])
def test_logprobs(dtype, rows, V, topk, temperature):
    gen = _gen(rows * V + topk)
    x = R.make_logits(rows, V, dtype, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    g = torch.randn(rows, generator=gen)
    h = torch.rand(rows, generator=gen)
    gk = torch.randn(rows, topk, generator=gen) if topk else None
    xg = x.clone().requires_grad_(True)
    out = K.token_logprobs(xg, tok, topk=topk, temperature=temperature)
    loss = (out.logprobs * g).sum() + (out.entropy * h).sum()
    if topk:
        loss = loss + (out.top_logprobs * gk).sum()
    loss.backward()
    R.check_logprobs(x, tok, topk, temperature, out, (g, h, gk), xg.grad)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("rows,V,k,temperature", [
    (1, 1, 1, 1.0), (4, 9, 9, 1.0), (5, 257, 20, 0.7), (2, 1000, 64, 2.0)])
def test_distillation(dtype, tail, rows, V, k, temperature):
    gen = _gen(rows * V + k)
    x = R.make_logits(rows, V, dtype, gen)
    tlp, tid = R.make_teacher(x, k, temperature, gen)
    g = torch.randn(rows, generator=gen)
    xg = x.clone().requires_grad_(True)
    loss = K.topk_distillation(xg, tlp, tid, temperature, tail)
    loss.backward(g)
    R.check_distill(x, tlp, tid, temperature, tail, loss, xg.grad, g)


def test_gradients_against_differences():
    gen = _gen(3)
    V, T, step = 11, 0.8, 1e-6
    x = R.make_logits(1, V, FP, gen)[0].double()
    tlp, tid = R.make_teacher(x[None].float(), 4, T, gen)
    tid[0, 3] = tid[0, 1]  # the same token twice

    def logp(v):
        lp, p = R.softmax_row(v, T)
        top = v.sort(descending=True, stable=True).indices[:3]
        w = torch.tensor([0.3, -0.5, 0.9], dtype=torch.float64)
        return (1.3 * lp[2] - 0.4 * -(p * lp).sum() + (w * lp[top]).sum())

    def loss(v, tail):
        return R.distill_row(v, list(zip(tlp[0].tolist(), tid[0].tolist())),
                             T, tail)[0]

    def differences(f):
        out = torch.zeros(V, dtype=torch.float64)
        for i in range(V):
            e = torch.zeros(V, dtype=torch.float64)
            e[i] = step
            out[i] = (float(f(x + e)) - float(f(x - e))) / (2 * step)
        return out

    # second-order differences of a smooth function: step^2 times its third
    # derivative (below 10 here) and 64-bit cancellation, 1e-15 / step
    tol = 10 * step ** 2 + 20 * 2e-15 / step
    xg = x.float()[None].requires_grad_(True)
    o = K.token_logprobs(xg, torch.tensor([2]), topk=3, temperature=T)
    w = torch.tensor([[0.3, -0.5, 0.9]])
    (1.3 * o.logprobs - 0.4 * o.entropy + (w * o.top_logprobs).sum(-1)).sum(
    ).backward()
    # the gradient comes in fp32, from fp32 weights
    assert torch.allclose(xg.grad[0].double(), differences(logp),
                          rtol=4 * R.U, atol=tol + 8 * R.U)
    for tail in ("renormalize", "bucket"):
        xg = x.float()[None].requires_grad_(True)
        K.topk_distillation(xg, tlp, tid, T, tail).backward(torch.ones(1))
        assert torch.allclose(xg.grad[0].double(),
                              differences(lambda v: loss(v, tail)),
                              rtol=4 * R.U, atol=tol + 8 * R.U)


def edge_logits(V, dtype):
    """Rows whose masks leave little or nothing."""
    low = torch.finfo(dtype).min
    gen = _gen(11)
    x = R.make_logits(10, V, dtype, gen)
    x[0] = -math.inf                      # nothing left
    x[1, 1:] = -math.inf                  # one token left, the first
    x[2, :-1] = -math.inf                 # one token left, the last
    x[3] = low                            # masked with the lowest value
    x[4, ::2] = low
    x[5, V // 2] = math.nan
    x[6, V // 3] = math.inf
    x[7] = 0.0
    x[7, ::2] = -0.0                      # equal, whatever the sign
    x[8, 5:] = -math.inf                  # fewer tokens than alternatives
    x[9, :V // 2] = x[9, 0]               # ties
    return x


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_edge_rows(dtype):
    V, topk = 300, 9
    x = edge_logits(V, dtype)
    tok = torch.tensor([3, 0, 0, 4, 2, 1, 1, 0, 3, V - 1])
    g, h = torch.ones(10), torch.full((10,), 0.5)
    xg = x.clone().requires_grad_(True)
    out = K.token_logprobs(xg, tok, topk=topk)
    torch.autograd.backward((out.logprobs, out.entropy), (g, h))
    R.check_logprobs(x, tok, topk, 1.0, out, (g, h, None), xg.grad)
    assert out.logprobs[2] == -math.inf  # a barred token
    gen = _gen(12)
    tlp, tid = R.make_teacher(R.make_logits(10, V, dtype, gen), 6, 1.0, gen)
    for tail in ("renormalize", "bucket"):
        xg = x.clone().requires_grad_(True)
        loss = K.topk_distillation(xg, tlp, tid, tail=tail)
        loss.backward(g)
        R.check_distill(x, tlp, tid, 1.0, tail, loss, xg.grad, g)
        assert loss[0] == math.inf and (xg.grad[0] == 0).all()


def edge_teachers(V, k, gen):
    x = R.make_logits(9, V, FP, gen)
    tlp, tid = R.make_teacher(x, k, 1.0, gen)
    tid[0] = -1                                # no entries
    tid[1, 1:] = -1                            # one
    tid[2, 2] = tid[2, 0]                      # the same token twice
    tlp[3] = -math.inf                         # entries without mass
    tlp[4, 1] = -math.inf
    tid[5, 0] = V                              # outside
    tlp[6, 2] = math.nan
    tlp[7] -= tlp[7].logsumexp(-1)             # nothing left for the rest
    x[8, tid[8]] += 60.0                       # nothing left of the student
    return x, tlp, tid


def far_teachers(V, k, gen, dtype=FP):
    """Students that leave the tokens that are not listed less than 32 bits
    hold, teachers whose entries have next to no mass."""
    x = R.make_logits(8, V, FP, gen)
    tlp, tid = R.make_teacher(x, k, 1.0, gen)
    for r, gap in enumerate((95.0, 130.0, 500.0)):
        x[r, tid[r]] += gap
    x[3] -= 110.0                              # a mask of about -100
    x[3, tid[3]] += 110.0
    x[4, tid[4, 0]] += 200.0                   # one token has it all
    tlp[5] -= 100.0
    tlp[6] -= 600.0
    tlp[7, 0] = -90.0
    tid[7, 1:] = -1
    return x.to(dtype), tlp, tid


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_far_teachers(tail):
    gen = _gen(6)
    x, tlp, tid = far_teachers(123, 7, gen)
    g = torch.randn(8, generator=gen)
    xg = x.clone().requires_grad_(True)
    loss = K.topk_distillation(xg, tlp, tid, tail=tail)
    loss.backward(g)
    R.check_distill(x, tlp, tid, 1.0, tail, loss, xg.grad, g)
    assert loss.isfinite().all()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_edge_teachers(tail):
    gen = _gen(5)
    x, tlp, tid = edge_teachers(123, 7, gen)
    g = torch.randn(9, generator=gen)
    xg = x.clone().requires_grad_(True)
    loss = K.topk_distillation(xg, tlp, tid, tail=tail)
    loss.backward(g)
    R.check_distill(x, tlp, tid, 1.0, tail, loss, xg.grad, g)
    assert loss[0] == 0 and (xg.grad[0] == 0).all()


def test_tokens_left_out_and_outside():
    x = R.make_logits(4, 50, FP, _gen(8)).requires_grad_(True)
    tok = torch.tensor([-100, 50, -1, 7])
    out = K.token_logprobs(x, tok, topk=2)
    (out.logprobs.sum() + out.top_logprobs.sum()).backward()
    assert out.logprobs[0] == 0 and out.entropy[0] == 0
    assert out.top_ids[0].tolist() == [-1, -1]
    assert (x.grad[0] == 0).all()
    assert out.logprobs[1].isnan() and out.logprobs[2].isnan()
    assert x.grad[1].isnan().all() and not x.grad[3].isnan().any()
    # another index than the default
    assert K.token_logprobs(x, tok, ignore_index=7).logprobs[3] == 0


def test_no_rows():
    x = torch.zeros(0, 3, 17, requires_grad=True)
    out = K.token_logprobs(x, torch.zeros(0, 3, dtype=torch.int64), topk=2)
    assert out.logprobs.shape == (0, 3) and out.top_ids.shape == (0, 3, 2)
    loss = K.topk_distillation(x, torch.zeros(0, 3, 2),
                               torch.zeros(0, 3, 2, dtype=torch.int64))
    (out.logprobs.sum() + loss.sum()).backward()
    assert x.grad.shape == x.shape


def test_shapes_and_views():
    gen = _gen(9)
    full = R.make_logits(2 * 6, 31, FP, gen).view(2, 6, 31)
    tok = torch.randint(0, 31, (2, 5), generator=gen)
    xg = full.clone().requires_grad_(True)
    out = K.token_logprobs(xg[:, :-1], tok, topk=3)
    out.logprobs.sum().backward()
    flat = full[:, :-1].reshape(10, 31)
    g = torch.ones(10)
    ref = K.TokenLogprobs(out.logprobs.reshape(-1), out.entropy.reshape(-1),
                          out.top_logprobs.reshape(10, 3),
                          out.top_ids.reshape(10, 3))
    R.check_logprobs(flat, tok.reshape(-1), 3, 1.0, ref, (g, None, None),
                     xg.grad[:, :-1].reshape(10, 31))
    assert (xg.grad[:, -1] == 0).all()
    # one row without leading dimensions
    one = K.token_logprobs(full[0, 0], tok[0, 0], topk=1)
    assert one.logprobs.shape == () and one.top_ids.shape == (1,)
    assert torch.equal(one.logprobs, out.logprobs[0, 0].detach())


def test_top_alternatives_feed_distillation():
    gen = _gen(10)
    teacher = R.make_logits(6, 200, FP, gen)
    tok = torch.tensor([1, 2, -100, 4, 5, 6])
    top = K.token_logprobs(teacher, tok, topk=16, temperature=1.5)
    # a student that equals its teacher has nothing to learn; the row left
    # out by the teacher counts nothing
    for tail in ("renormalize", "bucket"):
        s = teacher.clone().requires_grad_(True)
        loss = K.topk_distillation(s, top.top_logprobs, top.top_ids, 1.5,
                                   tail)
        loss.sum().backward()
        assert loss[2] == 0 and (s.grad[2] == 0).all()
        if tail == "bucket":
            # sixteen entries and the rest, each term's rounding at most
            # 2 u of |ln q| + |ln p| <= 40
            assert loss.abs().max() <= 17 * 2 * R.U * 40
            assert s.grad.abs().max() <= 40 * 4 * R.U


@pytest.mark.parametrize("kw,err", [
    (dict(topk=-1), ValueError), (dict(topk=18), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=-1.0), ValueError),
    (dict(temperature=math.inf), ValueError),
    (dict(temperature=math.nan), ValueError),
    (dict(tokens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(tokens=torch.zeros(2, 1, dtype=torch.int64)), ValueError),
    (dict(tokens=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(tokens=torch.zeros(2, dtype=torch.int64, device="meta")),
     ValueError),
    (dict(logits=torch.zeros(2, 17, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(2, 17, dtype=torch.int64)), TypeError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(())), ValueError),
    (dict(logits=torch.zeros(2, 1000), topk=257), ValueError),
    (dict(logits=torch.zeros(2, 524289), topk=1), ValueError),
])
def test_logprobs_refuses(kw, err):
    args = dict(logits=torch.zeros(2, 17),
                tokens=torch.zeros(2, dtype=torch.int64))
    args.update(kw)
    with pytest.raises(err):
        K.token_logprobs(**args)


@pytest.mark.parametrize("kw,err", [
    (dict(tail="drop"), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(teacher_ids=torch.zeros(2, 4, dtype=torch.int32)), TypeError),
    (dict(teacher_ids=torch.zeros(2, 5, dtype=torch.int64)), ValueError),
    (dict(teacher_ids=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(teacher_ids=torch.zeros(2, 0, dtype=torch.int64),
          teacher_logprobs=torch.zeros(2, 0)), ValueError),
    (dict(teacher_ids=torch.zeros(2, 257, dtype=torch.int64),
          teacher_logprobs=torch.zeros(2, 257)), ValueError),
    (dict(teacher_logprobs=torch.zeros(2, 4, dtype=torch.int64)), TypeError),
    (dict(teacher_logprobs=torch.zeros(2, 4, device="meta")), ValueError),
    (dict(logits=torch.zeros(3, 17)), ValueError),
    (dict(logits=torch.zeros(2, 17, dtype=torch.float64)), TypeError),
])
def test_distillation_refuses(kw, err):
    args = dict(logits=torch.zeros(2, 17), teacher_logprobs=torch.zeros(2, 4),
                teacher_ids=torch.zeros(2, 4, dtype=torch.int64))
    args.update(kw)
    with pytest.raises(err):
        K.topk_distillation(**args)


@pytest.mark.parametrize("T", [9e-31, 1.1e30, 1e-45, 1e300])
def test_temperatures_past_32_bits_are_refused(T):
    x = torch.zeros(2, 17)
    ids = torch.zeros(2, 4, dtype=torch.int64)
    with pytest.raises(ValueError):
        K.token_logprobs(x, temperature=T)
    with pytest.raises(ValueError):
        K.topk_distillation(x, torch.zeros(2, 4), ids, temperature=T)


@pytest.mark.parametrize("T", [1e-30, 1e30])
def test_extreme_temperatures(T):
    x = R.make_logits(4, 300, torch.float32, torch.Generator().manual_seed(5))
    tok = torch.tensor([0, 1, int(x[2].argmax()), 299])
    xg = x.clone().requires_grad_()
    out = K.token_logprobs(xg, tok, topk=3, temperature=T)
    g, h = torch.ones(4), torch.full((4,), 0.5)
    torch.autograd.backward([out.logprobs, out.entropy], [g, h])
    R.check_logprobs(x, tok, 3, T, out, (g, h, None), xg.grad)


def test_limit_matches_the_kernels():
    import os
    import re

    path = os.path.join(os.path.dirname(VO.__file__), "csrc", "vocab.h")
    with open(path) as f:
        assert int(re.search(r"VOCAB_MAX_K (\d+)", f.read()).group(1)) \
            == VO.MAX_TOPK


def check_rows_without_a_gradient(device):
    """Left-out rows and rows without a finite logit have a gradient of zero,
    whatever comes from above for them."""
    gen = _gen(13)
    V, k = 300, 5
    x = R.make_logits(5, V, FP, gen)
    x[1] = -math.inf
    tlp, tid = R.make_teacher(R.make_logits(5, V, FP, gen), k, 1.0, gen)
    tid[0] = -1
    tlp[2] = -math.inf          # nothing to scale to 1
    tok = torch.tensor([-100, 3, -100, 4, 5])
    x, tlp, tid, tok = (t.to(device) for t in (x, tlp, tid, tok))
    for bad in (math.nan, math.inf):
        g = torch.tensor([bad, bad, bad, 1.0, bad], device=device)
        for tail, zero in (("renormalize", (0, 1, 2)), ("bucket", (0, 1))):
            xg = x.clone().requires_grad_(True)
            loss = K.topk_distillation(xg, tlp, tid, tail=tail)
            loss.backward(g)
            for r in zero:
                assert (xg.grad[r] == 0).all(), (tail, bad, r)
            assert xg.grad[3].isfinite().all()
            assert not xg.grad[4].isfinite().any()
        xg = x.clone().requires_grad_(True)
        out = K.token_logprobs(xg, tok, topk=2)
        torch.autograd.backward((out.logprobs, out.entropy), (g, g))
        for r in (0, 1, 2):
            assert (xg.grad[r] == 0).all(), (bad, r)
        assert xg.grad[3].isfinite().all()


def test_rows_without_a_gradient():
    check_rows_without_a_gradient("cpu")
