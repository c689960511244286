"""Vocabulary kernels (csrc/vocab.hip) on the GPU against plain 64-bit forms:
types, odd sizes, strides, masks, ties, repeated ids, long offsets, streams
and graphs."""

import math

import pytest
import torch
import vocab_reference as R
from test_vocab_cpu import (check_rows_without_a_gradient, edge_logits,
                            edge_teachers, far_teachers)

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from simumax_amd.kernels import ops as K
else:
    pytest.skip("no GPU", allow_module_level=True)

DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def run_logprobs(x, tok, topk, T, grads, **kw):
    """x on the CPU, any strides; forward and backward on the GPU."""
    g, h, gk = grads
    xg = x.to(DEV).requires_grad_(True)
    out = K.token_logprobs(xg, None if tok is None else tok.to(DEV),
                           topk=topk, temperature=T, **kw)
    outs, ds = [], []
    for o, d in ((out.logprobs, g), (out.entropy, h),
                 (out.top_logprobs, gk)):
        if o is not None and d is not None:
            outs.append(o)
            ds.append(d.to(DEV))
    torch.autograd.backward(outs, ds)
    return out, xg.grad


def run_distill(x, tlp, tid, T, tail, g):
    xg = x.to(DEV).requires_grad_(True)
    loss = K.topk_distillation(xg, tlp.to(DEV), tid.to(DEV), T, tail)
    loss.backward(g.to(DEV))
    return loss, xg.grad


SIZES = [(1, 1, 1), (3, 7, 7), (2, 64, 20), (2, 2047, 5), (2, 2048, 64),
         (3, 2049, 256), (2, 4095, 1), (2, 4097, 128), (5, 8195, 20),
         (2, 50257, 100)]


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("rows,V,topk", SIZES)
def test_logprobs(dtype, rows, V, topk):
    gen = _gen(rows * V + topk)
    T = 1.0 if V % 3 else 0.7
    x = R.make_logits(rows, V, dtype, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    grads = (torch.randn(rows, generator=gen), torch.rand(rows, generator=gen),
             torch.randn(rows, topk, generator=gen))
    out, d = run_logprobs(x, tok, topk, T, grads)
    R.check_logprobs(x, tok, topk, T, out, grads, d)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("rows,V,k", SIZES)
def test_distillation(dtype, tail, rows, V, k):
    gen = _gen(rows * V + k + 1)
    T = 1.0 if V % 3 else 2.0
    x = R.make_logits(rows, V, dtype, gen)
    tlp, tid = R.make_teacher(x, k, T, gen)
    g = torch.randn(rows, generator=gen)
    loss, d = run_distill(x, tlp, tid, T, tail, g)
    R.check_distill(x, tlp, tid, T, tail, loss, d, g)


@pytest.mark.parametrize("which", ["logprobs", "entropy", "top", "all"])
def test_logprobs_gradients_alone(which):
    gen = _gen(21)
    rows, V, topk = 3, 5003, 12
    x = R.make_logits(rows, V, FP, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    g, h = torch.randn(rows, generator=gen), torch.rand(rows, generator=gen)
    gk = torch.randn(rows, topk, generator=gen)
    grads = (g if which in ("logprobs", "all") else None,
             h if which in ("entropy", "all") else None,
             gk if which in ("top", "all") else None)
    out, d = run_logprobs(x, tok, topk, 1.0, grads)
    R.check_logprobs(x, tok, topk, 1.0, out, grads, d)
    if which in ("entropy", "top"):
        # without given tokens
        out, d = run_logprobs(x, None, topk, 1.0, grads)
        R.check_logprobs(x, None, topk, 1.0, out, grads, d)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_edge_rows(dtype):
    V, topk = 4300, 9
    x = edge_logits(V, dtype)
    tok = torch.tensor([3, 0, 0, 4, 2, 1, 1, 0, 3, V - 1])
    grads = (torch.ones(10), torch.full((10,), 0.5), None)
    out, d = run_logprobs(x, tok, topk, 1.0, grads)
    R.check_logprobs(x, tok, topk, 1.0, out, grads, d)
    tlp, tid = R.make_teacher(R.make_logits(10, V, dtype, _gen(12)), 6, 1.0,
                              _gen(13))
    for tail in ("renormalize", "bucket"):
        loss, d = run_distill(x, tlp, tid, 1.0, tail, grads[0])
        R.check_distill(x, tlp, tid, 1.0, tail, loss, d, grads[0])


@pytest.mark.parametrize("T", [0.25, 3.0])
def test_edge_rows_at_a_temperature(T):
    # the type's lowest value over T < 1 passes the type's range
    V = 2500
    x = edge_logits(V, FP)
    tok = torch.tensor([3, 0, 0, 4, 2, 1, 1, 0, 3, V - 1])
    grads = (torch.ones(10), torch.full((10,), 0.5), None)
    out, d = run_logprobs(x, tok, 3, T, grads)
    R.check_logprobs(x, tok, 3, T, out, grads, d)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_huge_logits(dtype):
    # steps of the logits' own size, over several stretches
    V = 9000
    gen = _gen(14)
    x = torch.randn(6, V, generator=gen)
    x[0] *= 1e30
    x[1] = -1.7e38
    x[2] = 3e38
    x[3] += 3e6
    x[4] -= 2e5
    x[5, :V // 2] = -3e38
    x = x.to(dtype)
    tok = torch.tensor([0, 1, 2, int(x[3].float().argmax()), 4, V - 1])
    grads = (torch.ones(6), torch.full((6,), 0.5), None)
    for T in (1.0, 0.5):
        out, d = run_logprobs(x, tok, 4, T, grads)
        R.check_logprobs(x, tok, 4, T, out, grads, d)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T", [1e-30, 1e30])
def test_extreme_temperatures(dtype, T):
    V = 2500
    x = R.make_logits(4, V, dtype, _gen(15))
    tok = torch.tensor([0, 1, int(x[2].float().argmax()), V - 1])
    grads = (torch.ones(4), torch.full((4,), 0.5), None)
    out, d = run_logprobs(x, tok, 4, T, grads)
    R.check_logprobs(x, tok, 4, T, out, grads, d)
    tlp, tid = R.make_teacher(R.make_logits(4, V, dtype, _gen(16)), 6, 1.0,
                              _gen(17))
    for tail in ("renormalize", "bucket"):
        loss, d = run_distill(x, tlp, tid, T, tail, grads[0])
        R.check_distill(x, tlp, tid, T, tail, loss, d, grads[0])


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("V", [123, 9001])
def test_edge_teachers(tail, V):
    gen = _gen(5)
    x, tlp, tid = edge_teachers(V, 7, gen)
    g = torch.randn(9, generator=gen)
    loss, d = run_distill(x, tlp, tid, 1.0, tail, g)
    R.check_distill(x, tlp, tid, 1.0, tail, loss, d, g)
    assert loss[0] == 0 and (d[0] == 0).all()


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("V", [123, 9001])
def test_far_teachers(tail, dtype, V):
    gen = _gen(18)
    x, tlp, tid = far_teachers(V, 7, gen, dtype)
    g = torch.randn(8, generator=gen)
    loss, d = run_distill(x, tlp, tid, 1.0, tail, g)
    R.check_distill(x, tlp, tid, 1.0, tail, loss, d, g)
    assert loss.isfinite().all()


def test_teacher_in_one_place():
    # every entry within one stretch, one of them 200 times
    gen = _gen(6)
    V, k = 20001, 256
    x = R.make_logits(2, V, BF, gen)
    tid = torch.randint(9000, 9010, (2, k), generator=gen)
    tid[:, 50:250] = 9003
    tlp = torch.log_softmax(torch.randn(2, k, generator=gen), -1) - 0.1
    g = torch.ones(2)
    for tail in ("renormalize", "bucket"):
        loss, d = run_distill(x, tlp, tid, 1.0, tail, g)
        R.check_distill(x, tlp, tid, 1.0, tail, loss, d, g)


@pytest.mark.parametrize("kind", ["ascending", "descending", "equal", "two",
                                  "cluster", "strided", "masked"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("V,topk", [(30011, 256), (30011, 20), (300, 256),
                                    (262147, 128)])
def test_top_alternatives(kind, dtype, V, topk):
    """Orders of the vocabulary that a search for the largest could take
    badly."""
    gen = _gen(31)
    i = torch.arange(V)
    x = torch.randn(1, V, generator=gen)
    if kind == "ascending":
        x[0] = i / V * 20
    elif kind == "descending":
        x[0] = 20 - i / V * 20
    elif kind == "equal":
        x[0] = 1.5
    elif kind == "two":
        x[0] = (torch.rand(V, generator=gen) < 0.4).float()
    elif kind == "cluster":
        x[0, V // 2:V // 2 + min(1000, V // 2)] += 10
    elif kind == "strided":
        x[0, ::64] += 8
    else:
        x[0, torch.rand(V, generator=gen) < 0.9995] = -math.inf
    x = x.to(dtype)
    out = K.token_logprobs(x.to(DEV), topk=topk)
    R.check_logprobs(x, None, topk, 1.0, out)


def test_strides():
    gen = _gen(41)
    B, S, V, k = 2, 5, 4099, 6
    base = R.make_logits(B * S * 3, V, BF, gen).to(DEV)
    tok = torch.randint(0, V, (B, S), generator=gen)
    g = torch.randn(B, S, generator=gen)
    h = torch.rand(B, S, generator=gen)
    odd = torch.empty(B * S * V + 1, dtype=BF, device=DEV)
    odd[1:] = base[:B * S].reshape(-1)
    views = {
        "last position left out": base[:B * (S + 1)].view(B, S + 1, V)[:, :-1],
        "every third row": base.view(B * S, 3, V)[:, 1].view(B, S, V),
        "sequence first": base[:B * S].view(S, B, V).transpose(0, 1),
        "padded rows": base[:B * S].view(B, S, V)[..., :V - 6],
        "odd start": odd[1:].view(B, S, V),
        "one row for all": base[:1].view(1, 1, V).expand(B, S, V),
        "one row each": base[:B].view(B, 1, V).expand(B, S, V),
        "stride within a row": base[:B * S].view(B, S, V)[..., ::2],
        "three strides": base[:8 * 3].view(2, 3, 4, V)[:, :2, :3],
    }
    for name, v in views.items():
        print(name, tuple(v.shape), v.stride(), flush=True)
        lead, W = v.shape[:-1], v.shape[-1]
        rows = math.prod(lead)
        t = tok.reshape(-1).repeat(2)[:rows].clamp(max=W - 1).view(lead)
        gg = g.reshape(-1).repeat(2)[:rows]
        hh = h.reshape(-1).repeat(2)[:rows]
        x = v.detach().requires_grad_(True)
        out = K.token_logprobs(x, t.to(DEV), topk=k)
        d, = torch.autograd.grad((out.logprobs, out.entropy), x,
                                 (gg.view(lead).to(DEV),
                                  hh.view(lead).to(DEV)))
        cpu = v.cpu().reshape(rows, W)
        flat = K.TokenLogprobs(out.logprobs.reshape(-1),
                               out.entropy.reshape(-1),
                               out.top_logprobs.reshape(rows, k),
                               out.top_ids.reshape(rows, k))
        R.check_logprobs(cpu, t.reshape(-1), k, 1.0, flat, (gg, hh, None),
                         d.reshape(rows, W))
        tlp, tid = R.make_teacher(cpu, k, 1.0, gen)
        # the teacher's tensors and the loss's gradient have strides too
        wide = torch.zeros(rows, 2 * k, dtype=torch.int64)
        wide[:, ::2] = tid
        x = v.detach().requires_grad_(True)
        loss = K.topk_distillation(
            x, tlp.view(*lead, k).to(DEV),
            wide.view(*lead, 2 * k).to(DEV)[..., ::2], tail="bucket")
        d, = torch.autograd.grad(loss, x, torch.full(
            (), 0.5, device=DEV).expand(lead))
        R.check_distill(cpu, tlp, tid, 1.0, "bucket", loss.reshape(-1),
                        d.reshape(rows, W), torch.full((rows,), 0.5))


def test_broadcast_input_gradient():
    # one row read by four: its gradient is the sum of theirs
    gen = _gen(43)
    V = 3001
    x = R.make_logits(1, V, FP, gen)
    tok = torch.randint(0, V, (4,), generator=gen)
    xg = x.to(DEV).requires_grad_(True)
    K.token_logprobs(xg.expand(4, V), tok.to(DEV)).logprobs.sum().backward()
    refs = [R.logprobs_row(x[0], int(t), 0, 1.0, g=1.0) for t in tok]
    want = sum(r[4] for r in refs)
    # three more roundings of the sums
    room = sum(r[5] for r in refs) + 4 * R.U * sum(r[4].abs() for r in refs)
    R.assert_close(xg.grad[0], want, room, "gradient")


def test_rows_past_32_bit_offsets():
    V, gap = 4097, (1 << 30) + 3
    store = torch.empty(2 * gap + V, dtype=BF, device=DEV)
    x = store.as_strided((3, V), (gap, 1))
    cpu = R.make_logits(3, V, BF, _gen(51))
    x.copy_(cpu)
    tok = torch.tensor([1, 2, V - 1])
    xg = x.detach().requires_grad_(True)
    out = K.token_logprobs(xg, tok.to(DEV), topk=5)
    d, = torch.autograd.grad(out.logprobs, xg, torch.ones(3, device=DEV))
    R.check_logprobs(cpu, tok, 5, 1.0, out, (torch.ones(3), None, None), d)


def test_gradient_past_32_bit_offsets():
    rows, V = 17000, 128257
    assert rows * V > 2 ** 31
    x = torch.zeros(rows, V, dtype=BF, device=DEV)
    cpu = R.make_logits(2, V, BF, _gen(52))
    x[-2:] = cpu.to(DEV)
    tok = torch.full((rows,), 5, device=DEV)
    xg = x.requires_grad_(True)
    out = K.token_logprobs(xg, tok)
    d, = torch.autograd.grad(out.logprobs, xg,
                             torch.ones(rows, device=DEV))
    flat = K.TokenLogprobs(out.logprobs[-2:], out.entropy[-2:], None, None)
    R.check_logprobs(cpu, torch.tensor([5, 5]), 0, 1.0, flat,
                     (torch.ones(2), None, None), d[-2:])
    one = R.logprobs_row(torch.zeros(V, dtype=BF), 5, 0, 1.0, g=1.0)
    R.assert_close(d[0], one[4], one[5], "first row", BF)
    R.assert_close(d[12345], one[4], one[5], "a row between", BF)


def test_many_short_rows():
    rows, V = 70001, 3
    gen = _gen(53)
    x = R.make_logits(rows, V, HF, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    out = K.token_logprobs(x.to(DEV), tok.to(DEV), topk=3)
    lp = torch.log_softmax(x.double(), -1)
    R.assert_close(out.logprobs, lp.gather(1, tok[:, None])[:, 0],
                   R.SUM + 4 * R.U, "logprobs")
    order = x.double().sort(dim=-1, descending=True, stable=True)
    assert torch.equal(out.top_ids.cpu(), order.indices)


def test_padding_and_outside():
    gen = _gen(61)
    V = 6001
    x = R.make_logits(5, V, BF, gen)
    tok = torch.tensor([-100, V, -1, 7, V + 2 ** 33])
    grads = (torch.ones(5), torch.ones(5), None)
    out, d = run_logprobs(x, tok, 4, 1.0, grads)
    R.check_logprobs(x, tok, 4, 1.0, out, grads, d)
    assert (d[0] == 0).all() and out.top_ids[0].tolist() == [-1] * 4
    # a row left out is not read: what it holds does not matter
    y = x.clone()
    y[0] = math.nan
    out2, d2 = run_logprobs(y, tok, 4, 1.0, grads)
    assert torch.equal(out.entropy, out2.entropy)
    assert (d2[0] == 0).all()
    tid = torch.tensor([[-1, -1], [5, -1], [-7, 9]])
    loss, d = run_distill(y[:3], torch.full((3, 2), -1.0), tid, 1.0,
                          "renormalize", torch.ones(3))
    R.check_distill(y[:3], torch.full((3, 2), -1.0), tid, 1.0, "renormalize",
                    loss, d, torch.ones(3))


def test_no_rows():
    x = torch.zeros(0, 3, 17, device=DEV, requires_grad=True)
    ids = torch.zeros(0, 3, 2, dtype=torch.int64, device=DEV)
    out = K.token_logprobs(x, ids[..., 0], topk=2)
    loss = K.topk_distillation(x, torch.zeros(0, 3, 2, device=DEV), ids)
    (out.logprobs.sum() + loss.sum()).backward()
    assert out.top_ids.shape == (0, 3, 2) and x.grad.shape == x.shape


def test_same_input_same_bits():
    gen = _gen(71)
    rows, V, k = 33, 50257, 128
    x = R.make_logits(rows, V, BF, gen).to(DEV)
    tok = torch.randint(0, V, (rows,), generator=gen).to(DEV)
    tlp, tid = R.make_teacher(x.cpu(), k, 1.0, gen)
    tlp, tid = tlp.to(DEV), tid.to(DEV)
    tid[:, 3] = tid[:, 9]
    g = torch.randn(rows, generator=gen).to(DEV)

    def once():
        xg = x.detach().requires_grad_(True)
        o = K.token_logprobs(xg, tok, topk=k)
        loss = K.topk_distillation(xg, tlp, tid, tail="bucket")
        d1, = torch.autograd.grad((o.logprobs, o.entropy), xg, (g, g))
        d2, = torch.autograd.grad(loss, xg, g)
        return (o.logprobs, o.entropy, o.top_logprobs, o.top_ids, loss, d1,
                d2)

    first = once()
    for _ in range(3):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_on_another_stream():
    gen = _gen(72)
    rows, V, k = 9, 32003, 16
    x = R.make_logits(rows, V, BF, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    tlp, tid = R.make_teacher(x, k, 1.0, gen)
    g = torch.randn(rows, generator=gen)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, d = run_logprobs(x, tok, k, 1.0, (g, None, None))
        loss, dd = run_distill(x, tlp, tid, 1.0, "bucket", g)
    torch.cuda.current_stream().wait_stream(s)
    R.check_logprobs(x, tok, k, 1.0, out, (g, None, None), d)
    R.check_distill(x, tlp, tid, 1.0, "bucket", loss, dd, g)


def test_two_streams_at_once():
    # calls in flight together share no workspace
    k = 16
    jobs = []
    for i, (rows, V) in enumerate(((300, 32003), (40, 128257))):
        gen = _gen(74 + i)
        x = R.make_logits(rows, V, BF, gen)
        tok = torch.randint(0, V, (rows,), generator=gen)
        tlp, tid = R.make_teacher(x, k, 1.0, gen)
        jobs.append([t.to(DEV) for t in (x, tok, tlp, tid)])

    def work(x, tok, tlp, tid):
        xg = x.detach().requires_grad_(True)
        out = K.token_logprobs(xg, tok, topk=k)
        loss = K.topk_distillation(xg, tlp, tid, tail="bucket")
        d, = torch.autograd.grad(out.logprobs.sum() + loss.sum(), xg)
        return [*out, loss, d]

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(4):
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(*j))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs, want[i % 2]):
            assert torch.equal(a, b)


def test_two_captured_graphs():
    """Forward and backward of both operators, captured into two graphs that
    are replayed in turn on new inputs, with eager calls in between."""
    gen = _gen(73)
    V, k = 12001, 20
    graphs = []

    def work(x, tok, tlp, tid, g):
        xg = x.detach().requires_grad_(True)
        o = K.token_logprobs(xg, tok, topk=k)
        loss = K.topk_distillation(xg, tlp, tid, tail="bucket")
        d, = torch.autograd.grad((o.logprobs, o.entropy, loss), xg, (g, g, g))
        return o.logprobs, o.entropy, o.top_logprobs, o.top_ids, loss, d

    def inputs(rows, seed):
        gi = _gen(seed)
        x = R.make_logits(rows, V, BF, gi)
        tok = torch.randint(0, V, (rows,), generator=gi)
        tlp, tid = R.make_teacher(x, k, 1.0, gi)
        g = torch.randn(rows, generator=gi)
        return [t.to(DEV) for t in (x, tok, tlp, tid, g)]

    for rows in (7, 40):
        static = inputs(rows, rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(*static)
        graphs.append((rows, static, graph, outs))
    for turn in range(3):
        for rows, static, graph, outs in graphs:
            new = inputs(rows, 100 * turn + rows)
            for a, b in zip(static, new):
                a.copy_(b)
            graph.replay()
            want = work(*new)
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_refusals():
    x = torch.zeros(2, 17, device=DEV)
    with pytest.raises(ValueError):
        K.token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        K.topk_distillation(x, torch.zeros(2, 3, device=DEV),
                            torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(TypeError):
        K.token_logprobs(x.double())
    # the extension's own checks
    e = K.ext()
    ids = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError):
        e.token_logprobs_fwd(x, ids, 2, 1.0, -100)
    with pytest.raises(RuntimeError):
        e.token_logprobs_fwd(x, None, 18, 1.0, -100)
    with pytest.raises(RuntimeError):
        e.topk_distillation_fwd(x, torch.zeros(2, 3, device=DEV),
                                ids[:, :2].contiguous(), 1.0, True)
    with pytest.raises(RuntimeError):
        e.topk_distillation_fwd(x, torch.zeros(2, 3, device=DEV).half(),
                                ids, 1.0, True)


def test_in_situ_timing_takes_the_same_kernels():
    # while it records, the Python autograd functions run instead of the
    # extension's own
    from simumax_amd.kernels import insitu

    gen = _gen(81)
    rows, V, k = 5, 9001, 12
    x = R.make_logits(rows, V, BF, gen)
    tok = torch.randint(0, V, (rows,), generator=gen)
    tlp, tid = R.make_teacher(x, k, 1.0, gen)
    grads = (torch.randn(rows, generator=gen), torch.rand(rows, generator=gen),
             torch.randn(rows, k, generator=gen))

    def both():
        out, d = run_logprobs(x, tok, k, 1.0, grads)
        loss, dd = run_distill(x, tlp, tid, 1.0, "bucket", grads[0])
        return [*out, d, loss, dd]

    want = both()
    insitu.enable()
    try:
        got = both()
        recorded = {t for t, _ in insitu._RECORDS}
    finally:
        insitu.disable()
        insitu._RECORDS.clear()
    assert recorded == {"bw_token_logprobs", "bw_token_logprobs_bwd",
                        "bw_topk_distillation", "bw_topk_distillation_bwd"}
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_gradient_of_the_gradient_raises():
    x = torch.randn(2, 40, device=DEV, requires_grad=True)
    ids = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    for loss in (K.token_logprobs(x, ids[:, 0]).logprobs.sum(),
                 K.topk_distillation(x, ids.float(), ids).sum()):
        d, = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            d.sum().backward()


def test_tokens_and_entries_from_an_inference_pass():
    # a teacher under inference_mode or no_grad feeds a student that trains
    gen = _gen(82)
    x = R.make_logits(3, 5000, BF, gen).to(DEV)
    with torch.inference_mode():
        top = K.token_logprobs(x, topk=8)
    lp, ids = top.top_logprobs.clone(), top.top_ids.clone()
    xg = x.clone().requires_grad_(True)
    K.topk_distillation(xg, lp, ids, tail="bucket").sum().backward()
    # nothing to learn from itself: p - q, each off by its rounding
    assert xg.grad.abs().max() <= 2 ** -7
    with torch.no_grad():
        assert not K.token_logprobs(xg, ids[:, 0]).logprobs.requires_grad


def test_backward_into_leaves_captured():
    """loss.backward() of a leaf, captured and replayed: the gradient that it
    accumulates into is the graph's own memory."""
    gen = _gen(83)
    rows, V = 6, 7001
    x = R.make_logits(rows, V, FP, gen).to(DEV)
    tok = torch.randint(0, V, (rows,), generator=gen).to(DEV)
    leaf = x.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            leaf.grad = None
            K.token_logprobs(leaf, tok).logprobs.sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.token_logprobs(leaf, tok).logprobs.sum().backward()
    for turn in range(3):
        new = R.make_logits(rows, V, FP, _gen(84 + turn)).to(DEV)
        with torch.no_grad():
            leaf.copy_(new)
        graph.replay()
        eager = new.clone().requires_grad_(True)
        d, = torch.autograd.grad(
            K.token_logprobs(eager, tok).logprobs.sum(), eager)
        torch.cuda.synchronize()
        assert torch.equal(leaf.grad, d)


@pytest.mark.parametrize("kind", ["clustered", "equal", "masked", "steps"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("V,topk", [(700, 256), (5743, 256), (12345, 200),
                                    (24571, 256)])
def test_alternatives_of_few_groups(kind, dtype, V, topk):
    """Vocabularies whose groups are hardly more than the alternatives."""
    gen = _gen(91 + V)
    x = torch.randn(3, V, generator=gen) * 2
    if kind == "clustered":
        x[:, V // 3:V // 3 + 400] += 9
    elif kind == "equal":
        x = torch.where(torch.rand(3, V, generator=gen) < 0.5, 3.25, 3.0)
    elif kind == "masked":
        x[torch.rand(3, V, generator=gen) < 0.97] = -math.inf
    else:
        # far more octaves than the first count looks at
        x = torch.exp2(torch.randint(-30, 3, (3, V), generator=gen).float())
    x = x.to(dtype)
    out = K.token_logprobs(x.to(DEV), topk=topk)
    R.check_logprobs(x, None, topk, 1.0, out)


@pytest.mark.parametrize("fill", [-math.inf, -1e4, 0.0])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("V,topk", [(40000, 20), (40000, 256), (9001, 64)])
def test_fewer_tokens_than_alternatives(fill, dtype, V, topk):
    """A mask that leaves 0 to 300 tokens: what it fills is ranked by index."""
    gen = _gen(97)
    x = torch.full((5, V), fill)
    for r, left in enumerate((0, 1, 3, 19, 300)):
        at = torch.randperm(V, generator=gen)[:left]
        x[r, at] = torch.rand(left, generator=gen) * 8 + 1
    x[2, V - 1] = 0.5
    x = x.to(dtype)
    out = K.token_logprobs(x.to(DEV), topk=topk)
    R.check_logprobs(x, None, topk, 1.0, out)


def test_rows_of_every_alignment():
    """The same row at each of the 64 places within a cache line that a bf16
    row can begin at, read and written."""
    gen = _gen(95)
    for V in (3, 130, 4093, 8200):
        row = R.make_logits(1, V, BF, gen)
        tok = torch.full((64,), V // 2)
        tlp, tid = R.make_teacher(row, min(V, 9), 1.0, gen)
        store = torch.zeros(64 * (V + 129) + 64, dtype=BF, device=DEV)
        # rows of a stride that is 1 past a whole number of lines
        stride = (V + 63) // 64 * 64 + 1
        x = store.as_strided((64, V), (stride, 1))
        x.copy_(row.to(DEV).expand(64, V))
        k = min(V, 9)
        xg = x.detach().requires_grad_(True)
        out = K.token_logprobs(xg, tok.to(DEV), topk=k)
        loss = K.topk_distillation(xg, tlp.to(DEV).expand(64, k),
                                   tid.to(DEV).expand(64, k), tail="bucket")
        g = torch.ones(64, device=DEV)
        d1, = torch.autograd.grad((out.logprobs, out.entropy), xg, (g, g))
        d2, = torch.autograd.grad(loss, xg, g)
        one = torch.ones(64)
        cpu = row.expand(64, V)
        R.check_logprobs(cpu, tok, k, 1.0, out, (one, one, None), d1)
        R.check_distill(cpu, tlp.expand(64, k), tid.expand(64, k), 1.0,
                        "bucket", loss, d2, one)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("V,wider", [
    (65529, 0), (65535, 0), (131071, 0), (262143, 0),
    # whole numbers of groups per thread, in rows off the cache lines
    (65536, 3), (131072, 8), (262144, 5),
    # the last vocabulary whose stretches begin at lines, and the next one
    (524160, 0), (524161, 0)])
def test_alternatives_at_the_end(V, wider, dtype):
    """The largest tokens are a row's last ones, in rows that begin anywhere
    within a cache line: the groups of 64 are one more than V has."""
    gen = _gen(V + wider)
    rows = 3
    wide = R.make_logits(rows, V + wider, dtype, gen)
    x = wide[..., :V]
    x[:, V - 40:] = (20 + 5 * torch.rand(rows, 40, generator=gen)).to(dtype)
    x[2, :V - 30] = -math.inf  # nothing but the end is left
    xg = wide.to(DEV)[..., :V].detach().requires_grad_(True)
    for topk in (1, 20, 256):
        print("topk", topk, flush=True)
        gk = torch.randn(rows, topk, generator=gen)
        out = K.token_logprobs(xg, topk=topk)
        d, = torch.autograd.grad(out.top_logprobs, xg, gk.to(DEV))
        R.check_logprobs(x, None, topk, 1.0, out, (None, None, gk), d)


@pytest.mark.parametrize("tail", ["renormalize", "bucket"])
def test_entries_marked_absent_by_any_number_below_zero(tail):
    # numbers whose low 32 bits are a token, or lie far outside the row
    gen = _gen(101)
    V, k = 9001, 8
    x = R.make_logits(4, V, BF, gen)
    tlp, tid = R.make_teacher(x, k, 1.0, gen)
    tid[0, 2:7] = torch.tensor([-2 ** 63, -2 ** 32, -2 ** 32 + 5,
                                -2 ** 31 - 1, -2 ** 31])
    tid[1, 0] = -2 ** 32 + int(tid[1, 1])   # a token that is listed, too
    tid[2] = -2 ** 31 - 1 - torch.arange(k)
    tid[3, 1:] = -2 ** 40 + torch.arange(1, k)
    g = torch.randn(4, generator=gen)
    loss, d = run_distill(x, tlp, tid, 1.0, tail, g)
    R.check_distill(x, tlp, tid, 1.0, tail, loss, d, g)
    assert loss[2] == 0 and (d[2] == 0).all()
    same, d2 = run_distill(x, tlp, tid.clamp(min=-1), 1.0, tail, g)
    assert torch.equal(loss, same) and torch.equal(d, d2)


def test_rows_without_a_gradient():
    check_rows_without_a_gradient(DEV)


@pytest.mark.parametrize("dtype,V", [(BF, 4096), (HF, 4096), (FP, 2048)])
def test_many_small_terms_beside_a_large_one(dtype, V):
    """One token has all of a row but V terms of e^-17, each below half a step
    of 1 in 32 bits: a sum in order would lose every one of its lane's."""
    x = torch.full((3, V), -17.0, dtype=dtype)
    tok = torch.tensor([0, V // 2 + 5, V - 1])
    x[torch.arange(3), tok] = 0.0
    want = torch.full((3,), -math.log1p((V - 1) * math.exp(-17.0)),
                      dtype=torch.float64)
    # of one vector at most N - 1 terms, 0.7 u each, then a rounding for each
    # of the lane's other 7 vectors and of the wave's 6 additions, beside which
    # the terms' own errors (of V e^-17 < 2e-4) are below 1 u
    N = 4 if dtype == FP else 8
    bound = (0.7 * (N - 1) + 7 + 6 + 1) * R.U
    assert 0.7 * (8 * N - 1) * R.U > bound   # what a sum in order loses
    out = K.token_logprobs(x.to(DEV), tok.to(DEV))
    R.assert_close(out.logprobs, want, bound, "logprobs")
    loss = K.topk_distillation(x.to(DEV), torch.zeros(3, 1, device=DEV),
                               tok[:, None].to(DEV))
    R.assert_close(loss, -want, bound, "loss")
