"""Drawing tokens and learning from a teacher's top logits together, as UnifiedLM and its callers use them (needs an
MI355X): on-policy distillation, the decode loops, other streams, threads, HIP graphs and torch.compile."""
import math
import threading

import pytest
import torch

from helpers import rel, say, tiny_model

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402


def _batch(B, T, V, seed, ignored=0.1):
    gen = torch.Generator().manual_seed(seed)
    x, y = (torch.randint(0, V, (B, T), generator=gen) for _ in range(2))
    y[torch.rand(B, T, generator=gen) < ignored] = -1
    return x.cuda(), y.cuda()


def test_on_policy_distillation():
    """The student draws, the teacher scores what was drawn, the student learns from the teacher's top logits; clipped
    and stepped. The loss and its gradient are those of their formula on the student's logits."""
    say("on-policy distillation")
    student, teacher = tiny_model(0).cuda().train(), tiny_model(1).cuda()
    opt = student.configure_optimizers(0.0, 1e-3, (0.9, 0.95), "cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    prompt, _ = _batch(4, 5, 97, 3)
    for k in range(3):
        tokens, logprob = student.sample(prompt, 20, temperature=0.9, top_p=0.95, generator=gen)
        assert tokens.shape == (4, 21) and logprob.shape == (4, 16) and (logprob <= 0).all()
        assert torch.equal(tokens[:, :5], prompt) and (tokens >= 0).all() and (tokens < 97).all()
        told = teacher.score(tokens, top=12)
        assert (told.top_logprobs.exp().sum(-1) < 1 + 1e-5).all()
        opt.zero_grad(set_to_none=True)
        loss = student.distill(tokens[:, :-1], told.top_tokens, told.top_logprobs, rest=True)
        assert student.last_loss is loss
        loss.backward()
        with torch.no_grad():
            logp = student(tokens[:, :-1], tokens[:, 1:]).double().log_softmax(-1)
            lq = told.top_logprobs.double()
            listed = torch.zeros_like(logp).scatter_(-1, told.top_tokens, 1.0) > 0
            qr = 1 - lq.exp().sum(-1)
            lpr = logp.masked_fill(listed, -math.inf).logsumexp(-1)
            want = ((lq.exp() * (lq - logp.gather(-1, told.top_tokens))).sum(-1) + qr * (qr.log() - lpr)).mean()
        # the two forwards give one student's logits; fp32 sums of some hundred positions
        assert abs(loss.item() - want.item()) <= 1e-5 * (1 + abs(want.item()))
        assert all(p.grad is not None and p.grad.isfinite().all() for p in student.parameters())
        assert all(p.grad is None for p in teacher.parameters())
        before = {n: p.detach().clone() for n, p in student.named_parameters()}
        student.clip_grad_norm_(1.0)
        opt.step()
        assert any(not torch.equal(p, before[n]) for n, p in student.named_parameters())


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_against_its_formula(rest, autocast):
    """UnifiedLM.distill's loss and gradients against the formula in fp32 (float64 for the loss) of forward's logits.
    Under autocast the logits' gradients round to bf16 on both sides (2^-8 of each), as in the loss's own test."""
    say(f"distill against its formula rest={rest} autocast={autocast}")
    model = tiny_model(4, dim=64, hidden_dim=96).cuda()
    x, y = _batch(3, 29, 97, 5)
    gen = torch.Generator().manual_seed(6)
    ids = torch.rand(3, 29, 97, generator=gen).argsort(-1)[..., :7].cuda()
    t = torch.randn(3, 29, 7, generator=gen).cuda()
    T, weight = 2.0, 0.7
    if rest:
        t = torch.log_softmax(t, -1) - 0.2
    ids[0, 3], ids[1, 4, 2:] = -1, -1

    def formula(logits):
        there = ids != -1
        logp = (logits / T).log_softmax(-1)
        at = ids.clamp(min=0)
        z = (t if rest else t / T).to(logits.dtype).masked_fill(~there, -1e30)
        lq = z if rest else z.log_softmax(-1)
        q = torch.where(there, lq.exp(), 0.0)
        loss = (q * (torch.where(there, lq, 0.0) - logp.gather(-1, at))).sum(-1)
        if rest:
            listed = torch.zeros(logits.shape, device="cuda").scatter_add_(-1, at, there.float()) > 0
            qr = (1 - q.sum(-1)).clamp(min=0)
            loss = loss + qr * (qr.log() - logp.masked_fill(listed, -math.inf).logsumexp(-1))
        counted = y != -1
        on = there.any(-1) & counted
        own = logits.log_softmax(-1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
        return weight * T * T * loss[on].sum() / on.sum() - (1 - weight) * own[counted].sum() / counted.sum()
    res = []
    for own in (False, True):
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            if own:
                loss = model.distill(x, ids, t, y, T, weight, rest)
            else:
                logits = model(x, y)
        if not own:
            loss = formula(logits.float())
            want = formula(logits.detach().double()).item()
        loss.backward()
        res.append({n: p.grad.clone() for n, p in model.named_parameters()})
    assert abs(loss.item() - want) <= 256 * 2.0 ** -24 * (1 + abs(want))
    for n, g in res[0].items():
        assert rel(res[1][n], g) <= 1e-2, n
    assert model.distill(x, torch.full_like(ids, -1), t).isnan()
    assert model.distill(x, ids, t, torch.full_like(y, -1)).isnan()


def test_distill_of_a_padded_batch():
    """Targets of -1 leave a position out for the teacher too: what its entries hold changes neither loss nor gradients."""
    say("distill of a padded batch")
    model = tiny_model(4, dim=64, hidden_dim=96).cuda()
    x, y = _batch(3, 29, 97, 5)
    y = torch.where(torch.arange(29, device="cuda") < torch.tensor([[29], [11], [1]], device="cuda"), y, -1)
    gen = torch.Generator().manual_seed(6)
    ids = torch.rand(3, 29, 97, generator=gen).argsort(-1)[..., :7].cuda()
    t = torch.randn(3, 29, 7, generator=gen).cuda()
    res = []
    for fill in (None, math.nan):
        v, i = t.clone(), ids.clone()
        if fill is not None:
            v[y == -1] = fill
            i[2, 5:] = 97
        model.zero_grad(set_to_none=True)
        loss = model.distill(x, i, v, y, temperature=2.0)
        loss.backward()
        res.append([loss.detach()] + [p.grad.clone() for p in model.parameters()])
    assert all(a.isfinite().all() and torch.equal(a, b) for a, b in zip(*res))


def test_a_teacher_equal_to_the_student_teaches_nothing():
    """The whole vocabulary listed, the student's own logits: loss 0 and no gradient, to rounding."""
    say("a teacher equal to the student")
    gen = torch.Generator().manual_seed(7)
    x = (torch.randn(30, 60, generator=gen) * 3).cuda().requires_grad_(True)
    ids = torch.arange(60).expand(30, 60).cuda()
    for T in (1.0, 3.0):
        out = kernel.distillation(x, ids, x.detach(), temperature=T)
        g, = torch.autograd.grad(out.loss.sum(), x)
        # differences of two roundings of one number: the units of either, times the share
        assert out.loss.abs().max() <= 2.0 ** -24 * 400 and g.abs().max() <= 2.0 ** -24 * 200


def test_sample_loops():
    """sample at temperature 0 is decode_greedy; the given numbers fix the tokens; a step's draw is kernel.sample_tokens'."""
    say("UnifiedLM.sample and generate")
    model = tiny_model(8).cuda()
    prompt, _ = _batch(3, 6, 97, 9)
    for prefill in (True, False):
        toks, lp = model.sample(prompt, 25, temperature=0.0, prefill=prefill)
        assert torch.equal(toks, model.decode_greedy(prompt, 25, prefill)) and not lp.any()
    gen = torch.Generator(device="cuda").manual_seed(10)
    u = torch.rand(20, 3, device="cuda", generator=gen)
    how = dict(temperature=torch.tensor([0.7, 1.0, 0.0]).cuda(), top_k=torch.tensor([0, 20, 0]).cuda(), top_p=0.9)
    a, la = model.sample(prompt, 25, u=u, **how)
    b, lb = model.sample(prompt, 25, u=u, **how)
    assert torch.equal(a, b) and torch.equal(la, lb)
    logits, states = model.prefill(prompt)
    for i in range(20):
        one = kernel.sample_tokens(logits, u[i], **how)
        assert torch.equal(one.token, a[:, 6 + i]) and torch.equal(one.logprob, la[:, i])
        if i < 19:
            logits = model.step(one.token, states)
    gen.manual_seed(11)
    c = model.sample(prompt, 25, generator=gen)
    gen.manual_seed(11)
    assert torch.equal(c[0], model.sample(prompt, 25, u=torch.rand(20, 3, device="cuda", generator=gen))[0])
    torch.manual_seed(12)
    g = model.generate(prompt, 9, top_p=1e-9)
    assert torch.equal(g, model.generate(prompt, 9, temperature=0.0))
    torch.manual_seed(12)
    old = model.generate(prompt, 9, top_k=10)   # as before: through torch.multinomial
    torch.manual_seed(12)
    want, states = prompt, None
    logits, states = model.prefill(prompt)
    for _ in range(9):
        nxt = model._sample(logits.float(), 1.0, 10)
        want = torch.cat((want, nxt), 1)
        logits = model.step(nxt[:, 0], states)
    assert torch.equal(old, want)
    torch.manual_seed(13)
    assert model.generate(prompt, 60, temperature=0.8, top_k=5, top_p=0.9, min_p=0.01).shape == (3, 66)   # past the window


def test_sequences_that_cannot_go_on():
    """Logits that are no numbers: tokens -1 with log probability NaN, and no lookup of row -1."""
    say("UnifiedLM.sample of logits with NaN")
    model = tiny_model(14).cuda()
    prompt, _ = _batch(2, 5, 96, 15)
    with torch.no_grad():
        model.output.weight[96, 3] = math.nan
    toks, lp = model.sample(prompt, 12, top_k=5)
    assert (toks[:, 5:] == -1).all() and lp.isnan().all() and torch.equal(toks[:, :5], prompt)
    out = model.generate(prompt, 4, top_p=0.9)
    assert (out[:, 5:] == 0).all()
    torch.cuda.synchronize()


def _inputs(seed, rows=200, V=3001, K=20):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    u = torch.rand(rows, device="cuda", generator=gen)
    ids = torch.rand(rows, V, device="cuda", generator=gen).topk(K).indices
    t = torch.log_softmax(f(rows, K), -1) - 0.3
    tok = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    return f(rows, V) * 3, u, ids, t, tok, f(rows), f(rows), torch.rand(rows, device="cuda", generator=gen)


def _calls(x, u, ids, t, tok, da, db, T):
    """One of each, and the backward's entry."""
    a = kernel.sample_tokens(x, u, T, 50, 0.9)
    b = kernel.sample_tokens(x, u)
    c = kernel.distill_fwd(x, ids, t, tok, 2.0, True, -1)
    d = kernel.distillation(x, ids, t, temperature=1.5)
    g = kernel.distill_bwd(x, ids, t, tok, 2.0, True, -1, c[2], da, db)
    return [*a, *b, *c, d.loss, g]


def test_on_another_stream():
    say("drawing and distilling on another stream")
    want = [t.clone() for t in _calls(*_inputs(11))]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        fresh = _inputs(11)   # made there as well: nothing of it is ordered after the default stream
        got = _calls(*fresh)
        leaf = fresh[0].clone().requires_grad_(True)
        out = kernel.distillation(leaf, *fresh[2:5], 2.0, True)
        got.append(torch.autograd.grad(list(out), leaf, list(fresh[5:7]))[0])
    torch.cuda.current_stream().wait_stream(side)
    want.append(want[-1])
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


def test_from_two_threads():
    say("drawing and distilling from two threads at once")
    inputs = [_inputs(13), _inputs(17, rows=700, V=999)]
    want = [[t.clone() for t in _calls(*a)] for a in inputs]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = _calls(*inputs[k])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        bad.append(k)
        except Exception as e:   # noqa: BLE001 - reported below
            bad.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_graph_replays_equal_eager():
    """Captured once, two graphs of them, replayed in turns with eager work between."""
    say("drawing and distilling in HIP graphs")
    static = [_inputs(19), _inputs(23, rows=2, V=50000)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in static:
            _calls(*a)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for a in static:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_calls(*a))
    for rep in range(3):
        fresh = [_inputs(29 + rep), _inputs(31 + rep, rows=2, V=50000)]
        want = [[t.clone() for t in _calls(*a)] for a in fresh]
        for s, f in zip(static, fresh):
            for to, frm in zip(s, f):
                to.copy_(frm)
        for g in graphs if rep % 2 == 0 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            for i, (a, b) in enumerate(zip(outs[k], want[k])):
                assert torch.equal(a, b), (rep, k, i)


def test_backward_in_a_graph_of_its_own_leaves():
    """A forward and its backward captured on leaves that no eager graph holds; one that an eager graph holds is refused."""
    say("distilling: captured backward")
    x0, _, ids, t, tok, da, db, _ = _inputs(43)

    def step(x):
        out = kernel.distillation(x, ids, t, tok, 2.0)
        return [o.detach() for o in out] + list(torch.autograd.grad(list(out), x, [da, db]))
    want = [o.clone() for o in step(x0.clone().requires_grad_(True))]
    x = x0.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x)
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep
        assert all(torch.equal(a, b) for a, b in zip(step(x0.clone().requires_grad_(True)), want)), rep
    leaf = x0.clone().requires_grad_(True)
    held = kernel.distillation(leaf, ids, t).loss   # an eager graph of the leaf, on the default stream
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(other):
            kernel.distillation(leaf, ids, t)
    assert held.requires_grad


@pytest.mark.parametrize("backend", ["aot_eager"])
def test_compiled(backend):
    say(f"drawing and distilling under torch.compile {backend}")
    torch._dynamo.reset()
    x0, u, ids, t, tok, da, db, T = _inputs(37)

    def step(x):
        out = kernel.distillation(x, ids, t, tok, 2.0, True)
        only = kernel.distillation(x, ids, t)
        drawn = kernel.sample_tokens(x.detach(), u, T, 50, 0.9)
        return out.loss.sum() + (out.logprob * da).sum() + only.loss.mean(), *drawn
    res = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        x = x0.clone().requires_grad_(True)
        loss, *drawn = f(x)
        res.append([loss, *drawn, *torch.autograd.grad(loss, x)])
    for a, b in zip(*res):
        assert torch.equal(a, b) if not a.is_floating_point() else rel(b, a) <= 1e-5


def test_left_to_the_registered_ops():
    """Calls that the host module does not take give what it gives."""
    say("drawing and distilling: registered ops against the host module")
    x0, u, ids, t, tok, da, db, T = _inputs(41)
    for rest in (False, True):
        x = x0.clone().requires_grad_(True)
        a, b = kernel.distillation(x, ids, t, tok, 2.0, rest), kernel.distill_fwd(x, ids, t, tok, 2.0, rest, -1)
        ga, gb = (torch.autograd.grad([o[0], o[1]], x, [da, db]) for o in (a, b))
        assert torch.equal(ga[0], gb[0]) and torch.equal(a.loss, b[0]) and torch.equal(a.logprob, b[1])
        a, b = kernel.distillation(x, ids, t, None, 2.0, rest), kernel.distill_fwd(x, ids, t, None, 2.0, rest, -1)
        ga, gb = (torch.autograd.grad(o[0], x, da) for o in (a, b))
        assert torch.equal(ga[0], gb[0]) and a.logprob is None and b[1].shape == (0,)
    k = torch.full_like(tok, 30)
    a = kernel.sample_tokens(x0, u, T, k, 0.9, 0.01)
    b = kernel.sample_tokens_op(x0, u, 0.0, 0, 0.9, 0.01, T, k, None, None)
    assert all(torch.equal(s, q) for s, q in zip(a, b))

    class Sub(torch.Tensor):
        pass
    assert torch.equal(kernel.distillation(x0.as_subclass(Sub), ids, t).loss.as_subclass(torch.Tensor),
                       kernel.distillation(x0, ids, t).loss)
    assert torch.equal(kernel.sample_tokens(x0.as_subclass(Sub), u).token.as_subclass(torch.Tensor),
                       kernel.sample_tokens(x0, u).token)
    with torch.inference_mode():
        assert torch.equal(kernel.sample_tokens(x0, u, T).token, kernel.sample_tokens(x0, u, T).token)
        assert kernel.distillation(x0, ids, t).loss.shape == (200,)
    y = x0.clone().requires_grad_(True)
    g, = torch.autograd.grad(kernel.distillation(y, ids, t).loss.sum(), y, create_graph=True)
    with pytest.raises(RuntimeError):   # no second derivative
        torch.autograd.grad(g.square().sum(), y)
