"""The embedding, the token log probabilities and the clipping together, as UnifiedLM and its
callers use them (needs an MI355X): the loss and its gradients against the forward's, scoring
against decoding, a training step, other streams, threads, HIP graphs and torch.compile."""
import math
import threading

import pytest
import torch

from helpers import rel, say, tiny_model

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402


def _model(seed=0, **kw):
    return tiny_model(seed, **kw).cuda()


def _batch(B, T, V, seed, ignored=0.1):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(0, V, (B, T), generator=gen)
    y = torch.randint(0, V, (B, T), generator=gen)
    y[torch.rand(B, T, generator=gen) < ignored] = -1
    return x.cuda(), y.cuda()


@pytest.mark.parametrize("autocast", [False, True])
def test_loss_is_the_forwards(autocast):
    """UnifiedLM.loss against the float64 cross-entropy of forward's logits, and its gradients against
    those of their cross-entropy in fp32 (under autocast F.cross_entropy itself is coarser). The logits'
    gradients then differ by roundings of fp32 sums, which tip one in some thousand of the bf16 roundings
    that follow, 2^-8 of its value each."""
    say(f"loss against forward, autocast={autocast}")
    model = _model(dim=64, hidden_dim=96)
    x, y = _batch(3, 37, 97, 1)
    res = []
    for own in (False, True):
        model.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            if own:
                loss = model.loss(x, y)
                assert model.last_loss is loss
            else:
                logits = model(x, y)
                loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1).float(), y.flatten(), ignore_index=-1)
        loss.backward()
        res.append((loss.item(), {n: p.grad.clone() for n, p in model.named_parameters()}))
    want = torch.nn.functional.cross_entropy(logits.flatten(0, 1).double(), y.flatten(), ignore_index=-1).item()
    assert abs(want - res[1][0]) <= 64 * 2.0 ** -24 * want
    for n, g in res[0][1].items():
        assert rel(res[1][1][n], g) <= 1e-2, n


def test_loss_with_entropy():
    say("loss with an entropy bonus")
    model = _model()
    x, y = _batch(2, 30, 97, 2)
    with torch.no_grad():
        logp = model(x, y).double().log_softmax(-1)
    on = y != -1
    H = -(logp.exp() * logp).sum(-1)[on].mean()
    want = -logp.gather(-1, y.clamp(min=0)[..., None])[..., 0][on].mean() - 0.3 * H
    assert abs(model.loss(x, y, 0.3).item() - want.item()) <= 1e-6 * abs(want.item())
    assert model.loss(x, torch.full_like(y, -1)).isnan()
    with pytest.raises(ValueError, match="shape"):
        model.loss(x, y[:, :-1])


def test_score_against_decoding():
    """Scores of a prompt's own tokens are those of decoding it token by token, alternatives included."""
    say("score against decoding")
    model = _model(3)
    x, _ = _batch(3, 20, 97, 4)
    out = model.score(x, top=5)
    assert out.logprob.shape == (3, 19) and out.top_tokens.shape == (3, 19, 5) and not out.logprob.requires_grad
    states = model.init_states(3, x.device)
    for t in range(19):
        logits = model.step(x[:, t], states)
        one = kernel.token_logprobs(logits, x[:, t + 1], 5)
        # the block's two forms agree to bf16 roundings of their operands (2^-8 and less)
        assert (one.logprob - out.logprob[:, t]).abs().max() <= 2e-2 * (1 + one.logprob.abs().max())
        assert (one.entropy - out.entropy[:, t]).abs().max() <= 2e-2 * (1 + math.log(97))
        assert torch.equal(one.top_tokens[:, 0], logits.argmax(-1))
    y = torch.where(torch.arange(20, device="cuda") < 7, x.roll(-1, 1), -1)
    given = model.score(x, y)
    assert torch.equal(given.logprob[:, :7], out.logprob[:, :7]) and not given.logprob[:, 7:].any()
    assert model.score(x[:, :1]).logprob.shape == (3, 0) and model.score(x[:0]).logprob.shape == (0, 19)
    logits = model(x[:, :-1], x[:, 1:].contiguous()).double().log_softmax(-1)
    want = logits.gather(-1, x[:, 1:, None])[..., 0]
    assert (out.logprob - want).abs().max() <= 64 * 2.0 ** -24 * (1 + want.abs().max())


def test_a_training_step():
    """Loss, backward, clipping and an optimizer's step in a row; the clipped gradients are the gradients
    times the factor, and every parameter moves."""
    say("training step")
    model = _model(5).train()
    opt = model.configure_optimizers(0.1, 1e-3, (0.9, 0.95), "cuda")
    for k in range(3):
        x, y = _batch(4, 24, 97, 6 + k)
        opt.zero_grad(set_to_none=True)
        model.loss(x, y).backward()
        grads = {n: p.grad.clone() for n, p in model.named_parameters()}
        want = math.sqrt(sum(g.double().square().sum().item() for g in grads.values()))
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        norm = model.clip_grad_norm_(want / 2)
        assert abs(norm.item() - want) <= 2.0 ** -23 * want
        coef = want / 2 / (want + 1e-6)
        for n, p in model.named_parameters():
            assert ((p.grad.double() - grads[n].double() * coef).abs() <= 6 * 2.0 ** -24 * grads[n].double().abs() + 2.0 ** -126).all(), n
        opt.step()
        assert all(not torch.equal(p, before[n]) for n, p in model.named_parameters() if grads[n].any())
    assert model.clip_grad_norm_(1e9, float("inf")) == max(p.grad.abs().max() for p in model.parameters())


def test_gradients_of_a_step_against_differences():
    """d loss along random directions of the embedding against differences of the loss in float64 of the same
    embedding and loss (the blocks left out: a linear layer stands for them)."""
    say("embedding and loss against differences")
    gen = torch.Generator().manual_seed(8)
    W = torch.randn(50, 12, generator=gen)
    A = torch.randn(12, 12, generator=gen) * 0.5
    x, y = _batch(2, 15, 50, 9)
    w = W.cuda().requires_grad_(True)
    out = kernel.token_logprobs(kernel.embedding(w, x, 0.7) @ A.cuda() @ w.t(), y)
    loss = -out.logprob.sum() / (y != -1).sum() + 0.1 * out.entropy.mean()
    g, = torch.autograd.grad(loss, w)

    def value(z):
        logp = ((z[x.cpu()] * 0.7) @ A.double() @ z.t()).log_softmax(-1)
        on = y.cpu() != -1
        return (-logp.gather(-1, y.cpu().clamp(min=0)[..., None])[..., 0][on].mean()
                + 0.1 * -(logp.exp() * logp).sum(-1).mean())
    for _ in range(4):
        v = torch.randn(50, 12, generator=gen, dtype=torch.float64)
        slope = (value(W.double() + 1e-5 * v) - value(W.double() - 1e-5 * v)) / 2e-5
        got = (g.double().cpu() * v).sum()
        assert abs(got - slope) <= 1e-5 * (g.double().cpu() * v).abs().sum() + 1e-8


def _calls(logits, tokens, weight, dout, grads, out):
    """One of each, forward only."""
    a = kernel.token_logprobs(logits, tokens, 3)
    e = kernel.embedding(weight, tokens, 1.5)
    dw = kernel.embed_bwd(dout, tokens, weight.shape[0], 1.5)
    dx = kernel.token_logprobs_bwd(logits, tokens, 0, -1, stats=torch.stack([logits.amax(-1), (logits - logits.amax(-1, True)).exp()
                                                                               .sum(-1).log()], -1),
                                   entropy=a.entropy, top_tokens=a.top_tokens, dlogprob=a.entropy, dentropy=None, dtop=None)
    n, o = kernel.clip_grads(grads, 0.5, out=out)
    return [*a, e, dw, dx, n, *o]


def _inputs(seed, rows=200, V=3001, D=40):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    grads = [f(300, 41), f(7), f(9000)]
    return f(rows, V) * 3, tokens, f(V, D), f(rows, D), grads, [torch.empty_like(g) for g in grads]


def test_on_another_stream():
    say("step ends on another stream")
    args = _inputs(11)
    want = [t.clone() for t in _calls(*args)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fresh = _inputs(11)   # made there as well: nothing of it is ordered after the default stream
        got = _calls(*fresh)
        leaf = fresh[2].clone().requires_grad_(True)
        g, = torch.autograd.grad(kernel.embedding(leaf, fresh[1], 1.5), leaf, fresh[3])
        got.append(g)
    torch.cuda.current_stream().wait_stream(side)
    want.append(want[5])
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


def test_from_two_threads():
    say("step ends from two threads at once")
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
    """Every forward and the C backwards captured once, two graphs of them, replayed in turns with eager work between."""
    say("step ends in HIP graphs")
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
        want = [[t.clone() for t in _calls(*a)] for a in fresh]   # the program's own eager work
        for s, f in zip(static, fresh):
            for to, frm in zip((*s[:4], *s[4]), (*f[:4], *f[4])):
                to.copy_(frm)
        for g in graphs if rep % 2 == 0 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for k in range(2):
            for i, (a, b) in enumerate(zip(outs[k], want[k])):
                assert torch.equal(a, b), (rep, k, i)


@pytest.mark.parametrize("backend", ["aot_eager"])
def test_compiled(backend):
    say(f"step ends under torch.compile {backend}")
    torch._dynamo.reset()
    logits, tokens, weight, dout, grads, out = _inputs(37)

    def step(x, w):
        a = kernel.token_logprobs(x, tokens, 3)
        e = kernel.embedding(w, tokens, 1.5)
        return a.logprob.sum() + a.entropy.mean() + a.top_logprobs.sum(), (e * dout).sum(), a.top_tokens
    res = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        x, w = logits.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        p, q, ids = f(x, w)
        res.append([p, q, ids, *torch.autograd.grad(p + q, (x, w))])
    for a, b in zip(*res):
        assert torch.equal(a, b) if not a.is_floating_point() else rel(b, a) <= 1e-5

    def clip(*g):
        g = [t * 2 for t in g]
        n, o = kernel.clip_grads(g, 0.5)
        m = kernel.clip_grads(g, 0.25, out=g)[0]
        return kernel.grad_norm(o), n, m, *o, *g
    for a, b in zip(clip(*grads), torch.compile(clip, backend=backend, fullgraph=True)(*grads)):
        assert torch.equal(a, b)


def test_left_to_the_registered_ops():
    """Calls that the host module does not take give what it gives."""
    say("step ends: registered ops against the host module")
    logits, tokens, weight, dout, grads, out = _inputs(41)
    x = logits.clone().requires_grad_(True)
    a, b = kernel.token_logprobs(x, tokens, 3), kernel.token_logprobs_fwd(x, tokens, 3, -1)
    ups = [torch.randn_like(t) for t in a[:3]]
    ga, gb = (torch.autograd.grad(list(o[:3]), x, ups) for o in (a, b))
    assert torch.equal(ga[0], gb[0]) and all(torch.equal(s, t) for s, t in zip(a, b))
    w = weight.clone().requires_grad_(True)
    ga, gb = (torch.autograd.grad(f, w, dout) for f in (kernel.embedding(w, tokens, 1.5), kernel.embed_fwd(w, tokens, 1.5)))
    assert torch.equal(ga[0], gb[0])
    n, o = kernel.clip_grads(grads, 0.5)
    out = [torch.empty_like(g) for g in grads]
    assert torch.equal(kernel._clip_op(grads, out, 0.5, 2.0), n) and all(torch.equal(s, t) for s, t in zip(o, out))
    assert torch.equal(kernel._grad_norm_op(grads, 2.0), n)
    # written in place: autograd sees it
    v = out[0]._version
    kernel.clip_grads(grads, 0.5, out=out)
    assert out[0]._version > v
    y = torch.randn(5, device="cuda", requires_grad=True)
    z = (y * 2).square()
    kept = torch.ones(5, device="cuda")
    s = (z * kept).sum()
    kernel.clip_grads([kept], 0.1, out=[kept])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        s.backward()

    class Sub(torch.Tensor):
        pass
    assert torch.equal(kernel.token_logprobs(logits.as_subclass(Sub), tokens).logprob.as_subclass(torch.Tensor),
                       kernel.token_logprobs(logits, tokens).logprob)


def test_backward_in_a_graph_of_its_own_leaves():
    """A forward and its backward captured on leaves that no eager graph holds; one that an eager graph holds is refused."""
    say("step ends: captured backward")
    logits, tokens, weight, dout, _, _ = _inputs(43)

    def step(x, w):
        a = kernel.token_logprobs(x, tokens, 3)
        e = kernel.embedding(w, tokens, 1.5)
        g = torch.autograd.grad([a.logprob, a.entropy, e], [x, w], [a.entropy.detach(), a.logprob.detach(), dout])
        return [t.detach() for t in (*a, e, *g)]
    want = [t.clone() for t in step(logits.clone().requires_grad_(True), weight.clone().requires_grad_(True))]
    x, w = logits.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, w)
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep
        again = step(logits.clone().requires_grad_(True), weight.clone().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(again, want)), rep
    leaf = weight.clone().requires_grad_(True)
    held = kernel.embedding(leaf, tokens)   # an eager graph of the leaf, on the default stream
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(other):
            kernel.embedding(leaf, tokens)
    assert held.requires_grad
