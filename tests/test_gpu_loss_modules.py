"""UnifiedLM.loss and score with hooks on the token embedding, or another module in its place: what runs in forward
runs there (needs an MI355X)."""
import pytest
import torch
import torch.nn as nn

from helpers import rel, say, tiny_model

pytestmark = pytest.mark.gpu


def _batch(seed, B=2, T=21, V=97):
    gen = torch.Generator().manual_seed(seed)
    x, y = torch.randint(0, V, (2, B, T), generator=gen).cuda()
    y[0, ::5] = -1
    return x, y


def _check(model, x, y):
    """loss and score against the float64 cross-entropy of forward's logits, the embedding's gradient against
    forward's: sums of fp32 terms in another order, 2^-24 each, beside bf16 roundings that the difference tips."""
    model.zero_grad(set_to_none=True)
    logits = model(x, y)
    model.last_loss.backward()
    want, grad = logits.detach().double(), model.output.weight.grad.clone()
    model.zero_grad(set_to_none=True)
    loss = model.loss(x, y)
    loss.backward()
    ce = nn.functional.cross_entropy(want.flatten(0, 1), y.flatten(), ignore_index=-1).item()
    assert abs(loss.item() - ce) <= 64 * 2.0 ** -24 * ce
    assert rel(model.output.weight.grad, grad) <= 1e-2
    lp = want.log_softmax(-1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
    lp = torch.where(y == -1, torch.zeros_like(lp), lp)
    assert (model.score(x, y).logprob - lp).abs().max() <= 64 * 2.0 ** -24 * (1 + lp.abs().max())


def test_forward_hooks():
    say("loss with hooks on the embedding")
    model = tiny_model(1).cuda()
    x, y = _batch(1)
    plain = model.loss(x, y).item()
    for register in (lambda e: e.register_forward_hook(lambda m, i, o: 3 * o),
                     lambda e: e.register_forward_pre_hook(lambda m, i: (i[0].flip(-1),))):
        hook = register(model.tok_embeddings)
        _check(model, x, y)
        assert abs(model.loss(x, y).item() - plain) > 1e-3 * plain
        hook.remove()
        assert model.loss(x, y).item() == plain


def test_backward_hook():
    say("loss with a backward hook on the embedding")
    model = tiny_model(2).cuda()
    x, y = _batch(2)
    seen = []
    model.tok_embeddings.register_full_backward_hook(lambda m, gi, go: seen.append(go[0].shape))
    model.loss(x, y).backward()
    assert seen == [(2, 21, 32)]


def test_hook_of_every_module():
    say("loss with a hook of every module")
    model = tiny_model(3).cuda()
    x, y = _batch(3)
    seen = []
    handle = nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(type(m)))
    try:
        model.loss(x, y)
    finally:
        handle.remove()
    assert nn.Embedding in seen


@pytest.mark.parametrize("kind", ["subclass", "padding", "own forward", "module"])
def test_another_embedding(kind):
    say(f"loss with another embedding: {kind}")
    model = tiny_model(4).cuda()
    x, y = _batch(4)
    tied = model.output.weight
    if kind == "subclass":
        class Scaled(nn.Embedding):
            def forward(self, tokens):
                return 0.5 * super().forward(tokens)
        model.tok_embeddings = Scaled(97, 32, _weight=tied.detach())
    elif kind == "padding":
        x[:, ::3] = 5   # whose row then has no gradient from here
        model.tok_embeddings = nn.Embedding(97, 32, padding_idx=5, _weight=tied.detach())
    elif kind == "own forward":
        model.tok_embeddings.forward = lambda tokens: nn.functional.embedding(tokens.flip(0), tied)
    else:
        class Rows(nn.Module):
            def __init__(self):
                super().__init__()
                self.rows = tied

            def forward(self, tokens):
                return self.rows[tokens] + 0.25
        model.tok_embeddings = Rows()
    if hasattr(model.tok_embeddings, "weight"):
        model.tok_embeddings.weight = tied
    _check(model, x, y)


@pytest.mark.parametrize("hooked", [False, True])
def test_compiled_loss(hooked):
    say(f"loss under torch.compile, hooked={hooked}")
    torch._dynamo.reset()
    model = tiny_model(5).cuda()
    x, y = _batch(5)
    if hooked:
        model.tok_embeddings.register_forward_hook(lambda m, i, o: 2 * o)
    model(x, y)
    want = model.last_loss.item()
    got = torch.compile(model.loss, backend="aot_eager")(x, y)
    assert abs(got.item() - want) <= 64 * 2.0 ** -24 * want
