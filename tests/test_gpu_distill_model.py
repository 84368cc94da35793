"""UnifiedLM.distill's loss and the gradient that it gives the logits, against the definition in float64 of the same logits
(needs an MI355X)."""
import math

import pytest
import torch

from helpers import say, tiny_model
from test_gpu_distill import U, close, reference

pytestmark = pytest.mark.gpu

V = 97


def _batch(K=7, seed=5):
    gen = torch.Generator().manual_seed(seed)
    x, y = (torch.randint(0, V, (3, 29), generator=gen) for _ in range(2))
    y[torch.rand(3, 29, generator=gen) < 0.2] = -1
    ids = torch.rand(3, 29, V, generator=gen).argsort(-1)[..., :K]
    t = torch.log_softmax(torch.randn(3, 29, K, generator=gen), -1) - 0.2
    ids[0, 3], ids[1, 4, 2:] = -1, -1
    return x.cuda(), y.cuda(), ids.cuda(), t.cuda()


def _run(model, *args, **kw):
    """distill's loss, the logits that it saw and their gradient."""
    seen = []

    def keep(module, inputs, out):
        out.retain_grad()
        seen.append(out)
    hook = model.output.register_forward_hook(keep)
    model.zero_grad(set_to_none=True)
    loss = model.distill(*args, **kw)
    hook.remove()
    loss.backward()
    assert len(seen) == 1 and model.last_loss is loss
    return loss.detach(), seen[0].detach(), seen[0].grad


@pytest.mark.parametrize("labelled", [False, True])
@pytest.mark.parametrize("T,weight,rest", [(2.0, 0.7, False), (1.0, 0.5, True), (1.5, 0.0, False), (3.0, 1.0, True)])
def test_loss_and_logits_gradient(T, weight, rest, labelled):
    """fp32. Tolerances: the rows' own, weighted as the loss weights them; the sums of 87 rows add a unit a step, 87 in
    all, the quotients and weights 8 more; an upstream gradient is off by 8 units (products and quotients of counts), relatively."""
    say(f"distill of the model T={T} weight={weight} rest={rest} labelled={labelled}")
    model = tiny_model(4, dim=64, hidden_dim=96).cuda()
    x, y, ids, t = _batch()
    loss, logits, grad = _run(model, x, ids, t, y if labelled else None, T, weight, rest)
    on = (ids != -1).any(-1).cpu()
    up = [None, None]
    if labelled:
        counted = (y != -1).cpu()
        on &= counted
        up[1] = torch.full((3, 29), -(1 - weight) / counted.sum().item(), dtype=torch.float64) * counted
    share = (weight if labelled else 1.0) * T * T / on.sum().item()
    up[0] = on.double() * share
    want, tol = reference(logits, ids, t, y if labelled else None, T, rest, -1, up)
    terms, off = want[0] * up[0], tol[0] * up[0]
    if labelled:
        terms, off = terms + want[1] * up[1], off + tol[1] * up[1].abs()
        size = (want[0] * up[0]).abs() + (want[1] * up[1]).abs()
    else:
        size = terms.abs()
    assert abs(loss.item() - terms.sum().item()) <= U * (off + 96 * size).sum().item()
    p = torch.softmax(logits.double().cpu() / T, -1), torch.softmax(logits.double().cpu(), -1)
    each = up[0].abs()[..., None] / T * (p[0] + 1) + (0 if up[1] is None else up[1].abs()[..., None] * (p[1] + 1))
    close(grad, want[2], U * (tol[2] + 8 * each + want[2].abs()), "gradient")


@pytest.mark.parametrize("weight", [0.0, 0.3, 1.0])
def test_without_any_entry_the_text_still_teaches(weight):
    """No counted position has a teacher's entry: the teacher's part is 0, its gradient too, and the text's stays."""
    say(f"distill without entries weight={weight}")
    model = tiny_model(4, dim=64, hidden_dim=96).cuda()
    x, y, ids, t = _batch()
    none = torch.full_like(ids, -1)
    only_padding = torch.where((y == -1)[..., None], ids, -1)   # entries where no target counts
    for listed in (none, only_padding):
        loss, logits, grad = _run(model, x, listed, t, y, 2.0, weight)
        counted = y != -1
        own = logits.double().log_softmax(-1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
        want = -(1 - weight) * own[counted].sum() / counted.sum()
        assert abs(loss.item() - want.item()) <= 300 * U * (1 + abs(want.item()))   # 96 of the sums, 200 of a row's own
        at = torch.zeros_like(logits.double()).scatter_(-1, y.clamp(min=0)[..., None], 1.0)
        dx = (logits.double().softmax(-1) - at) * (counted * (1 - weight) / counted.sum())[..., None]
        assert (grad - dx).abs().max() <= 300 * U * (1 - weight) / counted.sum()
        text = model.loss(x, y)
        assert abs(loss.item() - (1 - weight) * text.item()) <= 300 * U * (1 + abs(text.item()))
    assert model.distill(x, none, t).isnan() and model.distill(x, ids, t, torch.full_like(y, -1)).isnan()
    assert not math.isnan(model.distill(x, ids, t).item())
