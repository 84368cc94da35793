"""A leaf that an eager graph on another stream holds is refused while a call is captured, on the registered ops' path
as on the host module's (needs an MI355X). Only forwards are captured here."""
import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402


class Own(torch.nn.Parameter):
    """A parameter that the host module leaves to the registered ops."""


def _calls(kind):
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 50, (7,), generator=gen).cuda()
    if kind == "embedding":
        return torch.randn(50, 12, generator=gen).cuda(), lambda w: kernel.embedding(w, tokens)
    return torch.randn(7, 50, generator=gen).cuda(), lambda x: kernel.token_logprobs(x, tokens, 2).logprob


@pytest.mark.parametrize("leaf_type", [torch.nn.Parameter, Own])
@pytest.mark.parametrize("kind", ["embedding", "token_logprobs"])
def test_held_leaf(kind, leaf_type):
    say(f"capture of {kind} of a held {leaf_type.__name__}")
    data, call = _calls(kind)
    leaf = leaf_type(data)
    held = call(leaf)                       # an eager graph, on the default stream
    assert held.requires_grad
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call(leaf)
    want = held.detach().as_subclass(torch.Tensor).clone()
    del held                                # let go: captured, with and without gradients
    for grad in (True, False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.set_grad_enabled(grad):
            out = call(leaf).detach()
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.as_subclass(torch.Tensor), want)
            assert torch.equal(call(leaf).detach().as_subclass(torch.Tensor), want)


@pytest.mark.parametrize("leaf_type", [torch.nn.Parameter, Own])
@pytest.mark.parametrize("kind", ["embedding", "token_logprobs"])
def test_without_gradients_a_held_leaf_is_captured(kind, leaf_type):
    say(f"capture of {kind} of a held {leaf_type.__name__} without gradients")
    data, call = _calls(kind)
    leaf = leaf_type(data)
    held = call(leaf)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        out = call(leaf)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.as_subclass(torch.Tensor), held.detach().as_subclass(torch.Tensor))
