"""embedding (ulm_embed_fwd / ulm_embed_bwd) against its definition (needs an MI355X).

The lookup is one fp32 product rounded to the type: equal to torch's bits. A row of the gradient is
a sum of n fp32 terms, each addition off by 2^-24 of the partial sum, which the sum of the
terms' sizes bounds; scaling and the rounding to the type (half a step) come on top."""
import math

import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def check(weight, tokens, scale, dout=None):
    w = weight.detach().requires_grad_(True)
    out = kernel.embedding(w, tokens, scale)
    V, D = weight.shape
    known = (tokens >= 0) & (tokens < V)
    want = (weight[torch.where(known, tokens, 0)].float() * torch.tensor(scale, dtype=torch.float32)).to(weight.dtype)
    want[~known] = math.nan
    assert out.dtype == weight.dtype and out.shape == (*tokens.shape, D)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(), want.nan_to_num())
    if dout is None:
        return out
    g, = torch.autograd.grad(out, w, dout)
    assert g.dtype == weight.dtype and g.shape == weight.shape
    d = dout.double().reshape(-1, D)[known.flatten()]
    t = tokens.flatten().long()[known.flatten()]
    f = lambda x: torch.zeros(V, D, device="cuda", dtype=torch.float64).index_add_(0, t, x)  # noqa: E731
    ref, size = f(d) * scale, f(d.abs()) * abs(scale)
    n = torch.bincount(t, minlength=V)[:, None]
    half = torch.finfo(weight.dtype).eps / 2
    tiny = 2.0 ** -25 if weight.dtype == torch.float16 else 2.0 ** -126
    tol = U * (n + 2) * size
    assert ((g.double() - ref).abs() <= tol + half * (ref.abs() + tol) + tiny).all()
    assert (g[n[:, 0] == 0] == 0).all()
    h, = torch.autograd.grad(kernel.embedding(w, tokens, scale), w, dout)
    assert torch.equal(g, h)
    return out


def make(N, V, D, dt, seed, skew=0.0):
    gen = torch.Generator().manual_seed(seed)
    weight = torch.randn(V, D, generator=gen).to(DT[dt]).cuda()
    if skew:
        p = 1.0 / (torch.arange(V) + 2.0) ** skew
        tokens = torch.multinomial(p, N, replacement=True, generator=gen).cuda()
    else:
        tokens = torch.randint(0, V, (N,), generator=gen).cuda()
    return weight, tokens, torch.randn(N, D, generator=gen).to(DT[dt]).cuda()


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 33, 7), (2, 2, 4), (31, 5, 255), (32, 5, 256), (33, 5, 257), (64, 1024, 8),
                                   (1000, 1023, 63), (1000, 1025, 512), (4096, 40, 96), (4097, 3000, 289), (5000, 1, 33),
                                   (9000, 32000, 64), (300, 70000, 40), (200, 1100000, 3)])
def test_lookup_and_gradient(N, V, D, dt):
    say(f"embedding N={N} V={V} D={D} {dt}")
    weight, tokens, dout = make(N, V, D, dt, N + V + D)
    check(weight, tokens, 1.0, dout)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("N,V,D,skew", [(16384, 4000, 130, 1.0), (20000, 300, 64, 1.5), (70000, 2000, 40, 1.0),
                                        (131073, 33, 24, 0.0)])
def test_frequent_tokens(N, V, D, skew, dt):
    say(f"embedding N={N} V={V} D={D} skew={skew} {dt}")
    weight, tokens, dout = make(N, V, D, dt, 3, skew)
    check(weight, tokens, math.sqrt(D), dout)


@pytest.mark.parametrize("N,V,where", [(10000, 1000, 0), (10000, 1000, 511), (10000, 1000, 512), (10000, 1000, 999),
                                       (10000, 5000, 4999), (32768, 32767, 32766), (32769, 32767, 7), (20000, 40000, 39999)])
def test_one_token_throughout(N, V, where):
    """All rows one token, but for another at the first or last place: runs over every chunk."""
    say(f"embedding one token throughout, N={N} V={V}, at {where}")
    weight, tokens, dout = make(N, V, 48, "fp32", 5)
    tokens.fill_(where)
    check(weight, tokens, 0.5, dout)
    tokens[0], tokens[-1] = 3, 998
    check(weight, tokens, 0.5, dout)


def test_every_token_once_in_any_order():
    say("embedding a permutation")
    weight, _, dout = make(4096, 4096, 20, "fp32", 7)
    tokens = torch.randperm(4096, generator=torch.Generator().manual_seed(8)).cuda()
    w = weight.requires_grad_(True)
    g, = torch.autograd.grad(kernel.embedding(w, tokens), w, dout)
    assert torch.equal(g[tokens], dout)   # sums of one term


def test_sums_go_in_the_order_of_the_positions():
    """Terms of 2^24 and 1: their fp32 sum depends on the order, which is the positions', 16 sorted
    rows at a time in a short sequence, and then those sums'."""
    say("embedding order of the sums")
    weight, tokens, dout = make(24, 3, 4, "fp32", 9)
    tokens.copy_(torch.tensor([2, 0] * 12))
    dout.fill_(1.0)
    dout[4], dout[20] = 2.0 ** 24, -2.0 ** 24
    w = weight.requires_grad_(True)
    g, = torch.autograd.grad(kernel.embedding(w, tokens), w, dout)
    parts = [torch.zeros(4), torch.zeros(4)]   # token 2's rows are the sorted ones from the 12th on
    for k, n in enumerate(range(0, 24, 2)):
        parts[(12 + k) // 16] += dout[n].cpu()
    assert torch.equal(g[2].cpu(), parts[0] + parts[1]) and (g[0] == 12).all() and (g[1] == 0).all()


@pytest.mark.parametrize("V", [1023, 1024, 5000, 32767, 32768])   # a digit, a digit and one, one launch's most, and one more
@pytest.mark.parametrize("N", [50, 5000, 40000])
def test_unknown_tokens(N, V):
    say(f"embedding unknown tokens N={N} V={V}")
    weight, tokens, dout = make(N, V, 33, "fp32", 11)
    tokens[0], tokens[5], tokens[7], tokens[N - 1] = -1, V, V - 1, 1 << 40
    check(weight, tokens, 2.0, dout)
    tokens.fill_(-100)
    check(weight, tokens, 1.0, dout)


def test_nan_and_infinity_stay_in_their_rows():
    say("embedding NaN and infinities")
    weight, tokens, dout = make(3000, 500, 16, "fp32", 13)
    tokens[100], tokens[200] = 7, 8
    dout[100, 3], dout[200, 4] = math.nan, math.inf
    w = weight.requires_grad_(True)
    g, = torch.autograd.grad(kernel.embedding(w, tokens), w, dout)
    assert g[7, 3].isnan() and g[8, 4].isinf()
    g[7, 3], g[8, 4] = 0, 0
    assert g.isfinite().all()


def test_views_types_and_shapes():
    say("embedding views")
    weight, tokens, dout = make(60, 50, 24, "fp32", 17)
    check(weight.t().contiguous().t(), tokens, 1.0, dout)
    check(torch.randn(51, 48, device="cuda")[1:, ::2], tokens.view(5, 12).t(), 1.5, dout.view(5, 12, 24).transpose(0, 1))
    check(weight, tokens.view(3, 4, 5), 1.0, dout[:, :1].expand(60, 24).view(3, 4, 5, 24))
    check(weight, tokens[0], 1.0, dout[0])
    check(weight.flatten()[:49 * 24].view(49, 24), tokens[:0], 1.0, dout[:0])
    check(torch.randn(1201, device="cuda")[1:].view(50, 24), tokens.to(torch.int32), 1.0, dout)
    a = kernel.embedding(weight, tokens)
    assert torch.equal(a, kernel.embedding(weight, tokens.to(torch.int16))) and not a.requires_grad


def test_offsets_past_32_bits():
    say("embedding weight and rows past 2^32 bytes")
    V, D = 1100000, 1024   # 4.5 GB
    weight = torch.empty(V, D, device="cuda")
    weight[-3:] = torch.randn(3, D, device="cuda")
    tokens = torch.tensor([V - 1, V - 3, V - 1, V - 2], device="cuda")
    w = weight.requires_grad_(True)
    out = kernel.embedding(w, tokens)
    assert torch.equal(out, weight.detach()[tokens])
    d = torch.randn(4, D, device="cuda")
    g, = torch.autograd.grad(out, w, d)
    assert torch.equal(g[-3:], torch.stack([d[1], d[3], d[0] + d[2]]))
    assert not g[:-3].any()
    del g, out, w, weight
    N = 1100000   # rows past 2^32 bytes, every token once but one
    tokens = torch.arange(N, device="cuda") % 1000
    w = torch.randn(1000, D, device="cuda").requires_grad_(True)
    out = kernel.embedding(w, tokens)
    assert torch.equal(out[-5:], w.detach()[tokens[-5:]])
    d = torch.zeros(N, D, device="cuda")
    d[-1], d[0] = 3.0, 5.0
    g, = torch.autograd.grad(out, w, d)
    assert (g[999] == 3).all() and (g[0] == 5).all() and not g[1:999].any()


def test_gradient_against_differences():
    say("embedding gradient against differences")
    weight, tokens, dout = make(40, 9, 5, "fp32", 19)
    w = weight.requires_grad_(True)
    g, = torch.autograd.grad(kernel.embedding(w, tokens, 1.25), w, dout)
    value = lambda z: (z[tokens].mul(1.25) * dout.double()).sum()  # noqa: E731
    v = torch.randn(9, 5, device="cuda", dtype=torch.float64)
    slope = (value(weight.double() + v) - value(weight.double() - v)) / 2   # linear: exact but for 2^-53
    assert abs((g.double() * v).sum() - slope) <= 1e-5 * (g.double() * v).abs().sum()


def test_refusals():
    say("embedding refusals")
    weight, tokens, _ = make(4, 5, 6, "fp32", 23)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.embedding(weight, tokens.cpu())
    with pytest.raises(TypeError):
        kernel.embedding(weight.double(), tokens)
