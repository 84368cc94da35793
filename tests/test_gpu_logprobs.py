"""token_logprobs (ulm_token_logprobs / _bwd) against its definition in float64 (needs an MI355X).

Tolerances, in units of 2^-24 (half a step of fp32): a row's sum of exponentials is off by at most
V/256 additions per thread and a few more to join them, each exponent by two roundings of d = x - m
(weighted by p they come to 2 ln V), the exponential and logarithm by a few units. ln s, and with
it every log probability, is then off by (V/256 + 2 ln V + 32) units absolutely, a log probability
by 4 |logprob| more. The gradient's G = a + sum_j c_j is a sum of top + 1 fp32 terms, off by at
most top units of |a| + sum_j |c_j|, whatever cancels in it. Every output rounds to its own type
by half a step."""
import math

import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def units(V):
    return V / 256 + 2 * math.log(V + 1) + 32


def reference(logits, tokens, top, ignore=-1, up=(None, None, None)):
    """The definition in float64: outputs, the gradient, and what its tolerance is made of."""
    x = logits.detach().double().cpu()
    t = tokens.cpu()
    V = x.shape[-1]
    m = x.amax(-1, keepdim=True)
    empty = (m == -math.inf)
    d = torch.where(empty, torch.full_like(x, -math.inf), x - m)
    s = d.exp().sum(-1, keepdim=True)
    logp = torch.where(empty, torch.full_like(x, -math.inf), d - s.log())
    p = torch.where(empty, torch.zeros_like(x), logp.exp())
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    H = -plogp.sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    known = (t >= 0) & (t < V)
    at = torch.where(known, t, torch.zeros_like(t))[..., None]
    lp = logp.gather(-1, at)[..., 0]
    lp = torch.where(known, lp, torch.full_like(lp, math.nan))
    lp = torch.where(t == ignore, torch.zeros_like(lp), lp)
    outs = (lp, H, logp.gather(-1, ids), ids)
    a, h, c = (None if u is None else u.double().cpu() for u in up)
    zero = torch.zeros_like(lp)
    a = zero if a is None else a
    a = torch.where(t == ignore, zero, torch.where(known, a, torch.full_like(a, math.nan)))
    G = a if c is None else a + c.sum(-1)
    f = G[..., None].expand_as(x)
    if h is not None:
        f = f + h[..., None] * torch.where(p == 0, torch.zeros_like(p), logp + H[..., None])
    dx = -p * f
    dx = dx.scatter_add(-1, at, torch.where(t == ignore, zero, a)[..., None])
    size = (p * f.abs()).scatter_add(-1, at, a.abs()[..., None])
    if c is not None:
        dx = dx.scatter_add(-1, ids, c)
        size = size.scatter_add(-1, ids, c.abs())
    if h is not None:   # H and ln p are off themselves
        size = size + p * h.abs()[..., None] * (1 + 2 * math.log(V + 1))
    if c is not None:   # G's own additions; what follows multiplies size by more than 1
        size = size + p * (top * (a.abs() + c.abs().sum(-1)) / (units(V) + 8))[..., None]
    dx, size = (torch.where(empty, torch.zeros_like(x), y) for y in (dx, size))
    depth = torch.where(p == 0, torch.zeros_like(p), -logp)
    return outs, dx, (size * (units(V) + 8 + 4 * depth))


def close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    ok = ~(nan | inf)
    err = (got - want).abs()[ok] - (tol.double().expand_as(want)[ok] if isinstance(tol, torch.Tensor) else tol)
    assert err.numel() == 0 or err.max().item() <= 0, (what, err.max().item())


def check(logits, tokens, top=0, ignore=-1, up=(None, None, None)):
    V, dt = logits.shape[-1], logits.dtype
    x = logits.detach().requires_grad_(True)
    out = kernel.token_logprobs(x, tokens, top, ignore)
    outs, dx, scale = reference(logits, tokens, top, ignore, up)
    n = units(V)
    close(out.logprob, outs[0], U * (n + 4 * outs[0].nan_to_num(0, 0, 0).abs()), "logprob")
    close(out.entropy, outs[1], U * 3 * n * (1 + math.log(V + 1)), "entropy")
    close(out.top_logprobs, outs[2], U * (n + 4 * outs[2].nan_to_num(0, 0, 0).abs()), "top_logprobs")
    assert torch.equal(out.top_tokens.cpu(), outs[3]), "top_tokens"
    assert out.top_tokens.dtype == torch.int64 and out.logprob.dtype == torch.float32
    used = [(o, u) for o, u in zip(out, up) if u is not None]
    if used:
        got, = torch.autograd.grad([o for o, _ in used], [x], [u for _, u in used])
        assert got.dtype == dt and got.shape == logits.shape
        half = torch.finfo(dt).eps / 2
        close(got, dx, U * scale + half * (dx.abs() + U * scale) + TINY[dt], "dlogits")
    return out


def make(rows, V, dt, seed, std=3.0):
    gen = torch.Generator().manual_seed(seed)
    shape = (rows,) if isinstance(rows, int) else rows
    logits = (torch.randn(*shape, V, generator=gen) * std).to(DT[dt]).cuda()
    tokens = torch.randint(0, V, shape, generator=gen).cuda()
    return logits, tokens, gen


def ups(gen, shape, top, which="aht"):
    f = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    return (f(*shape) if "a" in which else None, f(*shape) if "h" in which else None,
            f(*shape, top) if "t" in which and top else None)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 2, 2), (3, 7, 3), (5, 63, 63), (2, 64, 64), (700, 65, 5), (1, 1000, 0),
                                        (4, 2047, 20), (3, 4096, 1), (2, 8191, 64), (2, 8193, 7), (1, 32000, 5),
                                        (513, 3001, 3), (600, 8200, 0), (6, 50001, 64)])
def test_outputs_and_gradient(rows, V, top, dt):
    say(f"token_logprobs rows={rows} V={V} top={top} {dt}")
    logits, tokens, gen = make(rows, V, dt, rows + V)
    check(logits, tokens, top, up=ups(gen, (rows,), top))


@pytest.mark.parametrize("which", ["a", "h", "t", "ah", "at", "ht"])
def test_gradient_of_some_outputs(which):
    say(f"token_logprobs gradients of {which}")
    logits, tokens, gen = make(40, 777, "bf16", 3)
    check(logits, tokens, 4, up=ups(gen, (40,), 4, which))


@pytest.mark.parametrize("rows", [3, 600])
def test_ignored_and_unknown_tokens(rows):
    say(f"token_logprobs ignored and unknown tokens rows={rows}")
    logits, tokens, gen = make(rows, 300, "fp32", 5)
    tokens[0] = -1
    tokens[1] = 300
    check(logits, tokens, 2, up=ups(gen, (rows,), 2))
    tokens[1] = -2
    check(logits, tokens, 2, up=ups(gen, (rows,), 2))
    tokens[1], tokens[2] = 7, 7
    check(logits, tokens, 0, ignore=7, up=ups(gen, (rows,), 0, "a"))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [4, 520])
def test_masks(rows, dt):
    """-inf and the type's lowest value in masked places, rows with one or no entry left."""
    say(f"token_logprobs masks rows={rows} {dt}")
    V = 5000
    logits, tokens, gen = make(rows, V, dt, 11)
    hide = torch.rand(rows, V, generator=gen).cuda() < 0.7
    for value in (-math.inf, torch.finfo(DT[dt]).min):
        x = logits.masked_fill(hide, value)
        x[0] = value                                 # nothing left
        x[1] = value
        x[1, 4321] = 1.5                             # one entry left
        tokens[1] = 4321
        x[2, :V - 1] = value                         # the last entry left; the token itself masked
        tokens[2] = 17
        check(x, tokens, 6, up=ups(gen, (rows,), 6))
        x[0, 0], tokens[0] = value, -1
        check(x, tokens, 1, up=ups(gen, (rows,), 1, "at"))


@pytest.mark.parametrize("rows", [2, 512])
def test_nan_and_infinity_stay_in_their_rows(rows):
    say(f"token_logprobs NaN and infinities rows={rows}")
    logits, tokens, _ = make(rows, 9000, "fp32", 13)
    clean = kernel.token_logprobs(logits, tokens, 5)
    logits[0, 8888] = math.nan
    out = kernel.token_logprobs(logits, tokens, 5)
    assert out.logprob[0].isnan() and out.entropy[0].isnan() and out.top_logprobs[0].isnan().all()
    assert out.top_tokens[0, 0] == 8888 and torch.equal(out.top_tokens[0, 1:], clean.top_tokens[0, :4])
    for a, b in zip(out, clean):
        assert torch.equal(a[1:], b[1:])
    logits[0, 8888] = math.inf
    out = kernel.token_logprobs(logits, tokens, 5)
    assert out.logprob[0].isnan() and out.entropy[0].isnan() and out.top_tokens[0, 0] == 8888
    logits[0] = math.nan
    out = kernel.token_logprobs(logits, tokens, 5)
    assert out.logprob[0].isnan() and out.top_tokens[0].tolist() == [0, 1, 2, 3, 4]
    x = logits.clone().requires_grad_(True)
    g, = torch.autograd.grad(kernel.token_logprobs(x, tokens).logprob.sum(), x)
    assert g[0].isnan().all() and g[1:].isfinite().all()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [2, 514])
def test_ties_go_to_the_lower_index(rows, dt):
    say(f"token_logprobs ties rows={rows} {dt}")
    logits, tokens, gen = make(rows, 20000, dt, 17)
    logits = logits.round()   # a dozen distinct values
    logits[0] = 0.0
    logits[0, ::2] = -0.0     # one value
    check(logits, tokens, 64, up=ups(gen, (rows,), 64, "at"))


@pytest.mark.parametrize("dt,V,vec", [("bf16", 131072, 8), ("fp32", 65536, 4)])
@pytest.mark.parametrize("order", ["rising", "falling", "equal"])
def test_largest_entries_all_in_a_few_threads(dt, V, vec, order):
    """More candidates than the list holds: the large entries lie where only a few threads read."""
    say(f"token_logprobs crowded candidates {dt} {order}")
    rows = 513
    logits, tokens, _ = make(rows, V, dt, 19, std=0.5)
    where = torch.nonzero((torch.arange(V) // vec) % 64 < 8).flatten().cuda()
    n = where.numel()
    rise = torch.linspace(4, 30, n).cuda()
    logits[:, where] = {"rising": rise, "falling": rise.flip(0), "equal": torch.full_like(rise, 9.0)}[order].to(DT[dt])
    out = kernel.token_logprobs(logits, tokens, 64)
    for r in (0, rows - 1):
        ids = torch.sort(logits[r].float(), descending=True, stable=True).indices[:64]
        assert torch.equal(out.top_tokens[r], ids)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 2100])
def test_many_ties_at_the_last_place(rows, dt):
    """The top-th entry is one of thousands of equal ones, spread or at the row's end, with or without larger ones."""
    say(f"token_logprobs thousands of ties rows={rows} {dt}")
    V = 40000
    logits, tokens, gen = make(rows, V, dt, 53, std=0.1)
    logits.clamp_(max=0.0)          # half of them 0
    logits[0, :V - 700] = -3.0      # equal ones at the end only
    if rows > 1:
        logits[1, torch.randperm(V, generator=gen)[:40].cuda()] = 2.5
        logits[2] = -math.inf
        logits[2, [5, 39999]] = 1.0
        tokens[2] = 5
    for top in (1, 17, 64):
        out = kernel.token_logprobs(logits, tokens, top)
        ids = torch.sort(logits[:3].float().cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(out.top_tokens[:3].cpu(), ids)


@pytest.mark.parametrize("rows", [1, 2100])
def test_wide_rows_are_joined_from_parts(rows):
    """More columns than one workgroup's table holds."""
    say(f"token_logprobs wide rows={rows}")
    gen = torch.Generator(device="cuda").manual_seed(59)
    V = 200001 if rows == 1 else 70001
    logits = torch.randn(rows, V, device="cuda", generator=gen) * 2
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=gen)
    logits[0, V - 1] = 20.0
    out = kernel.token_logprobs(logits, tokens, 20)
    few = logits[:2].contiguous()
    want, _, _ = reference(few, tokens[:2], 20)
    assert torch.equal(out.top_tokens[:2].cpu(), want[3])
    n = units(V)
    close(out.logprob[:2], want[0], U * (n + 4 * want[0].abs()), "logprob")
    close(out.top_logprobs[:2], want[2], U * (n + 4 * want[2].abs()), "top_logprobs")
    close(out.entropy[:2], want[1], U * 3 * n * (1 + math.log(V + 1)), "entropy")


def _views(V, dt):
    gen = torch.Generator().manual_seed(23)
    f = lambda *s: (torch.randn(*s, generator=gen) * 2).to(DT[dt]).cuda()  # noqa: E731
    return {"ahead": f(3, 9, V)[:, :-1], "column": f(4, 5, V)[:, 2], "swapped": f(5, 3, V).transpose(0, 1),
            "wider": f(6, V + 3)[:, 1:V + 1], "three": f(2, 5, 3, V)[:, 1:4, :2], "expanded": f(1, V).expand(7, V),
            "every other": f(6, 2 * V)[:, ::2], "row": f(V), "none": f(0, V), "no rows": f(4, 0, 3, V)}


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("view", ["ahead", "column", "swapped", "wider", "three", "expanded", "every other", "row", "none",
                                  "no rows"])
def test_views(view, dt):
    say(f"token_logprobs view {view} {dt}")
    x = _views(333, dt)[view]
    gen = torch.Generator().manual_seed(29)
    tokens = torch.randint(0, 333, x.shape[:-1], generator=gen).cuda()
    check(x, tokens, 3, up=ups(gen, x.shape[:-1], 3))
    if tokens.dim() == 2 and tokens.numel():   # ids of another integer type, in another order
        a = kernel.token_logprobs(x, tokens, 3)
        b = kernel.token_logprobs(x, tokens.t().contiguous().t().to(torch.int32), 3)
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 5), (2, 3, 4), (600, 2)])
def test_rows_repeated_over_a_leading_dimension(shape, dt):
    """One block of rows expanded in front: the rows' outer stride is 0."""
    say(f"token_logprobs expanded leading dimension {shape} {dt}")
    gen = torch.Generator().manual_seed(43)
    V = 333
    x = (torch.randn(1, *shape[1:], V, generator=gen) * 2).to(DT[dt]).cuda().expand(*shape, V)
    assert x.stride(0) == 0
    tokens = torch.randint(0, V, shape, generator=gen).cuda()
    check(x, tokens, 3, up=ups(gen, shape, 3))
    a, b = kernel.token_logprobs(x, tokens, 3), kernel.token_logprobs(x.contiguous(), tokens, 3)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_a_row_does_not_depend_on_the_others():
    """Equal bits however many rows come along, as long as they take workgroups of one size (more than 512 rows)."""
    say("token_logprobs rows alone")
    logits, tokens, _ = make(4096, 4001, "bf16", 31)
    a, b = kernel.token_logprobs(logits, tokens, 4), kernel.token_logprobs(logits[1024:], tokens[1024:], 4)
    assert all(torch.equal(s[1024:], t) for s, t in zip(a, b))
    c = kernel.token_logprobs(logits, tokens, 4)
    assert all(torch.equal(s, t) for s, t in zip(a, c))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_more_rows_than_one_grid_dimension_counts(dt):
    """2^20 + 1537 rows, a block of 1024 over and over: every copy has the first one's bits, its gradients too."""
    say(f"token_logprobs rows past 2^20 {dt}")
    rows, V, top = (1 << 20) + 1537, 27, 2
    block, some, gen = make(1024, V, dt, 47)
    a, h, c = ups(gen, (1024,), top)
    out = check(block, some, top, up=(a, h, c))
    again = lambda t: t.repeat(1026, *[1] * (t.dim() - 1))[:rows]  # noqa: E731
    x = again(block).requires_grad_(True)
    many = kernel.token_logprobs(x, again(some), top)
    assert all(torch.equal(m, again(o)) for m, o in zip(many, out))
    for upstream in ((a,), (a, h, c)):   # a vector a thread, and two
        y = block.requires_grad_(True)
        want, = torch.autograd.grad(kernel.token_logprobs(y, some, top)[:len(upstream)], y, upstream)
        got, = torch.autograd.grad(many[:len(upstream)], x, [again(u) for u in upstream], retain_graph=True)
        assert torch.equal(got, again(want))


def test_offsets_past_32_bits():
    say("token_logprobs rows past 2^32 bytes and 2^31 elements")
    rows, V = 70000, 32000
    logits = torch.empty(rows, V, device="cuda", dtype=torch.bfloat16)   # 4.5 GB, 2.24e9 elements
    logits[:-2] = 0
    gen = torch.Generator().manual_seed(37)
    last = (torch.randn(2, V, generator=gen) * 3).to(torch.bfloat16).cuda()
    logits[-2:] = last
    tokens = torch.randint(0, V, (rows,), generator=gen).cuda()
    x = logits.requires_grad_(True)
    out = kernel.token_logprobs(x, tokens, 2)
    few = kernel.token_logprobs(last.repeat(1050, 1), tokens[-2:].repeat(1050), 2)   # workgroups of the same size
    assert all(torch.equal(a[-2:], b[:2]) for a, b in zip(out, few))
    assert (out.logprob[:-2] + math.log(V)).abs().max() <= U * (units(V) + 44)
    g, = torch.autograd.grad(out.logprob.sum(), x)
    y = last.clone().requires_grad_(True)
    h, = torch.autograd.grad(kernel.token_logprobs(y.repeat(1050, 1), tokens[-2:].repeat(1050), 2).logprob[:2].sum(), y)
    assert torch.equal(g[-2:], h)


def test_gradient_against_differences():
    """Central differences of the float64 definition along random directions."""
    say("token_logprobs gradient against differences")
    logits, tokens, gen = make(6, 501, "fp32", 41)
    up = ups(gen, (6,), 3)
    x = logits.clone().requires_grad_(True)
    out = kernel.token_logprobs(x, tokens, 3)
    g, = torch.autograd.grad(list(out[:3]), [x], list(up))
    value = lambda z: sum((o * u.double().cpu()).sum() for o, u in zip(reference(z, tokens, 3)[0][:3], up))  # noqa: E731
    for k in range(4):
        v = torch.randn(6, 501, generator=gen, dtype=torch.float64)
        step = 1e-5
        z = logits.double().cpu()
        slope = (value(z + step * v) - value(z - step * v)) / (2 * step)
        got = (g.double().cpu() * v).sum()
        # the difference quotient is off by step^2 and by 1e-16 / step
        assert abs(got - slope) <= 1e-6 * (g.double().cpu().abs() * v.abs()).sum() + 1e-8


def test_gradient_of_an_expanded_upstream_and_twice():
    say("token_logprobs upstream views, two backwards")
    logits, tokens, _ = make(30, 200, "fp32", 43)
    x = logits.clone().requires_grad_(True)
    out = kernel.token_logprobs(x, tokens)
    a, = torch.autograd.grad(out.logprob.sum(), x, retain_graph=True)   # an expanded gradient
    b, = torch.autograd.grad(out.logprob, x, torch.ones(30, device="cuda"))
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError):   # no second derivative
        g, = torch.autograd.grad(kernel.token_logprobs(x, tokens).logprob.sum(), x, create_graph=True)
        torch.autograd.grad(g.square().sum(), x)


def test_refusals():
    say("token_logprobs refusals")
    logits, tokens, _ = make(4, 50, "fp32", 47)
    with pytest.raises(TypeError):
        kernel.token_logprobs(logits.double(), tokens)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.token_logprobs(logits, tokens.cpu())
    with pytest.raises(ValueError, match="top"):
        kernel.token_logprobs(logits, tokens, 51)
