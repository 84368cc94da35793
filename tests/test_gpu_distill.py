"""distillation (ulm_distill / _bwd) against its definition in float64 (needs an MI355X).

Tolerances, in units of 2^-24 (half a step of fp32). A row's sum of exponentials adds at most V/256 + 64 terms in a
thread and a few more to join them; each exponent is off by three roundings of d / T (difference, product, log2(e) / T;
weighted by p they come to 3 ln V), the exponential by 2 and a logarithm by a few: ln s by n(V) = V/256 + 3 ln V + 80. A
log probability is off by that and 4 (|ln p| + ln V) for its own d / T. ln q of the teacher's K entries likewise by
n(K); with the rest it is the given value, and q_r, formed in double, is rounded once. The loss adds
its terms in K/64 + 8 steps. A probability is off by its logarithm's error and 4 more, relatively. Every output
rounds to its own type by half a step."""
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
    return V / 256 + 3 * math.log(V + 1) + 80


def nz(t):
    """Infinities and NaN as 0, for tolerances."""
    return t.nan_to_num(0.0, 0.0, 0.0)


def reference(logits, ids, values, tokens, T, rest, ignore=-1, up=(None, None)):
    """The definition in float64 on the CPU: (loss, logprob, dlogits) and their tolerances (without the outputs'
    own roundings)."""
    x = logits.detach().double().cpu()
    ids, t = ids.cpu().long(), values.detach().double().cpu()
    V, K = x.shape[-1], ids.shape[-1]
    x, ids, t = x.reshape(-1, V), ids.reshape(-1, K), t.reshape(-1, K)
    there = (ids >= 0) & (ids < V)
    broken = ((ids != -1) & ~there).any(-1)
    at = torch.where(there, ids, torch.zeros_like(ids))
    empty = (x == -math.inf).all(-1)
    logp = torch.where(empty[:, None], torch.full_like(x, -math.inf), torch.log_softmax(x / T, -1))
    p = torch.where(empty[:, None], torch.zeros_like(x), logp.exp())
    lp = logp.gather(-1, at)
    z = torch.where(there, t if rest else t / T, torch.full_like(t, -math.inf))
    if rest:
        lq, nq = z, 6.0
    else:
        none = (z == -math.inf).all(-1, keepdim=True)
        lq, nq = torch.where(none, z, torch.log_softmax(z, -1)), units(K)
    q = lq.exp()
    term = torch.where(q == 0, torch.zeros_like(q), q * (lq - lp))
    elp = units(V) + 4 * (nz(lp).abs() + math.log(V + 1))        # of ln p
    elq = nq + 4 * (nz(lq).abs() + math.log(K + 1))              # of ln q, and of q relatively
    loss = term.sum(-1)
    tol = (q * (elp + elq) + nz(term).abs() * (elq + K / 64 + 8)).sum(-1)
    listed = torch.zeros_like(x)
    listed.scatter_add_(-1, at, there.double())
    qj = torch.zeros_like(x).scatter_add_(-1, at, torch.where(there, q, torch.zeros_like(q)))
    eqj = torch.zeros_like(x).scatter_add_(-1, at, torch.where(there, q * (elq + 4), torch.zeros_like(q)))
    ep = p * (units(V) + 8 + 4 * (nz(logp).abs() + math.log(V + 1)))   # of p, absolutely
    g = torch.zeros(x.shape[0], dtype=torch.float64) if up[0] is None else up[0].double().cpu().reshape(-1)
    Q = q.sum(-1, keepdim=True)
    if rest:
        qr = torch.where(there.any(-1, keepdim=True), (1 - Q).clamp(min=0), torch.zeros_like(Q))
        others = torch.where(listed > 0, torch.zeros_like(p), p)
        pr = others.sum(-1, keepdim=True)
        lpr = torch.where(listed > 0, torch.full_like(x, -math.inf), logp).logsumexp(-1, keepdim=True)
        more = torch.where(qr == 0, torch.zeros_like(qr), qr * (qr.log() - lpr))
        elpr = 2 * units(V) + 4 * (nz(lpr).abs() + math.log(V + 1))
        loss = loss + more[:, 0]
        tol = tol + (qr * (elpr + 4 * nz(qr.log()).abs() + 8) + nz(more).abs() * 8 + 2 * (1 + nz(qr.log() - lpr).abs()))[:, 0]
        Q = Q + qr
        z = torch.where(listed > 0, torch.full_like(x, -math.inf), x / T)   # not p / p_r: both may be below float64's range
        share = torch.where((z == -math.inf).all(-1, keepdim=True), torch.zeros_like(p), torch.softmax(z, -1))
        dx = torch.where(listed > 0, Q * p - qj, share * (Q * pr - qr))
        size = torch.where(listed > 0, Q * ep + eqj + p * 8,
                           share * (Q * pr * (elpr + 8) + 8 * qr + 8 + (Q * pr - qr).abs() *
                                    (units(V) + 8 + 4 * (nz(share.log()).abs() + math.log(V + 1)))))
    else:
        dx, size = Q * p - qj, Q * ep + eqj
    dx, size = dx * g[:, None] / T, (size + dx.abs() * 8) * g.abs()[:, None] / T
    tol = tol + 4 * nz(loss).abs()
    logprob = lptol = None
    if tokens is not None:
        tok = tokens.cpu().long().reshape(-1)
        known = (tok >= 0) & (tok < V)
        own = torch.where(known, tok, torch.zeros_like(tok))[:, None]
        logp1 = torch.where(empty[:, None], torch.full_like(x, -math.inf), torch.log_softmax(x, -1))
        p1 = torch.where(empty[:, None], torch.zeros_like(x), logp1.exp())
        logprob = torch.where(known, logp1.gather(-1, own)[:, 0], torch.full_like(g, math.nan))
        logprob = torch.where(tok == ignore, torch.zeros_like(g), logprob)
        lptol = units(V) + 4 * nz(logprob).abs()
        a = torch.zeros_like(g) if up[1] is None else up[1].double().cpu().reshape(-1)
        a = torch.where(tok == ignore, torch.zeros_like(a), torch.where(known, a, torch.full_like(a, math.nan)))
        dx = dx - p1 * a[:, None]
        size = size + p1 * nz(a).abs()[:, None] * (units(V) + 8 + 4 * (nz(logp1).abs() + math.log(V + 1)))
        dx = dx.scatter_add(-1, own, torch.where(tok == ignore, torch.zeros_like(a), a)[:, None])
        size = size.scatter_add(-1, own, 4 * nz(a).abs()[:, None])
    loss = torch.where(broken, torch.full_like(loss, math.nan), loss)
    dx = torch.where((broken & ~empty)[:, None], torch.full_like(dx, math.nan), dx)
    dx, size = (torch.where(empty[:, None], torch.zeros_like(s), s) for s in (dx, size))
    lead = logits.shape[:-1]
    shaped = lambda s: None if s is None else s.reshape((*lead, *s.shape[1:]))  # noqa: E731
    return [shaped(s) for s in (loss, logprob, dx)], [shaped(s) for s in (tol, lptol, size)]


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    ok = ~(nan | inf)
    err = (got - want).abs()[ok] - tol.expand_as(want)[ok]
    assert err.numel() == 0 or err.max().item() <= 0, (what, err.max().item(), (got - want).abs()[ok].max().item())


def check(logits, ids, values, tokens=None, T=1.0, rest=False, ignore=-1, up=(None, None)):
    dt = logits.dtype
    x = logits.detach().requires_grad_(True)
    out = kernel.distillation(x, ids, values, tokens, T, rest, ignore)
    want, tol = reference(logits, ids, values, tokens, T, rest, ignore, up)
    assert out.loss.dtype == torch.float32
    close(out.loss, want[0], U * tol[0], "loss")
    outs = [out.loss]
    if tokens is None:
        assert out.logprob is None
    else:
        close(out.logprob, want[1], U * tol[1], "logprob")
        outs.append(out.logprob)
    used = [(o, u) for o, u in zip(outs, up) if u is not None]
    if used:
        got, = torch.autograd.grad([o for o, _ in used], [x], [u for _, u in used])
        assert got.dtype == dt and got.shape == logits.shape
        half = torch.finfo(dt).eps / 2
        close(got, want[2], U * tol[2] + half * (nz(want[2]).abs() + U * tol[2]) + TINY[dt], "dlogits")
        with torch.no_grad():
            again = kernel.distillation(logits, ids, values, tokens, T, rest, ignore)
        assert torch.equal(again.loss.nan_to_num(7), out.loss.detach().nan_to_num(7))
    return out


def make(lead, V, K, dt, seed, rest=False, T=1.0, tdt="fp32", std=2.0, absent=0.0):
    """A student, a teacher's distinct entries whose first few the student knows, tokens and upstream gradients."""
    gen = torch.Generator().manual_seed(seed)
    lead = (lead,) if isinstance(lead, int) else lead
    x = torch.randn(*lead, V, generator=gen) * std
    ids = torch.rand(*lead, V, generator=gen).argsort(-1)[..., :K]
    t = torch.randn(*lead, K, generator=gen) * 2
    x.scatter_add_(-1, ids[..., :3], 4 + torch.rand(*ids[..., :3].shape, generator=gen))
    if rest:
        t = torch.log_softmax(t / T, -1) + torch.log(0.5 + 0.49 * torch.rand(*lead, 1, generator=gen))
    if absent:
        ids = torch.where(torch.rand(ids.shape, generator=gen) < absent, -1, ids)
    tokens = torch.randint(0, V, lead, generator=gen)
    up = (torch.randn(lead, generator=gen).cuda(), torch.randn(lead, generator=gen).cuda())
    return x.to(DT[dt]).cuda(), ids.cuda(), t.to(DT[tdt]).cuda(), tokens.cuda(), up


SIZES = [(1, 1, 1), (1, 2, 1), (3, 7, 7), (5, 63, 20), (2, 64, 64), (700, 65, 5), (3, 511, 1), (2, 2047, 65), (3, 4096, 64),
         (2, 8193, 100), (1, 32000, 64), (513, 3001, 16), (4, 50001, 300), (2, 2100, 1024)]


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,V,K", SIZES)
def test_loss_and_gradient(rows, V, K, dt):
    say(f"distillation rows={rows} V={V} K={K} {dt}")
    x, ids, t, _, up = make(rows, V, K, dt, rows + V)
    check(x, ids, t, up=(up[0], None))
    check(x, ids, t, T=2.5, up=(up[0], None))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,V,K", SIZES)
def test_with_the_rest(rows, V, K, dt):
    say(f"distillation with the rest rows={rows} V={V} K={K} {dt}")
    for T in (1.0, 0.7):
        x, ids, t, _, up = make(rows, V, K, dt, rows + V + 1, rest=True, T=T)
        check(x, ids, t, T=T, rest=True, up=(up[0], None))


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [1.0, 2.0, 3.0])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("which", ["both", "loss", "logprob"])
def test_with_tokens(rest, T, which, dt):
    """The row's own token beside the teacher, at its own temperature; gradients of either output or both."""
    say(f"distillation with tokens rest={rest} T={T} {which} {dt}")
    x, ids, t, tokens, up = make((4, 9), 1003, 12, dt, 3, rest, T)
    tokens[0, 0], tokens[1, 2], tokens[2, 3] = -1, ids[1, 2, 0], ids[2, 3, 11]
    check(x, ids, t, tokens, T, rest, up=(up[0] if which != "logprob" else None, up[1] if which != "loss" else None))


@pytest.mark.parametrize("tdt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rest", [False, True])
def test_teachers_types(rest, tdt):
    say(f"distillation teacher in {tdt} rest={rest}")
    x, ids, t, tokens, up = make(20, 700, 9, "bf16", 4, rest, tdt=tdt)
    check(x, ids.to(torch.int32), t, tokens.to(torch.int16), 1.0, rest, up=up)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("V,K", [(300, 10), (9000, 200)])
def test_lists_of_different_lengths(V, K, rest):
    say(f"distillation with absent entries V={V} K={K} rest={rest}")
    x, ids, t, tokens, up = make(30, V, K, "fp32", 5, rest, absent=0.4)
    ids[0] = -1                         # nothing listed
    ids[1, 1:] = -1                     # one entry, first or last
    ids[2, :-1] = -1
    t[3] = torch.where(ids[3] < 0, math.nan, t[3])   # what stands in absent places is not read
    check(x, ids, t, tokens, 1.0, rest, up=up)
    out = kernel.distillation(x, ids, t, rest=rest)
    assert out.loss[0] == 0


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("K", [6, 130])
def test_a_token_listed_again(K, rest):
    say(f"distillation with repeated tokens K={K} rest={rest}")
    x, ids, t, tokens, up = make(12, 400, K, "fp32", 6, rest)
    ids[0] = ids[0, 0]                   # all the same
    ids[1, 1::2] = ids[1, 0:-1:2]        # pairs
    ids[2, -1] = ids[2, 0]
    if rest:
        t[0] -= math.log(3.0)
    check(x, ids, t, tokens, 1.0, rest, up=up)
    a = [kernel.distillation(x.clone().requires_grad_(True), ids, t, tokens, 2.0, rest).loss for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


@pytest.mark.parametrize("rest", [False, True])
def test_unknown_tokens_give_nan(rest):
    say(f"distillation unknown tokens rest={rest}")
    x, ids, t, tokens, up = make(8, 100, 5, "fp32", 7, rest)
    ids[0, 2], ids[1, 0] = 100, -2
    tokens[2], tokens[3], tokens[4] = 100, -2, -1
    check(x, ids, t, tokens, 1.0, rest, up=up)
    check(x, ids, t, torch.where(tokens == -1, 50, tokens), 2.0, rest, ignore=50, up=up)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rest", [False, True])
def test_masks(rest, dt):
    """-inf and the type's lowest value in masked places of the student: a row with nothing left, with one entry, with the
    listed ones or all others masked; entries of -inf in the teacher's list."""
    say(f"distillation masks rest={rest} {dt}")
    V, K = 3000, 8
    x, ids, t, tokens, up = make(12, V, K, dt, 8, rest)
    gen = torch.Generator().manual_seed(9)
    hide = torch.rand(12, V, generator=gen).cuda() < 0.6
    for value in (-math.inf, torch.finfo(DT[dt]).min):
        y = x.masked_fill(hide, value)
        y.scatter_(-1, ids, x.gather(-1, ids))       # the teacher's tokens are not masked, but for
        y[0] = value                                  # nothing left
        y[1] = value                                  # the first listed left
        y[1, ids[1, 0]] = 1.5
        y[2] = value                                  # the listed ones left: no rest
        y[2, ids[2]] = 0.5
        y[3, ids[3]] = value if value == -math.inf else max(value, -1e30)   # the listed ones masked; the loss stays in range
        tt = t.clone()
        tt[4, 1:] = -math.inf                         # one entry weighs all
        tt[5] = -math.inf                             # none weighs anything
        # a rest or listed tokens of almost no mass: the loss is huge, or +inf with -inf
        check(y, ids, tt, None, 1.0, rest, up=(up[0], None))
        check(y[4:], ids[4:], tt[4:], tokens[4:], 1.0, rest, up=(up[0][4:], up[1][4:]))


@pytest.mark.parametrize("rest", [False, True])
def test_a_small_rest_keeps_its_digits(rest):
    """A student that knows the teacher's tokens: what it leaves to the others is far below fp32's step of 1."""
    say(f"distillation of a student that is sure rest={rest}")
    x, ids, t, tokens, up = make(6, 5000, 8, "fp32", 10, rest)
    for lift in (15.0, 25.0, 60.0):
        y = x.scatter_add(-1, ids, torch.full(ids.shape, lift, device="cuda"))
        check(y, ids, t, tokens, 1.0, rest, up=up)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_offsets_do_not_matter(dt):
    say(f"distillation about large offsets {dt}")
    x, ids, t, tokens, up = make(6, 800, 8, "bf16", 11)
    for off in (3e3, -3e3):
        y = (x.float().round() + off).to(DT[dt])   # offsets shift the logits' own roundings: the reference sees them too
        check(y, ids, t + off, tokens, 1.0, False, up=up)


def test_nan_and_infinity_stay_in_their_rows():
    say("distillation NaN and infinities")
    for rest in (False, True):
        x, ids, t, tokens, up = make(9, 9000, 8, "fp32", 12, rest)
        clean = kernel.distillation(x, ids, t, tokens, 2.0, rest)
        for where in (8888, int(ids[4, 3])):
            for bad in (math.nan, math.inf):
                y = x.clone()
                y[4, where] = bad
                y.requires_grad_(True)
                out = kernel.distillation(y, ids, t, tokens, 2.0, rest)
                g, = torch.autograd.grad([out.loss.sum(), out.logprob.sum()], y)
                assert out.loss[4].isnan() and out.logprob[4].isnan() and g[4].isnan().all()
                keep = torch.arange(9, device="cuda") != 4
                assert torch.equal(out.loss[keep], clean.loss[keep]) and g[keep].isfinite().all()
        tt = t.clone()
        tt[2, 1] = math.nan
        y = x.clone().requires_grad_(True)
        out = kernel.distillation(y, ids, tt, tokens, 2.0, rest)
        g, = torch.autograd.grad(out.loss.sum(), y)
        assert out.loss[2].isnan() and g[2].isnan().all() and out.logprob.isfinite().all() and g[3:].isfinite().all()


@pytest.mark.parametrize("T", [1.0, 2.0, 3.0])
@pytest.mark.parametrize("rest", [False, True])
def test_padding_takes_nothing_from_its_entries(rest, T):
    """Positions left out of the loss by torch.where: NaN, infinities and unknown tokens among their entries leave the
    gradient that clean entries give: the formula's, and the same bits. (With the rest the listed tokens are a sum apart, so
    that where the list itself is another, rows 3 and 7, the sum of all is rounded in another order: there the formula
    and its tolerance alone.)"""
    say(f"distillation padded positions rest={rest} T={T}")
    x, ids, t, tokens, up = make(9, 5000, 8, "fp32", 30, rest, T)
    pad = torch.arange(9, device="cuda") % 2 == 1
    bad_ids, bad_t = ids.clone(), t.clone()
    bad_t[1, 2], bad_t[3], bad_t[5, 0] = math.nan, math.inf, 1e30
    bad_ids[7, 4] = 5000
    bad_ids[3, 1] = bad_ids[3, 0]
    for labels in (None, tokens):
        got = []
        for i, v in ((ids, t), (bad_ids, bad_t)):
            y = x.clone().requires_grad_(True)
            out = kernel.distillation(y, i, v, labels, T, rest)
            total = (torch.where(pad, 0.0, out.loss) * up[0]).sum()
            if labels is not None:
                total = total + (out.logprob * up[1]).sum()
            got += torch.autograd.grad(total, y)
        want, tol = reference(x, ids, t, labels, T, rest, -1, (torch.where(pad, 0.0, up[0]), None if labels is None else up[1]))
        for g in got:
            assert g.isfinite().all()
            close(g, want[2], U * tol[2] + torch.finfo(x.dtype).eps / 2 * (want[2].abs() + U * tol[2]) + TINY[x.dtype], "dlogits")
        same = torch.tensor([r for r in range(9) if not rest or r not in (3, 7)], device="cuda")
        assert torch.equal(got[0][same], got[1][same])
        if labels is None:
            assert all((g[pad] == 0).all() for g in got)


@pytest.mark.parametrize("dt,rows,V", [("fp32", 2200, 32001), ("bf16", 4200, 32008), ("fp16", 70001, 2003)])
@pytest.mark.parametrize("T,rest", [(1.0, True), (2.0, False), (1.5, False)])
def test_more_logits_than_the_cache_holds(dt, rows, V, T, rest):
    """More than 256 MiB of logits are read otherwise: each row as in a call of few rows, and a few by the formula."""
    say(f"distillation of many logits {dt} T={T} rest={rest}")
    assert rows * V * DT[dt].itemsize > 1 << 28
    x, ids, t, tokens, up = make(300, V, 20, dt, 31, rest, T)
    few = torch.arange(rows, device="cuda") % 300

    def both(at):
        y = x[at].requires_grad_(True)
        out = kernel.distillation(y, ids[at], t[at], tokens[at], T, rest)
        return out.loss.detach(), out.logprob.detach(), torch.autograd.grad([out.loss, out.logprob], y, [u[at] for u in up])[0]
    want = both(torch.arange(300, device="cuda"))
    for got, w in zip(both(few), want):
        assert all(torch.equal(got[i:i + 300], w[:rows - i]) for i in range(0, rows, 300))
    check(x[:5], ids[:5], t[:5], tokens[:5], T, rest, up=(up[0][:5], up[1][:5]))


def _views(V, dt):
    gen = torch.Generator().manual_seed(23)
    f = lambda *s: (torch.randn(*s, generator=gen) * 2).to(DT[dt]).cuda()  # noqa: E731
    return {"ahead": f(3, 9, V)[:, :-1], "column": f(4, 5, V)[:, 2], "swapped": f(5, 3, V).transpose(0, 1),
            "wider": f(6, V + 3)[:, 1:V + 1], "three": f(2, 5, 3, V)[:, 1:4, :2], "expanded": f(1, V).expand(7, V),
            "in front": f(1, 4, V).expand(3, 4, V), "every other": f(6, 2 * V)[:, ::2], "row": f(V), "none": f(0, V),
            "no rows": f(4, 0, 3, V)}


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("view", ["ahead", "column", "swapped", "wider", "three", "expanded", "in front", "every other", "row",
                                  "none", "no rows"])
def test_views(view, rest, dt):
    say(f"distillation view {view} rest={rest} {dt}")
    x = _views(333, dt)[view]
    gen = torch.Generator().manual_seed(29)
    lead = x.shape[:-1]
    ids = torch.rand(*lead, 333, generator=gen).argsort(-1)[..., :14].cuda()
    t = torch.log_softmax(torch.randn(*lead, 14, generator=gen), -1).cuda() - 0.1
    tokens = torch.randint(0, 333, lead, generator=gen).cuda()
    up = tuple(torch.randn(lead, generator=gen).cuda() for _ in range(2))
    check(x, ids[..., ::2], t[..., ::2], tokens, 1.0, rest, up=up)   # the teacher's as views, too


def test_a_row_does_not_depend_on_the_others():
    say("distillation rows alone and together")
    x, ids, t, tokens, up = make(600, 2500, 20, "bf16", 13)
    y = x.clone().requires_grad_(True)
    out = kernel.distillation(y, ids, t, tokens, 2.0)
    g, = torch.autograd.grad(list(out), y, list(up))
    for i in (0, 311, 599):
        z = x[i:i + 1].clone().requires_grad_(True)
        one = kernel.distillation(z, ids[i:i + 1], t[i:i + 1], tokens[i:i + 1], 2.0)
        h, = torch.autograd.grad(list(one), z, [u[i:i + 1] for u in up])
        assert torch.equal(one.loss[0], out.loss[i]) and torch.equal(one.logprob[0], out.logprob[i]) and torch.equal(h[0], g[i])


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T", [1.0, 1.7])
def test_gradient_against_differences(rest, T):
    """Along random directions, against differences of the float64 loss."""
    say(f"distillation gradient against differences rest={rest} T={T}")
    x, ids, t, tokens, _ = make(5, 40, 6, "fp32", 14, rest, T)
    y = x.clone().requires_grad_(True)
    out = kernel.distillation(y, ids, t, tokens, T, rest)
    g, = torch.autograd.grad(0.7 * out.loss.sum() - 0.3 * out.logprob.sum(), y)
    gen = torch.Generator().manual_seed(15)

    def value(z):
        (loss, logprob, _), _ = reference(z, ids, t, tokens, T, rest)
        return 0.7 * loss.sum() - 0.3 * logprob.sum()
    x64 = x.double().cpu()
    for _ in range(4):
        v = torch.randn(x64.shape, generator=gen, dtype=torch.float64)
        slope = (value(x64 + 1e-5 * v) - value(x64 - 1e-5 * v)) / 2e-5
        got = (g.double().cpu() * v).sum()
        assert abs(got - slope) <= 1e-5 * (g.double().cpu() * v).abs().sum() + 1e-8


def test_the_largest_rows():
    """The widest rows with the rest, and a wide one without."""
    say("distillation widest rows")
    x, ids, t, tokens, up = make(2, 1 << 18, 50, "bf16", 16, True)
    ids[0, 0], ids[1, 0] = (1 << 18) - 1, 0
    check(x, ids, t, tokens, 1.0, True, up=up)
    x, ids, t, tokens, up = make(1, 600011, 1024, "fp32", 17)
    check(x, ids, t, tokens, 2.0, False, up=up)


def test_many_rows():
    """More rows, and tiles of the gradient, than one grid dimension takes; the last rows against the definition."""
    say("distillation of 2^20 + 3 rows")
    n, V, K = (1 << 20) + 3, 5, 2
    gen = torch.Generator(device="cuda").manual_seed(18)
    x = torch.randn(n, V, device="cuda", generator=gen)
    ids = torch.tensor([[3, 1]], device="cuda").expand(n, 2).contiguous()
    t = torch.randn(n, K, device="cuda", generator=gen)
    y = x.clone().requires_grad_(True)
    out = kernel.distillation(y, ids, t)
    g, = torch.autograd.grad(out.loss.sum(), y)
    some = torch.tensor([0, 77777, (1 << 20) - 1, 1 << 20, n - 1], device="cuda")
    want, tol = reference(x[some], ids[some], t[some], None, 1.0, False, up=(torch.ones(5), None))
    close(out.loss[some], want[0], U * tol[0], "loss")
    close(g[some], want[2], U * tol[2] + U * nz(want[2]).abs() + TINY[torch.float32], "dlogits")


def test_no_gradient_goes_to_the_teacher():
    say("distillation teacher's gradient")
    x, ids, t, _, _ = make(4, 50, 5, "fp32", 19)
    t.requires_grad_(True)
    assert not kernel.distillation(x, ids, t).loss.requires_grad
    y = x.clone().requires_grad_(True)
    kernel.distillation(y, ids, t).loss.sum().backward()
    assert t.grad is None and y.grad is not None
    with torch.no_grad():
        assert not kernel.distillation(y, ids, t).loss.requires_grad
