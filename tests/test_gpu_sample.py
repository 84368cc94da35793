"""sample_tokens (ulm_sample_tokens) against its definition in float64 (needs an MI355X).

Tokens and counts have to be equal: shares and their sums are off by about 1e-12 of a row's mass on either side, and the
settings and random numbers here come no nearer to a border than chance brings them. A log probability is
rounded once from float64: within half a step of fp32, 2^-24 of it, and 1e-9 for the sums'
own resolution."""
import math

import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def column(v, rows):
    return v.double().cpu().reshape(-1) if isinstance(v, torch.Tensor) else torch.full((rows,), float(v), dtype=torch.float64)


def reference(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Row by row in float64 on the CPU: (token, logprob, kept, the kept mask)."""
    V = logits.shape[-1]
    x = logits.double().cpu().reshape(-1, V)
    n = x.shape[0]
    u, T, k, p, m = (column(v, n) for v in (u, temperature, top_k, top_p, min_p))
    token, logprob, kept = torch.full((n,), -1), torch.full((n,), math.nan, dtype=torch.float64), torch.zeros(n, dtype=torch.int64)
    masks = torch.zeros(n, V, dtype=torch.bool)
    for r in range(n):
        row = x[r]
        if row.isnan().any() or (row == math.inf).any() or (row == -math.inf).all() or not 0 <= T[r] < math.inf \
                or p[r].isnan() or m[r].isnan():
            continue
        best, order = torch.sort(row, descending=True, stable=True)
        order = order[best > -math.inf]
        if T[r] == 0:
            order = order[:1]
        elif 0 < k[r] < order.numel():
            order = order[:int(k[r])]
        w = ((row[order] - best[0]) / (T[r] if T[r] > 0 else 1.0)).exp()
        if p[r] < 1:
            before = torch.cumsum(w, 0) - w
            order = order[:max(1, int((before < p[r] * w.sum()).sum()))]
        order = order[:max(1, int((w[:order.numel()] >= m[r]).sum()))] if m[r] <= 1 else order[:1]
        masks[r, order] = True
        w = torch.where(masks[r], ((row - best[0]) / (T[r] if T[r] > 0 else 1.0)).exp(), 0.0)
        c = torch.cumsum(w, 0)
        above = torch.nonzero(c > u[r] * c[-1])
        token[r] = above[0, 0] if above.numel() else torch.nonzero(w > 0)[-1, 0]
        logprob[r] = (row[token[r]] - best[0]) / (T[r] if T[r] > 0 else 1.0) - c[-1].log()
        kept[r] = order.numel()
    lead = logits.shape[:-1]
    return token.reshape(lead), logprob.reshape(lead), kept.reshape(lead), masks.reshape(logits.shape)


def check(logits, u, **how):
    out = kernel.sample_tokens(logits, u, **how)
    token, logprob, kept, _ = reference(logits, u, **how)
    assert out.token.dtype == out.kept.dtype == torch.int64 and out.logprob.dtype == torch.float32
    assert torch.equal(out.kept.cpu(), kept), ("kept", out.kept.cpu()[out.kept.cpu() != kept], kept[out.kept.cpu() != kept])
    assert torch.equal(out.token.cpu(), token), "token"
    got = out.logprob.double().cpu()
    assert torch.equal(got.isnan(), logprob.isnan())
    err = (got - logprob).abs() - (2.0 ** -24 * logprob.abs() + 1e-9)
    assert err.nan_to_num(-1).numel() == 0 or err.nan_to_num(-1).max() <= 0, "logprob"
    return out


def make(lead, V, dt, seed, std=2.0, likely=6):
    gen = torch.Generator().manual_seed(seed)
    lead = (lead,) if isinstance(lead, int) else lead
    x = torch.randn(*lead, V, generator=gen) * std
    at = torch.randint(0, V, (*lead, likely), generator=gen)
    x.scatter_add_(-1, at, 3 + 4 * torch.rand(*lead, likely, generator=gen))
    return x.to(DT[dt]).cuda(), torch.rand(lead, generator=gen).cuda(), gen


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_p=0.97),
            dict(top_k=40, top_p=0.8), dict(temperature=0.5, top_k=100, top_p=0.95, min_p=0.01), dict(temperature=0.0),
            dict(top_k=1), dict(top_p=0.0), dict(top_p=0.05), dict(temperature=2.0, top_k=700), dict(min_p=1.0),
            dict(temperature=1.5, min_p=1e-4), dict(top_p=0.999), dict(temperature=8.0, top_p=0.6)]


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,V", [(1, 1), (5, 2), (3, 7), (40, 63), (9, 64), (9, 65), (33, 511), (5, 1025), (7, 4096), (7, 4097),
                                    (5, 8191), (300, 1000), (4, 32000), (3, 50001)])
def test_draws(rows, V, dt):
    say(f"sample_tokens rows={rows} V={V} {dt}")
    x, u, gen = make(rows, V, dt, rows + V)
    for how in SETTINGS:
        check(x, u, **how)


MORE = [dict(top_k=65), dict(top_k=128, top_p=0.9), dict(top_k=129), dict(top_k=3000, top_p=0.99), dict(top_p=1 - 1e-9),
        dict(temperature=8.0, top_p=0.9999), dict(top_p=0.9, min_p=1e-3), dict(top_p=0.3, min_p=1e-3), dict(top_p=0.99, min_p=0.02),
        dict(temperature=0.05, top_p=0.9), dict(top_k=300, min_p=0.01), dict(temperature=3.0, top_k=128)]


@pytest.mark.parametrize("V,dt", [(9000, "fp32"), (9001, "bf16"), (40000, "fp16"), (2001, "fp32"), (150001, "bf16")])
def test_few_and_many_rows_alike(V, dt):
    """Every setting over more rows than CUs and over few: equal bits, and the definition's tokens."""
    say(f"sample_tokens few and many rows V={V} {dt}")
    n = 270
    x, u, gen = make(n, V, dt, V + 1, std=2.5)
    x[5] = x[5].round()
    x[6, 200:] = -math.inf
    some = torch.tensor([0, 5, 6, 269], device="cuda")
    for how in SETTINGS + MORE:
        out = kernel.sample_tokens(x, u, **how)
        for i in (0, 135):
            part = kernel.sample_tokens(x[i:i + 135], u[i:i + 135], **how)
            assert all(torch.equal(a.nan_to_num(9), b[i:i + 135].nan_to_num(9)) for a, b in zip(part, out)), how
        want = reference(x[some], u[some], **how)
        assert torch.equal(out.token[some].cpu(), want[0]) and torch.equal(out.kept[some].cpu(), want[2]), how


@pytest.mark.parametrize("V,dt", [(131072, "bf16"), (131073, "fp32"), (200003, "fp16"), (1 << 20, "bf16")])
def test_large_vocabularies(V, dt):
    say(f"sample_tokens V={V} {dt}")
    x, u, _ = make(2, V, dt, V)
    for how in SETTINGS[:8] + SETTINGS[12:]:
        check(x, u, **how)


@pytest.mark.parametrize("V,dt", [(300, "fp32"), (9000, "bf16"), (33000, "fp32")])
def test_settings_of_each_row(V, dt):
    """A row's own settings draw what a call with these numbers draws."""
    say(f"sample_tokens rows' own settings V={V} {dt}")
    n = 60
    x, u, gen = make(n, V, dt, 5)
    f = lambda: torch.rand(n, generator=gen).cuda()  # noqa: E731
    T = torch.where(f() < 0.2, 0.0, 0.3 + 1.2 * f())
    k = (f() * 80).long() * (f() < 0.6)
    p = torch.where(f() < 0.3, 1.0, 0.4 + 0.59 * f())
    m = torch.where(f() < 0.5, 0.0, 0.2 * f())
    out = check(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    check(x, u.double(), temperature=T.double(), top_k=k.to(torch.int32), top_p=0.9, min_p=m.bfloat16())
    for i in (0, 17, 59):
        one = kernel.sample_tokens(x[i], u[i], T[i].item(), k[i].item(), p[i].item(), m[i].item())
        assert all(torch.equal(a, b[i]) for a, b in zip(one, out))


def test_rows_that_cannot_be_drawn():
    say("sample_tokens rows without a draw")
    x, u, _ = make(12, 5000, "fp32", 6)
    x[0] = -math.inf
    x[1, 4999] = math.nan
    x[2, 0] = math.inf
    x[3, 1:] = -math.inf
    x[4, :4998] = -math.inf
    T, p, m = torch.ones(12).cuda(), torch.full((12,), 0.9).cuda(), torch.zeros(12).cuda()
    T[5], T[6], T[7], p[8], m[9] = -1.0, math.nan, math.inf, math.nan, math.nan
    k = torch.full((12,), 3).cuda()
    k[10], k[11] = -5, 1 << 40
    out = check(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert out.token[[0, 1, 2, 5, 6, 7, 8, 9]].tolist() == [-1] * 8 and out.kept[[0, 1, 2, 5, 6, 7, 8, 9]].tolist() == [0] * 8
    assert out.token[3] == 0 and out.logprob[3] == 0
    for how in SETTINGS:
        check(x, u, **how)
    p[0], p[3], m[4], m[10] = -1.0, 2.0, 3.0, -1.0
    check(x, u, top_p=p, min_p=m)


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_masks(dt):
    """-inf and the type's lowest value in masked places."""
    say(f"sample_tokens masks {dt}")
    x, u, gen = make(20, 6000, dt, 7)
    hide = torch.rand(6000, generator=gen).cuda() < 0.8
    for value in (-math.inf, torch.finfo(DT[dt]).min, -1e4):
        y = x.masked_fill(hide, value)
        y[1] = value
        y[1, 5999] = 2.0
        for how in SETTINGS:
            out = check(y, u, **how)
        assert not hide[out.token[2:]].any()


@pytest.mark.parametrize("V", [1024, 4096, 16384, 131072])
def test_equal_logits_and_borders_met_exactly(V):
    """All equal: shares and borders are whole numbers, and the lower indices are kept."""
    say(f"sample_tokens equal logits V={V}")
    n = 40
    x = torch.full((n, V), 1.25).cuda()
    x[1::2] = -1.25
    j = torch.arange(n) * (V // n)
    u = (j / V).double().cuda()
    out = check(x, u)
    assert torch.equal(out.token.cpu(), j) and (out.kept == V).all()
    out = check(x, u, top_p=0.5)
    assert (out.kept == V // 2).all()
    out = check(x, u, top_k=V // 4, top_p=0.25)
    assert (out.kept == V // 16).all() and (out.token < V // 16).all()
    assert (check(x, u, top_k=777).kept == 777).all()
    x[:, ::2] = -0.0
    x[:, 1::2] = 0.0     # one value
    assert (check(x, u, top_p=0.5, min_p=1.0).kept == V // 2).all()


@pytest.mark.parametrize("V,dt", [(32000, "bf16"), (8000, "fp32")])
def test_large_entries_in_a_few_threads(V, dt):
    """More entries than the short way holds, all where only a few threads read; a bin with more than the waves hold."""
    say(f"sample_tokens crowded entries V={V} {dt}")
    x, u, gen = make(6, V, dt, 18, std=0.5)
    x[:, 1000:2200] = 9.0
    x[1, 1000:2200] = torch.linspace(8.9, 9.0, 1200).to(DT[dt]).cuda()
    x[2, 1000:2200] = torch.linspace(4.0, 30.0, 1200).to(DT[dt]).cuda()
    for how in (dict(top_k=50), dict(top_k=128), dict(top_k=1100), dict(top_p=0.5), dict(top_k=900, top_p=0.4),
                dict(top_p=0.97, min_p=0.5)):
        check(x, u, **how)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_many_ties_at_the_border(dt):
    """A few values only: the last kept one is one of thousands of equals, of which the lower indices stay."""
    say(f"sample_tokens ties at the border {dt}")
    x, u, gen = make(24, 40000, dt, 8)
    x = x.round()
    x[0] = 0
    x[0, -300:] = 3
    x[1, :] = -2
    x[1, torch.randperm(40000, generator=gen)[:5000].cuda()] = -1
    for how in (dict(top_k=10), dict(top_k=3000), dict(top_k=20000), dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.99),
                dict(top_k=5000, top_p=0.77), dict(top_p=0.95, min_p=0.1), dict(temperature=0.0)):
        check(x, u, **how)


@pytest.mark.parametrize("rows,V,dt", [(24, 32000, "bf16"), (260, 6000, "fp16"), (5, 140001, "fp32"), (3, 900, "fp32")])
def test_top_p_behind_a_large_top_k(rows, V, dt):
    """top_p's share is of what top_k keeps; ties, masked rows with fewer entries than top_k, and both zeros at top_k's border."""
    say(f"sample_tokens top_p behind a large top_k rows={rows} V={V} {dt}")
    x, u, gen = make(rows, V, dt, 21)
    x[0] = (x[0].float() * 2).round() / 2
    x[1, 150:] = -math.inf
    x[2] = -3.0
    x[2, 5::3], x[2, 1::9] = -0.0, 0.0
    for k in (129, 200, 1000, 2500):
        for p, m in ((0.3, 0.0), (0.95, 0.0), (0.9999, 0.0), (0.95, 0.02), (0.9, 1e-4)):
            check(x, u, top_k=k, top_p=p, min_p=m)
    check(x, u, top_k=500, top_p=0.9, temperature=0.02)
    check(x, u, top_k=500, top_p=0.9, temperature=1e4)


def test_the_ends_of_the_random_numbers():
    """u = 0 draws the first kept token, numbers next to 1 the last one with a share; outside [0, 1) likewise."""
    say("sample_tokens ends of u")
    x, _, _ = make(1, 3000, "fp32", 9)
    u = torch.tensor([0.0, 2.0 ** -60, 1 - 2.0 ** -53, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, math.nan], dtype=torch.float64).cuda()
    for how in (dict(top_k=9), dict(top_p=0.8), dict(min_p=0.01)):
        mask = reference(x, u[:1], **how)[3][0]
        first, last = torch.nonzero(mask)[0, 0], torch.nonzero(mask)[-1, 0]
        got = kernel.sample_tokens(x.expand(8, 3000), u, **how).token.cpu()
        assert got.tolist() == [first, first, last, last, last, last, first, first]


@pytest.mark.parametrize("how", [dict(), dict(temperature=0.6, top_p=0.9), dict(top_k=20), dict(min_p=0.02)])
def test_shares_of_many_draws(how):
    """Over evenly spaced random numbers every token comes out as often as its share says, to one draw."""
    say(f"sample_tokens shares {how}")
    x, _, _ = make(1, 2000, "fp32", 10)
    n = 20000
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).cuda()
    out = kernel.sample_tokens(x.expand(n, 2000), u, **how)
    mask = reference(x, u[:1], **how)[3][0]
    z = (x[0].double().cpu() / how.get("temperature", 1.0)).masked_fill(~mask, -math.inf)
    want = torch.softmax(z, -1) * n
    got = torch.bincount(out.token.cpu(), minlength=2000)
    assert ((got - want).abs() <= 1 + 1e-6).all() and not got[~mask].any()
    assert (out.token[1:] >= out.token[:-1]).all()   # in the order of the tokens' numbers
    lp = torch.log_softmax(z, -1)[out.token.cpu()]
    assert ((out.logprob.cpu() - lp).abs() <= 2.0 ** -24 * lp.abs() + 1e-9).all()


def test_extreme_temperatures():
    say("sample_tokens extreme temperatures")
    x, u, _ = make(16, 3000, "fp32", 11)
    for T in (1e-30, 1e-4, 1e4, 1e30, 1e300):
        for how in (dict(), dict(top_k=50), dict(top_p=0.7), dict(top_k=9, top_p=0.5, min_p=0.2)):
            check(x, u, temperature=T, **how)
    y = x * 1e30
    for T in (1.0, 1e30):
        for how in SETTINGS[:1] + [dict(top_k=50), dict(top_p=0.7)]:
            check(y, u, **{**how, "temperature": T})
    check(x + 1e6, u, top_p=0.9)
    check(x - 1e6, u, top_p=0.9, top_k=200)


def _views(V, dt):
    gen = torch.Generator().manual_seed(23)
    f = lambda *s: (torch.randn(*s, generator=gen) * 2).to(DT[dt]).cuda()  # noqa: E731
    return {"last": f(3, 9, V)[:, -1], "swapped": f(5, 3, V).transpose(0, 1), "wider": f(6, V + 3)[:, 1:V + 1],
            "three": f(2, 5, 3, V)[:, 1:4, :2], "expanded": f(1, V).expand(7, V), "in front": f(1, 4, V).expand(3, 4, V),
            "every other": f(6, 2 * V)[:, ::2], "row": f(V), "none": f(0, V), "no rows": f(4, 0, 3, V)}


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("view", ["last", "swapped", "wider", "three", "expanded", "in front", "every other", "row", "none",
                                  "no rows"])
def test_views(view, dt):
    say(f"sample_tokens view {view} {dt}")
    x = _views(1333, dt)[view]
    gen = torch.Generator().manual_seed(29)
    u = torch.rand(x.shape[:-1], generator=gen).cuda()
    T = 0.5 + torch.rand(x.shape[:-1], generator=gen).cuda()
    for how in (dict(), dict(top_k=10, top_p=0.9), dict(temperature=T, top_p=0.8)):
        check(x, u, **how)
    if u.dim() == 2 and u.numel():
        a, b = (kernel.sample_tokens(x, v, T) for v in (u, u.t().contiguous().t()))
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_a_row_does_not_depend_on_the_others():
    say("sample_tokens rows alone and together")
    x, u, _ = make(700, 33000, "bf16", 12)
    out = kernel.sample_tokens(x, u, 0.9, 50, 0.95)
    free = kernel.sample_tokens(x, u)
    for i in (0, 255, 256, 699):
        one = kernel.sample_tokens(x[i:i + 1], u[i:i + 1], 0.9, 50, 0.95)
        assert all(torch.equal(a[0], b[i]) for a, b in zip(one, out))
        one = kernel.sample_tokens(x[i], u[i])
        assert all(torch.equal(a, b[i]) for a, b in zip(one, free))
    again = kernel.sample_tokens(x, u, 0.9, 50, 0.95)
    assert all(torch.equal(a, b) for a, b in zip(again, out))
    some = torch.tensor([0, 1, 2, 350, 698, 699], device="cuda")
    for how, got in ((dict(temperature=0.9, top_k=50, top_p=0.95), out), (dict(), free)):
        want = reference(x[some], u[some], **how)
        assert torch.equal(got.token[some].cpu(), want[0]) and torch.equal(got.kept[some].cpu(), want[2])


def test_many_rows():
    say("sample_tokens of 2^20 + 3 rows")
    n = (1 << 20) + 3
    gen = torch.Generator(device="cuda").manual_seed(13)
    x = torch.randn(n, 5, device="cuda", generator=gen)
    u = torch.rand(n, device="cuda", generator=gen)
    out = kernel.sample_tokens(x, u, top_k=3)
    some = torch.tensor([0, 77777, (1 << 20) - 1, 1 << 20, n - 1], device="cuda")
    want = reference(x[some], u[some], top_k=3)
    assert torch.equal(out.token[some].cpu(), want[0]) and torch.equal(out.kept[some].cpu(), want[2])


def test_against_greedy_and_log_probabilities():
    """Temperature 0 is the argmax; the unfiltered draw's log probability is the token's own."""
    say("sample_tokens against token_logprobs")
    x, u, _ = make((6, 50), 997, "fp32", 14)
    assert torch.equal(kernel.sample_tokens(x, u, 0.0).token, x.argmax(-1))
    out = kernel.sample_tokens(x, u)
    own = kernel.token_logprobs(x, out.token)
    assert (own.logprob - out.logprob).abs().max() <= 2.0 ** -24 * (997 / 256 + 2 * math.log(998) + 40 + 4 * own.logprob.abs().max())
