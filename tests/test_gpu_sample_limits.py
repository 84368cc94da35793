"""sample_tokens at the ends of its types' ranges, against test_gpu_sample's definition in float64 (needs an MI355X)."""
import math

import pytest
import torch

from helpers import say
from test_gpu_sample import check

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402


def _u(n):
    """Random numbers over all of [0, 1), the last ones next to 1."""
    u = (torch.arange(n, dtype=torch.float64) + 0.37) / n
    u[-3:] = torch.tensor([0.999, 1 - 2.0 ** -24, 1 - 2.0 ** -53])
    return u.cuda()


def _rows(n, V, top, some, seed):
    """Rows whose largest entry is `top`: all of it, with -inf among it, one entry only, and beside lower ones `some`."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.full((n, V), top, dtype=torch.float64)
    f = lambda: torch.rand(n, V, generator=gen)  # noqa: E731
    kind = torch.arange(n)[:, None] % 4
    x[(kind == 1) & (f() < 0.5)] = -math.inf
    x[(kind == 2).expand(n, V)] = -math.inf
    x[(kind == 3) & (f() < 0.3)] = some
    x[torch.arange(n), torch.randint(0, V, (n,), generator=gen)] = top
    return x


LOWEST = torch.finfo(torch.float32).min
HOW = [dict(), dict(temperature=0.7), dict(top_p=0.9), dict(top_p=0.5, min_p=0.05), dict(top_k=7), dict(top_k=7, top_p=0.6),
       dict(top_k=200), dict(top_k=200, top_p=0.9), dict(min_p=0.05), dict(min_p=1.0), dict(temperature=1e30),
       dict(temperature=1e30, top_p=0.9), dict(temperature=1e300, top_p=0.9), dict(temperature=0.0)]


@pytest.mark.parametrize("V", [1, 97, 300, 1000, 6000, 31999, 50257])
def test_rows_of_the_lowest_float(V):
    """Nothing but masked entries of the lowest value: drawn from alike, with -inf entries and what lies past the row's end
    having no part."""
    say(f"sample_tokens rows of the lowest float V={V}")
    x = _rows(24, V, LOWEST, -math.inf, V).float().cuda()
    for how in HOW:
        check(x, _u(24), **how)


@pytest.mark.parametrize("dt,T", [(torch.bfloat16, 1e34), (torch.bfloat16, 1e35), (torch.bfloat16, 1e36), (torch.float32, 3e35),
                                  (torch.float16, 1e37)])
def test_low_rows_at_temperatures_that_reach_the_lowest_float(dt, T):
    """The lowest float lies within a few temperatures of the row's entries."""
    say(f"sample_tokens low rows {dt} temperature {T}")
    low = torch.finfo(dt).min
    x = _rows(24, 1500, low if dt != torch.float32 else LOWEST * 0.998, low, 5).to(dt).cuda()
    for how in HOW[:10]:
        check(x, _u(24), **{**how, "temperature": T})


@pytest.mark.parametrize("T", [5e-324, 1e-310, 5e-309, 1e-300, 1e-200])
def test_temperatures_whose_reciprocal_is_no_number(T):
    """The tokens of the largest value share the draw, and its log probability is a number."""
    say(f"sample_tokens temperature {T}")
    gen = torch.Generator().manual_seed(3)
    x = (torch.randn(24, 3000, generator=gen) * 2).cuda()
    x[::2] = x[::2].round()
    for how in (dict(), dict(top_k=50), dict(top_k=300), dict(top_p=0.7), dict(top_k=9, top_p=0.5, min_p=0.2), dict(min_p=0.5)):
        out = check(x, _u(24), temperature=T, **how)
        assert out.logprob.isfinite().all() and (out.token >= 0).all()


def test_min_p_between_masses_that_rounding_turns_round():
    """Masses as formed are off by 4e-14, so that an entry a little larger than another may weigh a little less. Whichever of the
    two a min_p between them keeps, a token comes out of what is kept."""
    say("sample_tokens min_p between two masses")
    x = torch.full((64, 5000), -30.0)
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 0.0, -1e-15
    T = 2 / math.log(2)   # both weigh 2^-1/2 to 1e-15
    u = ((torch.arange(64, dtype=torch.float64) + 0.5) / 64).cuda()
    for k in (0, 200):
        out = kernel.sample_tokens(x.cuda(), u, T, k, 0.95, 0.707106781186528)
        assert ((out.kept == 2) | (out.kept == 3)).all(), out.kept
        assert ((out.token >= 0) & (out.token < 3)).all(), out.token
        z = 1 + (out.kept.double() - 1) * 2 ** -0.5
        want = torch.where(out.token == 0, 0.0, -0.5 * math.log(2)) - z.log()
        assert ((out.logprob - want).abs() <= 2.0 ** -24 * want.abs() + 1e-9).all()
