"""token_logprobs over the whole range of finite logits: masks of any finite value, single large logits
(needs an MI355X). Definition, tolerances and their derivation: test_gpu_logprobs.py. No term there
depends on the logits' magnitude: x - m is exact or off by half a step of itself, whatever m is."""
import math

import pytest
import torch

from helpers import say
from test_gpu_logprobs import DT, TINY, U, check, close, make, reference, units, ups

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402

# masks and single logits, in the types that hold them
LARGE = [1e4, 1e6, 2.0 ** 24, 1e9, 3e9, 5e9, 1e10, 1e12, 1e15, 1e20, 1e28, 2.0 ** 95, 2.0 ** 96, 1e30]
CASES = [(dt, value) for dt in DT for value in LARGE + [torch.finfo(DT[dt]).max] if value <= torch.finfo(DT[dt]).max]
SIZES = [(9, 32000), (520, 3001)]   # fewer and more rows than 512: workgroups of both sizes


@pytest.mark.parametrize("dt,value", CASES)
def test_masked_with_a_large_negative_number(dt, value):
    """Whole rows, all but a few entries, stretches longer than a workgroup's batch of loads, single places."""
    for rows, V in SIZES:
        say(f"token_logprobs masked with {-value:g} rows={rows} V={V} {dt}")
        logits, tokens, gen = make(rows, V, dt, 61)
        hide = torch.zeros(rows, V, dtype=torch.bool)
        hide[0] = True                                          # nothing left
        few = torch.randperm(V, generator=gen)[:10]
        hide[1:3] = True
        hide[1:3, few] = False                                  # ten left, the token one of them or not
        hide[3, : 2 * V // 3] = True                            # a leading stretch
        hide[4, V // 3:] = True                                 # a trailing one
        hide[5, : V - 1] = True                                 # the last entry left
        hide[6, 1:] = True                                      # the first
        hide[7] = torch.rand(V, generator=gen) < 0.7
        hide[8, V // 2] = True                                  # one entry masked
        tokens[1], tokens[2], tokens[5], tokens[6] = few[3], (few[0] + 1) % V, V - 1, 0
        x = logits.masked_fill(hide.cuda(), -value)
        check(x, tokens, 6, up=ups(gen, (rows,), 6))
        check(x, tokens, 0, up=ups(gen, (rows,), 0, "a"))


@pytest.mark.parametrize("dt,value", CASES)
def test_one_large_logit(dt, value):
    for rows, V in SIZES:
        say(f"token_logprobs one logit of {value:g} rows={rows} V={V} {dt}")
        x, tokens, gen = make(rows, V, dt, 67)
        x[0, 0] = x[1, V // 2] = x[2, V - 1] = value
        x[3, 7], x[3, V - 7] = value, value                     # two alike
        x[4, 7], x[4, V - 7] = value, -value
        x[5] = value                                            # nothing else
        tokens[0], tokens[1], tokens[3] = 0, 3, 7
        check(x, tokens, 5, up=ups(gen, (rows,), 5))


def check_spread(logits, tokens, top, up):
    """`check` for rows whose spread takes p below 2^-126, where the hardware's power of two is 0: the
    gradient's element -p f is then off by 2^-126 |f| besides, with |f| = |G + h (ln p + H)| at most
    |a| + sum |c_j| + |h| (m - x_i + 2 ln V), as ln p = x_i - m - ln s, s <= V, H <= ln V."""
    V, dt, n = logits.shape[-1], logits.dtype, units(logits.shape[-1])
    x = logits.detach().requires_grad_(True)
    out = kernel.token_logprobs(x, tokens, top)
    outs, dx, scale = reference(logits, tokens, top, -1, up)
    close(out.logprob, outs[0], U * (n + 4 * outs[0].abs()), "logprob")
    close(out.entropy, outs[1], U * 3 * n * (1 + math.log(V + 1)), "entropy")
    close(out.top_logprobs, outs[2], U * (n + 4 * outs[2].abs()), "top_logprobs")
    assert torch.equal(out.top_tokens.cpu(), outs[3]), "top_tokens"
    got, = torch.autograd.grad(list(out[:3]), [x], list(up))
    a, h, c = (u.double().cpu() for u in up)
    d = logits.double().cpu()
    d = d.amax(-1, keepdim=True) - d
    f = (a.abs() + c.abs().sum(-1))[..., None] + h.abs()[..., None] * (d + 2 * math.log(V + 1))
    half = torch.finfo(dt).eps / 2
    close(got, dx, U * scale + half * (dx.abs() + U * scale) + TINY[dt] + 2.0 ** -126 * f, "dlogits")


OFFSETS = [(dt, sign * value) for dt, values in
           (("fp32", [1e3, 1e4, 6e4, 1e6, 2.0 ** 24 - 64, 2.0 ** 24, 2.0 ** 25, 1e9]), ("bf16", [1e3, 6e4, 1e6, 2.0 ** 24]),
            ("fp16", [1e3, 6e4])) for value in values for sign in (1, -1)]


@pytest.mark.parametrize("dt,offset", OFFSETS)
def test_logits_about_an_offset(dt, offset):
    """Ordinary logits with a constant added: every output but for the logits' own rounding to the type."""
    for rows, V in SIZES:
        say(f"token_logprobs logits about {offset:g} rows={rows} V={V} {dt}")
        gen = torch.Generator().manual_seed(71)
        x = torch.randn(rows, V, generator=gen) * 3
        x[1] = x[1].sort().values                      # every batch has a new maximum
        x[2] = x[2].sort(descending=True).values
        x[3] *= 10
        x = (x.double() + offset).to(DT[dt]).cuda()
        tokens = torch.randint(0, V, (rows,), generator=gen).cuda()
        check_spread(x, tokens, 5, ups(gen, (rows,), 5))
