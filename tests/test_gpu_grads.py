"""grad_norm, clip_grads and clip_grad_norm_ against their definitions in float64 (needs an MI355X).

The squares are exact in double and summed in it: the norm is off by its one rounding to fp32. The
factor takes three more roundings (the sum with 1e-6, the quotient, the product) and the result
rounds to its type."""
import math

import pytest
import torch

from helpers import say

pytestmark = pytest.mark.gpu

import kernel  # noqa: E402

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def true_norm(grads, kind=2.0):
    if kind == 2.0:
        return math.sqrt(math.fsum(g.detach().double().square().sum().item() for g in grads))
    return max((g.detach().double().abs().max().item() for g in grads if g.numel()), default=0.0)


def make(shapes, dts, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * std * 10.0 ** (-(i % 3))).to(DT[dts[i % len(dts)]]).cuda()
            for i, s in enumerate(shapes)]


def check(grads, factor, out_dts=None, kind=2.0):
    norm = true_norm(grads, kind)
    bound = norm * factor
    got = kernel.grad_norm(grads, kind)
    assert got.dtype == torch.float32 and got.shape == () and abs(got.item() - norm) <= 1.001 * U * norm
    out = [torch.full_like(g, 7, dtype=DT[out_dts[i % len(out_dts)]]) for i, g in enumerate(grads)] if out_dts else None
    before = [g.clone() for g in grads]
    n2, res = kernel.clip_grads(grads, bound, out=out, norm_type=kind)
    assert torch.equal(n2, got) and all(torch.equal(a, b) for a, b in zip(before, grads))
    assert out is None or all(a is b for a, b in zip(res, out))
    coef = min(1.0, bound / (norm + 1e-6))
    for g, r in zip(grads, res):
        assert r.shape == g.shape and (out is not None or r.dtype == g.dtype)
        want = g.double() * coef
        half, tiny = torch.finfo(r.dtype).eps / 2, 2.0 ** -25 if r.dtype == torch.float16 else 2.0 ** -126
        tol = 4 * U * want.abs()
        assert ((r.double() - want).abs() <= tol + half * (want.abs() + tol) + tiny).all()
    # in place: the same bits
    if out is None or all(o.dtype == g.dtype for o, g in zip(out, grads)):
        n3, same = kernel.clip_grads(grads, bound, out=grads, norm_type=kind)
        assert torch.equal(n3, got) and all(torch.equal(a, b) and a is g for a, b, g in zip(same, res, grads))


SHAPES = {
    "one": [(1,)], "scalars": [(), (1,), ()], "odd": [(7,), (3, 5), (), (1, 1, 9)], "with empty": [(0,), (5,), (4, 0), (8192,)],
    "chunks": [(8191,), (8192,), (8193,), (3, 8192), (16385,)], "matrices": [(300, 77), (1000, 129), (64, 64), (5,)],
    "many": [(i % 13 + 1, i % 7 + 1) for i in range(300)], "large": [(3000, 4001), (17,), (1 << 20,)],
    "a model": [(500, 96), (96,)] + [s for _ in range(12) for s in
                                     ((96,), (96, 1, 4), (200, 96), (200,), (96, 200), (96, 96), (200,), (), ())],
}


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("dts,out_dts", [(["fp32"], None), (["bf16"], ["fp32"]), (["fp16", "fp32", "bf16"], None),
                                         (["fp32", "bf16", "fp16"], ["bf16", "fp16", "fp32", "fp32"])])
@pytest.mark.parametrize("which", list(SHAPES))
def test_norm_and_clip(which, dts, out_dts, kind):
    say(f"clip_grads {which} {dts} -> {out_dts} norm {kind}")
    for factor in (0.25, 4.0):
        check(make(SHAPES[which], dts, seed=len(which)), factor, out_dts, kind)


def test_order_and_alignment_of_views():
    """Views of a bucket at any offset, of either alignment; transposed and strided ones."""
    say("clip_grads views")
    for dt in DT.values():
        flat = torch.randn(40000, device="cuda").to(dt)
        check([flat[1:8194].view(8193), flat[8194:8201], flat[8201:8202].view(()), flat[8203:40000]], 0.5)
        base = torch.randn(60, 50, device="cuda").to(dt)
        check([base.t(), torch.randn(9, 8, 7, device="cuda").to(dt).permute(2, 0, 1)], 0.5)
    strided = torch.randn(40, 30, device="cuda")
    keep = strided.clone()
    with pytest.raises(ValueError, match="share memory"):   # interleaved: one region
        kernel.clip_grads([strided[:, ::3], strided[:, 1::3]], 1.0, out=[strided[:, ::3], strided[:, 1::3]])
    g = [strided[:20, ::3], strided[20:, 1::3][::2]]
    norm = true_norm(g)
    kernel.clip_grads(g, norm / 2, out=g)
    touched = torch.zeros(40, 30, dtype=torch.bool, device="cuda")
    touched[:20, ::3] = True
    touched[20::2, 1::3] = True
    assert torch.equal(strided[~touched], keep[~touched])
    coef = norm / 2 / (norm + 1e-6)
    assert ((strided.double() - keep.double() * coef).abs()[touched] <= 5 * U * keep.double().abs()[touched]).all()
    # results in another order than their gradients
    a = torch.randn(30, 20, device="cuda")
    o = torch.empty(20, 30, device="cuda").t()
    n, _ = kernel.clip_grads([a], 1.0, out=[o])
    assert torch.equal(o, kernel.clip_grads([a], 1.0)[1][0])


def test_extremes():
    """Squares far past fp32's range either way, an overflow of the norm itself, NaN and infinity."""
    say("clip_grads extremes")
    for v in (1e-30, 1e30):
        check([torch.full((1000,), v, device="cuda"), torch.full((3,), -v, device="cuda")], 0.5 if v > 1 else 1e5)
    tiny = torch.full((10000,), 2.0 ** -149, device="cuda")   # the smallest fp32 value
    assert kernel.grad_norm(tiny).item() == 100 * 2.0 ** -149
    big = torch.full((4,), 3e38, device="cuda")
    assert kernel.grad_norm([big]).item() == math.inf and kernel.grad_norm([big], math.inf).item() == big[0].item()
    for bad in (math.nan, math.inf):
        for kind in (2.0, math.inf):
            g = [torch.ones(9000, device="cuda"), torch.ones(5, device="cuda")]
            g[1][2] = bad
            norm, out = kernel.clip_grads(g, 1.0, norm_type=kind)
            if math.isnan(bad):
                assert norm.isnan() and all(o.isnan().all() for o in out)
            else:
                assert norm.isinf() and (out[0] == 0).all() and out[1][2].isnan() and (out[1][:2] == 0).all()
    # a bound of 0 and one of infinity
    g = [torch.ones(10, device="cuda")]
    assert (kernel.clip_grads(g, 0.0)[1][0] == 0).all() and torch.equal(kernel.clip_grads(g, math.inf)[1][0], g[0])
    z = [torch.zeros(10, device="cuda")]
    norm, out = kernel.clip_grads(z, 1.0)
    assert norm == 0 and (out[0] == 0).all()


def test_offsets_past_32_bits():
    say("clip_grads past 2^32 elements")
    n = (1 << 32) + 5000
    g = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    g.zero_()
    g[-1], g[0] = 3.0, 4.0
    norm, _ = kernel.clip_grads([g], 2.5, out=[g])
    assert norm.item() == 5.0
    coef = torch.tensor(2.5) / (torch.tensor(5.0) + 1e-6)
    assert g[-1].item() == (3 * coef).bfloat16().item() and g[0].item() == (4 * coef).bfloat16().item()
    assert not g[1:-1].any()


def test_clip_grad_norm_of_parameters():
    say("clip_grad_norm_")
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((30, 20), (7,), ())]
    params.append(torch.nn.Parameter(torch.zeros(3, device="cuda")))   # has no gradient
    for p in params[:3]:
        p.grad = torch.randn_like(p)
    before = [p.grad.clone() for p in params[:3]]
    want = true_norm(before)
    norm = kernel.clip_grad_norm_(iter(params), 0.5)
    assert abs(norm.item() - want) <= 1.001 * U * want and params[3].grad is None
    got = true_norm([p.grad for p in params[:3]])
    assert abs(got - 0.5 * want / (want + 1e-6)) <= 4 * U * 0.5
    kept = [p.grad.clone() for p in params[:3]]
    kernel.clip_grad_norm_(params, 10.0)
    assert all(torch.equal(p.grad, k) for p, k in zip(params, kept))
    assert kernel.clip_grad_norm_(params[1], 10.0).item() == kernel.grad_norm(params[1].grad).item()
    params[0].grad[0, 0] = math.nan
    kept = [p.grad.clone() for p in params[1:3]]
    with pytest.raises(RuntimeError, match="norm is nan"):
        kernel.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(p.grad, k) for p, k in zip(params[1:3], kept))
    assert kernel.clip_grad_norm_([], 1.0).item() == 0 and kernel.clip_grad_norm_([params[3]], 1.0).item() == 0


def test_refusals():
    say("clip_grads refusals")
    g = torch.randn(100, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        kernel.clip_grads([g, g], 1.0, out=[g, g])
    with pytest.raises(ValueError, match="share memory"):
        grads = [g[:60], g[50:]]
        kernel.clip_grads(grads, 1.0, out=grads)
    with pytest.raises(ValueError, match="share memory"):
        kernel.clip_grads([g[:50], g[50:]], 1.0, out=[g[50:], g[:50]])
    with pytest.raises(ValueError, match="share memory"):
        e = [g[:1].expand(5)]
        kernel.clip_grads(e, 1.0, out=e)
    assert torch.equal(kernel.grad_norm([g, g]), kernel.grad_norm([torch.cat([g, g])]))   # reading twice is fine
    a, b = kernel.clip_grads([g, g], 1.0)[1]
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.grad_norm([g, g.cpu()])
    with pytest.raises(ValueError, match="shape"):
        kernel.clip_grads([g], 1.0, out=[g[:50]])
    with pytest.raises(ValueError, match="shape"):
        kernel.clip_grads([g], 1.0, out=[])
