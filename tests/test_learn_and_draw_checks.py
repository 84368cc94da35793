"""The refusals of distillation and sample_tokens: on the host, before any HIP call (CPU only)."""
import ctypes
import math

import pytest
import torch

import kernel
import ulm_native as nat
from helpers import tiny_model

X = ctypes.c_void_p(256)


def test_distillation_refuses():
    x, ids, t = torch.zeros(2, 3, 10), torch.zeros(2, 3, 4, dtype=torch.int64), torch.zeros(2, 3, 4)
    lab = torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.distillation(x, ids, t)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.distillation(x, ids, t, lab, 2.0, True)
    for bad in (x.long(), x.double(), None):
        with pytest.raises(TypeError):
            kernel.distillation(bad, ids, t)
    for bad in (t.long(), t.double(), [0.0]):
        with pytest.raises(TypeError):
            kernel.distillation(x, ids, bad)
    for bad in (t, ids.bool(), [1]):
        with pytest.raises(TypeError, match="tokens"):
            kernel.distillation(x, bad, t)
    with pytest.raises(TypeError, match="tokens"):
        kernel.distillation(x, ids, t, lab.float())
    with pytest.raises(ValueError, match="teacher_tokens"):
        kernel.distillation(x, ids[:, :2], t[:, :2])
    with pytest.raises(ValueError, match="teacher_tokens"):
        kernel.distillation(x, ids[..., 0], t[..., 0])
    with pytest.raises(ValueError, match="teacher_logits"):
        kernel.distillation(x, ids, t[..., :3])
    for k in (0, 1025):
        with pytest.raises(ValueError, match="entries"):
            kernel.distillation(x, torch.zeros(2, 3, k, dtype=torch.int64), torch.zeros(2, 3, k))
    with pytest.raises(ValueError, match="leading shape"):
        kernel.distillation(x, ids, t, lab[:, :2])
    with pytest.raises(ValueError, match=r"\(\.\.\., V\)"):
        kernel.distillation(x[..., :0], ids, t)
    for T in (0.0, -1.0, 1e-7, 1e7, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            kernel.distillation(x, ids, t, None, T)
    with pytest.raises(TypeError, match="temperature"):
        kernel.distillation(x, ids, t, None, torch.ones(()))
    with pytest.raises(TypeError):
        kernel.distillation(x, ids, t, lab, 1.0, False, 0.5)
    one = torch.zeros(1, 1, dtype=torch.int64)
    wide = torch.zeros(1).expand(1, (1 << 18) + 1)   # no memory behind it
    with pytest.raises(ValueError, match="2\\^18"):
        kernel.distillation(wide, one, one.float(), None, 1.0, True)
    with pytest.raises(ValueError, match="2\\^30"):
        kernel.distillation(torch.zeros(1).expand(1, (1 << 30) + 1), one, one.float())


def test_sample_tokens_refuses():
    x, u = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.sample_tokens(x, u)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.sample_tokens(x, u, u, u.long(), u, u)
    for bad in (x.long(), x.double(), None):
        with pytest.raises(TypeError):
            kernel.sample_tokens(bad, u)
    for bad in (u.bfloat16(), u.long(), 0.5):
        with pytest.raises(TypeError, match="u must|must be a tensor"):
            kernel.sample_tokens(x, bad)
    with pytest.raises(ValueError, match=r"\(\.\.\., V\)"):
        kernel.sample_tokens(x[..., :0], u)
    with pytest.raises(ValueError, match="leading shape"):
        kernel.sample_tokens(x, u[:, :2])
    with pytest.raises(ValueError, match="2\\^22"):
        kernel.sample_tokens(torch.zeros(1).expand(1, (1 << 22) + 1), u[0, :1])
    for kw, what in ((dict(temperature=-0.1), "temperature"), (dict(temperature=math.inf), "temperature"),
                     (dict(temperature=math.nan), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_k=1 << 63), "top_k"),
                     (dict(top_p=-0.1), "top_p"), (dict(top_p=1.1), "top_p"), (dict(top_p=math.nan), "top_p"),
                     (dict(min_p=-0.1), "min_p"), (dict(min_p=1.5), "min_p")):
        with pytest.raises(ValueError, match=what):
            kernel.sample_tokens(x, u, **kw)
    for kw in (dict(temperature=u[:, :1]), dict(top_p=u[0]), dict(min_p=torch.zeros(())), dict(top_k=u.long()[..., None])):
        with pytest.raises(ValueError, match="leading shape"):
            kernel.sample_tokens(x, u, **kw)
    for kw in (dict(temperature=u.long()), dict(top_k=u), dict(top_k=2.0), dict(min_p="a")):
        with pytest.raises((TypeError, ValueError)):
            kernel.sample_tokens(x, u, **kw)


def test_the_models_calls_refuse():
    model = tiny_model()
    x, ids = torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2, 5, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="teacher_tokens"):
        model.distill(x, ids[:, :4], ids[:, :4].float())
    with pytest.raises(ValueError, match="targets"):
        model.distill(x, ids, ids.float(), x[:, :4])
    with pytest.raises(ValueError, match="shorter"):
        model.sample(x, 4)
    with pytest.raises(ValueError, match="u "):
        model.sample(x, 7, u=torch.zeros(2, 3))


def test_the_entries_refuse_before_any_hip_call():
    lib = nat.lib()
    base = dict(logits=256, teacher_tokens=256, teacher_logits=256, tokens=None, rows=4, inner=4, outer_stride=0,
                row_stride=10, ignore_index=-1, V=10, K=3, dtype=0, teacher_dtype=0, rest=0, temperature=1.0)
    fwd = lambda loss=X, logprob=None, **kw: lib.ulm_distill(  # noqa: E731
        ctypes.byref(nat.Distillation(**{**base, **kw})), loss, logprob, X, None)
    bwd = lambda stats=X, out=ctypes.c_void_p(512), dlogprob=None, **kw: lib.ulm_distill_bwd(  # noqa: E731
        ctypes.byref(nat.Distillation(**{**base, **kw})), stats, X, dlogprob, out, None)
    for kw, msg in ((dict(rows=0), b"bad sizes"), (dict(V=0), b"bad sizes"), (dict(inner=0), b"bad sizes"), (dict(K=0), b"K=0"),
                    (dict(K=1025), b"K=1025"), (dict(rest=1, V=(1 << 18) + 1), b"rest"), (dict(dtype=7), b"bad dtype"),
                    (dict(teacher_dtype=-1), b"bad dtype"), (dict(temperature=0.0), b"temperature"),
                    (dict(temperature=math.nan), b"temperature"), (dict(logits=None), b"null pointer"),
                    (dict(teacher_tokens=None), b"null pointer"), (dict(teacher_logits=None), b"null pointer")):
        for f in (fwd, bwd):
            assert f(**kw) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error(), kw
    assert fwd(loss=None) == nat.ULM_ERR_INVALID and fwd(logprob=X) == nat.ULM_ERR_INVALID   # log probabilities of no tokens
    assert lib.ulm_distill(None, X, None, X, None) == nat.ULM_ERR_INVALID
    for kw, msg in ((dict(stats=None), b"null"), (dict(out=None), b"null"), (dict(dlogprob=X), b"null"),
                    (dict(out=X), b"alias")):
        assert bwd(**kw) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error(), kw
    assert lib.ulm_distill_max_entries() == kernel.MAX_ENTRIES and lib.ulm_distill_stats() == kernel.DISTILL_STATS
    how = nat.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None)
    draw = lambda x=X, dt=0, rows=4, inner=4, V=10, u=X, how=ctypes.byref(how), token=X: lib.ulm_sample_tokens(  # noqa: E731
        x, dt, rows, inner, 0, 10, V, u, 0, how, token, X, X, None)
    for kw, msg in ((dict(rows=0), b"bad sizes"), (dict(V=(1 << 22) + 1), b"bad sizes"), (dict(inner=0), b"bad sizes"),
                    (dict(dt=3), b"bad dtype"), (dict(x=None), b"null"), (dict(u=None), b"null"), (dict(how=None), b"null"),
                    (dict(token=None), b"null")):
        assert draw(**kw) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error(), kw


def test_fake_outputs_have_the_real_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dtype=torch.int64: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        x, ids, t, lab = e(2, 3, 10, dtype=torch.bfloat16), e(2, 3, 4), e(2, 3, 4, dtype=torch.float32), e(2, 3)
        loss, logprob, stats = kernel.distill_fwd(x, ids, t, lab, 1.0, False, -1)
        assert loss.shape == logprob.shape == (2, 3) and stats.shape == (2, 3, kernel.DISTILL_STATS)
        assert kernel.distill_fwd(x, ids, t, None, 1.0, False, -1)[1].shape == (0,)
        dx = kernel.distill_bwd(x, ids, t, lab, 1.0, False, -1, stats, loss, None)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        out = kernel.sample_tokens_op(x, e(2, 3, dtype=torch.float32), 1.0, 0, 1.0, 0.0, None, None, None, None)
        assert [o.shape for o in out] == [(2, 3)] * 3
        assert [o.dtype for o in out] == [torch.int64, torch.float32, torch.int64]
