"""The refusals of token_logprobs, embedding, grad_norm and clip_grads: on the host, before any HIP call (CPU only)."""
import ctypes
import math

import pytest
import torch

import kernel
import ulm_native as nat

X = ctypes.c_void_p(256)


def test_token_logprobs_refuses():
    x, t = torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.token_logprobs(x, t)
    with pytest.raises(TypeError, match="floating"):
        kernel.token_logprobs(x.long(), t)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        kernel.token_logprobs(x.double(), t)
    for bad in (t.float(), t.bool(), [0]):
        with pytest.raises(TypeError, match="tokens"):
            kernel.token_logprobs(x, bad)
    with pytest.raises(ValueError, match="leading shape"):
        kernel.token_logprobs(x, t[:, :2])
    with pytest.raises(ValueError, match="leading shape"):
        kernel.token_logprobs(x, t[..., None])
    for top in (-1, 11, 65):
        with pytest.raises(ValueError, match="top must be"):
            kernel.token_logprobs(x, t, top)
    with pytest.raises(ValueError, match=r"\(\.\.\., V\)"):
        kernel.token_logprobs(x[..., :0], t)
    with pytest.raises(TypeError, match="tensor"):
        kernel.token_logprobs(None, t)
    with pytest.raises(TypeError):
        kernel.token_logprobs(x, t, 1.5)
    wide = torch.zeros(1).expand(1, (1 << 22) + 1)   # no memory behind it
    with pytest.raises(ValueError, match="2\\^22"):
        kernel.token_logprobs(wide, t[0, :1], 1)
    with pytest.raises(ValueError, match="2\\^30"):
        kernel.token_logprobs(torch.zeros(1).expand(1, (1 << 30) + 1), t[0, :1])


def test_embedding_refuses():
    w, t = torch.zeros(10, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.embedding(w, t)
    with pytest.raises(TypeError, match="floating"):
        kernel.embedding(w.long(), t)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        kernel.embedding(w.double(), t)
    with pytest.raises(TypeError, match="tokens"):
        kernel.embedding(w, t.float())
    with pytest.raises(TypeError, match="scale"):
        kernel.embedding(w, t, torch.ones(()))
    with pytest.raises(ValueError, match="2\\^28"):
        kernel.embedding(torch.zeros(1).expand((1 << 28) + 1, 1), t)
    with pytest.raises(ValueError, match="2\\^20"):
        kernel.embedding(torch.zeros(1).expand(1, (1 << 20) + 1), t)
    for bad in (w[0], w[:0], w[:, :0], w[None]):
        with pytest.raises(ValueError, match=r"\(V, D\)"):
            kernel.embedding(bad, t)


def test_clipping_refuses():
    g = torch.ones(4)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.grad_norm([g])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        kernel.clip_grads([g], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        kernel.grad_norm([g], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            kernel.clip_grads([g], bad)
    for bad in (g.double(), g.long(), g.to_sparse(), 3.0):
        with pytest.raises(TypeError):
            kernel.grad_norm([bad])
    assert kernel.grad_norm([]).item() == 0
    norm, out = kernel.clip_grads([], 1.0)
    assert norm.item() == 0 and out == []


def test_overlaps_of_results_are_found():
    flat = torch.zeros(100)
    a, b, c = flat[:40], flat[40:60], flat[60:]
    ok, bad = kernel._check_regions, lambda g, o: pytest.raises(ValueError, kernel._check_regions, g, o)
    ok([a, b, c], [a, b, c])
    ok([a, a], [b[:20], c])           # a gradient read twice
    ok([a, flat[:0]], [a, flat[:0]])
    bad([a, a], [a, a])
    bad([a, b], [b.expand(20), a])
    bad([a, flat[39:50]], [a, flat[39:50]])
    bad([a, b], [a, flat[30:50]])
    bad([flat[:1].expand(3)], [flat[:1].expand(3)])
    bad([a, b], [c, a[:20]])          # written where another gradient is read
    assert kernel._dense(flat.view(20, 5).t()) and not kernel._dense(flat[::2]) and not kernel._dense(flat[:1].expand(4))


def test_rows_of_a_view():
    """Views that the kernels read in place, and those that are copied."""
    x = torch.zeros(4, 6, 5, 8)

    def spans(t):
        y, inner, outer, row = kernel._rows(t)
        n = t.numel() // t.shape[-1]
        at = [(r // inner) * outer + (r % inner) * row for r in range(n)]
        want = [(y.as_strided((1,), (1,), y.storage_offset() + o)).data_ptr() for o in at]
        rows = y.reshape(-1, y.shape[-1]) if y is not t else None
        flat = [t[i].data_ptr() for i in __import__("itertools").product(*map(range, t.shape[:-1]))] if y is t else \
            [rows[i].data_ptr() for i in range(n)]
        assert want == flat
        return y is t
    assert spans(x) and spans(x[:, :3]) and spans(x[:, 2]) and spans(x[1, 2]) and spans(x[1, 2, 3]) and spans(x[..., 1:5])
    assert spans(x[:, :, 1:2]) and spans(x.view(24, 5, 8).transpose(0, 1)) and spans(x[:1].expand(3, 6, 5, 8)[:, 1])
    assert not spans(x[:, 1:3, 1:3]) and not spans(x[..., ::2]) and not spans(x.transpose(-1, -2))


def test_the_entries_refuse_before_any_hip_call():
    lib = nat.lib()
    lp = lambda *a: lib.ulm_token_logprobs(*a)  # noqa: E731
    args = lambda rows=4, V=10, top=0, dt=nat.ULM_F32, inner=4, x=X, ws=X, n=1 << 20: (  # noqa: E731
        x, dt, X, rows, inner, 0, 10, V, top, -1, X, X, X, X, X, ws, n, None)
    for kw, msg in ((dict(rows=0), b"bad sizes"), (dict(V=0), b"bad sizes"), (dict(inner=0), b"bad sizes"), (dict(top=11), b"top"),
                    (dict(top=-1), b"top"), (dict(V=100, top=65), b"top"), (dict(dt=7), b"bad dtype"),
                    (dict(x=None), b"null pointer"), (dict(V=1 << 20, top=1, n=0), b"workspace"),
                    (dict(V=(1 << 22) + 1, top=1), b"top=1 with")):
        assert lp(*args(**kw)) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error(), kw
    bw = lambda x=X, out=ctypes.c_void_p(512), dtop=None, dent=None, ent=X: (  # noqa: E731
        x, nat.ULM_F32, X, 4, 4, 0, 10, 10, 0, -1, X, ent, X, X, dent, dtop, out, None)
    for a, msg in ((bw(out=X), b"alias"), (bw(out=None), b"null"), (bw(dtop=X), b"null"), (bw(dent=X, ent=None), b"null")):
        assert lib.ulm_token_logprobs_bwd(*a) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error()
    assert lib.ulm_token_logprobs_max_top() == kernel.MAX_TOP == 64
    for a, msg in (((X, 9, X, 4, 10, 8, 1.0, X, None), b"bad dtype"), ((X, 0, X, 0, 10, 8, 1.0, X, None), b"bad sizes"),
                   ((X, 0, None, 4, 10, 8, 1.0, X, None), b"null"), ((X, 0, X, (1 << 30) + 1, 10, 8, 1.0, X, None), b"bad sizes")):
        assert lib.ulm_embed_fwd(*a) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error()
    need = lib.ulm_embed_bwd_workspace_bytes(4, 10, 8)
    assert need > 0 and lib.ulm_embed_bwd_workspace_bytes(0, 10, 8) == 0
    for a, msg in (((X, 0, X, 4, 10, 8, 1.0, X, X, need - 1, None), b"workspace"),
                   ((X, 0, X, 4, 10, 8, 1.0, None, X, need, None), b"null")):
        assert lib.ulm_embed_bwd(*a) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error()
    grad = lambda **kw: (nat.Grad * 1)(  # noqa: E731
        nat.Grad(**{**dict(src=256, dst=512, numel=5, src_dtype=0, dst_dtype=0), **kw}))
    clip = lambda g, n=1, kind=2, bound=1.0, ws=1 << 20: lib.ulm_clip_grads(g, n, kind, bound, X, X, ws, None)  # noqa: E731
    for g, kw, msg in ((grad(numel=-1), {}, b"elements"), (grad(src_dtype=5), {}, b"bad dtype"),
                       (grad(dst_dtype=5), {}, b"bad dtype"),
                       (grad(src=None), {}, b"null pointer"), (grad(dst=None), {}, b"null pointer"), (None, {}, b"null pointer"),
                       (grad(dst=256, dst_dtype=1), {}, b"in place"), (grad(), dict(kind=1), b"norm type"),
                       (grad(), dict(bound=-1.0), b"negative"), (grad(), dict(bound=math.nan), b"negative"),
                       (grad(), dict(ws=7), b"workspace")):
        assert clip(g, **kw) == nat.ULM_ERR_INVALID and msg in lib.ulm_last_error(), msg


def test_fake_outputs_have_the_real_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, t = torch.empty(2, 3, 10, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 3, dtype=torch.int64, device="cuda")
        outs = kernel.token_logprobs_fwd(x, t, 4, -1)
        assert [tuple(o.shape) for o in outs] == [(2, 3), (2, 3), (2, 3, 4), (2, 3, 4), (2, 3, 2)]
        assert [o.dtype for o in outs] == [torch.float32] * 3 + [torch.int64, torch.float32]
        dx = kernel.token_logprobs_bwd(x, t, 4, -1, outs[4], outs[1], outs[3], outs[0], None, None)
        assert dx.shape == x.shape and dx.dtype == x.dtype
        w = torch.empty(10, 6, device="cuda")
        y = kernel.embed_fwd(w, t, 1.0)
        assert y.shape == (2, 3, 6) and kernel.embed_bwd(y, t, 10, 1.0).shape == (10, 6)
