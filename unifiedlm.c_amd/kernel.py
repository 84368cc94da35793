"""UnifiedBlock's fast memory on MI355X: the operator surface of the reference's
kernel.py (kernel.py:1-15, 199-238), computed by hand-written gfx950 HIP
kernels in libulm_fm.so.

unified_memory(r, v, g, w) -> (q, fast), for every batch row and position t:

    k_t    = r_{t-1}                                     (k_0 = 0, write address)
    c_t    = w + sum_{s<=t} lam^(t-s) k_s                (slot evidence mass, lam = exp(g))
    q_t    = r_t / c_t
    fast_t = sum_{s<=t} lam^(t-s) (q_t . k_s) v_s

Matmul operands are bf16 with fp32 accumulation and an fp32 chunk state kept
on chip; c, q and all their gradients are fp32, as in the reference.

Besides the operator this module exposes the relu^2 slot address
(model.py:70-72) as an autograd Function, the three per-token decode
kernels used by UnifiedBlock.step, and the two ends of a step: the embedding
lookup, the log probabilities of given tokens (the loss), and the gradients'
norm and clipping.
"""
import math
import operator
from collections import namedtuple
from typing import Optional

import torch
from torch.utils._device import DeviceContext

import ulm_native as nat
from ulm_native import call, ptr

CHUNK = 64          # kernel.py:20


def _check_float(name, t):
    if not torch.is_floating_point(t):
        raise TypeError(f"{name} must be a floating tensor, got {t.dtype}")


def _check_fm(r, v, g, w):
    for name, t in (("r", r), ("v", v), ("g", g), ("w", w)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        _check_float(name, t)
    if r.dim() != 3 or v.dim() != 3:
        raise ValueError(f"r and v must be (B, T, A) and (B, T, D); got {tuple(r.shape)} and {tuple(v.shape)}")
    B, T, A = r.shape
    if v.shape[:2] != r.shape[:2]:
        raise ValueError(f"r {tuple(r.shape)} and v {tuple(v.shape)} disagree on (B, T)")
    if B == 0 or T == 0 or A == 0 or v.shape[2] == 0:
        raise ValueError(f"empty input: r {tuple(r.shape)}, v {tuple(v.shape)}")
    if w.shape != (A,):
        raise ValueError(f"w must have shape ({A},), got {tuple(w.shape)}")
    if g.numel() != 1:
        raise ValueError(f"g must hold one scalar, got shape {tuple(g.shape)}")
    nat.dtype_code(v.dtype)
    nat.require_device(r, v, g, w)


# The operators below are registered torch ops (torch.library.custom_op) with
# fake (meta) implementations and registered autograd, so torch.compile traces
# models that use them without graph breaks: each op is one opaque node whose
# output shapes the fake implementation gives. Their real implementations
# launch the native kernels on the current stream. Outputs never alias inputs;
# what a backward needs of an input's cast is recomputed from the input.

Tensor = torch.Tensor


def _fm_fwd_impl(r: Tensor, v: Tensor, g: Tensor, w: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """(q fp32, fast in v's dtype, saved uint8): ulm_fm_fwd."""
    B, T, A = r.shape
    D = v.shape[-1]
    r32 = r.float().contiguous()
    vc = v.contiguous()
    g1 = g.float().reshape(1).contiguous()
    w32 = w.float().contiguous()
    q = torch.empty(B, T, A, device=r.device, dtype=torch.float32)
    fast = torch.empty(B, T, D, device=r.device, dtype=v.dtype)
    vdt = nat.dtype_code(v.dtype)
    saved_bytes = nat.lib().ulm_fm_saved_bytes(B, T, A, D, vdt)
    saved = torch.empty(saved_bytes, device=r.device, dtype=torch.uint8)
    ws_bytes = nat.lib().ulm_fm_fwd_workspace_bytes(B, T, A, D, vdt)
    ws = torch.empty(max(ws_bytes, 1), device=r.device, dtype=torch.uint8)
    call("ulm_fm_fwd", ptr(r32), ptr(vc), vdt, ptr(g1), ptr(w32), ptr(q), ptr(fast), vdt, ptr(saved), saved_bytes,
         ptr(ws), ws_bytes, B, T, A, D, nat.stream_of(r))
    return q, fast, saved


fm_fwd = torch.library.custom_op("ulm::fm_fwd", mutates_args=())(_fm_fwd_impl)


@fm_fwd.register_fake
def _fm_fwd_fake(r, v, g, w):
    B, T, A = r.shape
    D = v.shape[-1]
    saved_bytes = nat.lib().ulm_fm_saved_bytes(B, T, A, D, nat.dtype_code(v.dtype))
    return (r.new_empty(B, T, A, dtype=torch.float32), v.new_empty(B, T, D),
            r.new_empty(saved_bytes, dtype=torch.uint8))


def _fm_bwd_impl(r: Tensor, g: Tensor, w: Tensor, saved: Tensor, v_dtype: torch.dtype, dq_out: Optional[Tensor],
                 dfast: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """(dr fp32, dv in dfast's dtype, dg (1,), dw (A,)): ulm_fm_bwd."""
    B, T, A = r.shape
    D = dfast.shape[-1]
    r32 = r.float().contiguous()
    g1 = g.float().reshape(1).contiguous()
    w32 = w.float().contiguous()
    ddt = nat.dtype_code(dfast.dtype)
    dfast = dfast.contiguous()
    dqo = dq_out.float().contiguous() if dq_out is not None else None
    dr = torch.empty(B, T, A, device=r.device, dtype=torch.float32)
    dv = torch.empty(B, T, D, device=r.device, dtype=dfast.dtype)
    dg = torch.empty(1, device=r.device, dtype=torch.float32)
    dw = torch.empty(A, device=r.device, dtype=torch.float32)
    # the saved buffer's size names the form its forward used; the backward follows it
    ws_bytes = nat.lib().ulm_fm_bwd_workspace_bytes(B, T, A, D, ddt, saved.numel(), nat.dtype_code(v_dtype))
    ws = torch.empty(max(ws_bytes, 1), device=r.device, dtype=torch.uint8)
    call("ulm_fm_bwd", ptr(r32), ptr(g1), ptr(w32), ptr(saved), saved.numel(), nat.dtype_code(v_dtype), ptr(dfast),
         ddt, ptr(dqo), ptr(dr), ptr(dv), ddt, ptr(dg), ptr(dw), ptr(ws), ws_bytes, B, T, A, D, nat.stream_of(r))
    return dr, dv, dg, dw


fm_bwd = torch.library.custom_op("ulm::fm_bwd", mutates_args=())(_fm_bwd_impl)


@fm_bwd.register_fake
def _fm_bwd_fake(r, g, w, saved, v_dtype, dq_out, dfast):
    B, T, A = r.shape
    D = dfast.shape[-1]
    return (r.new_empty(B, T, A, dtype=torch.float32), dfast.new_empty(B, T, D),
            r.new_empty(1, dtype=torch.float32), r.new_empty(A, dtype=torch.float32))


def _fm_setup(ctx, inputs, output):
    r, v, g, w = inputs
    _, _, saved = output
    ctx.save_for_backward(r, g, w, saved)
    ctx.v_dtype, ctx.D = v.dtype, v.shape[-1]
    ctx.mark_non_differentiable(saved)
    # no zero-filled stand-ins for absent gradients (the saved buffer's above all)
    ctx.set_materialize_grads(False)


def _fm_backward(ctx, dq_out, dfast, _dsaved):
    r, g, w, saved = ctx.saved_tensors
    if dq_out is None and dfast is None:
        return None, None, None, None
    if dfast is None:
        dfast = r.new_zeros(*r.shape[:2], ctx.D, dtype=torch.float32)
    dr, dv, dg, dw = fm_bwd(r, g, w, saved, ctx.v_dtype, dq_out, dfast)
    return dr, dv, dg.reshape(g.shape), dw


torch.library.register_autograd("ulm::fm_fwd", _fm_backward, setup_context=_fm_setup)


# the number of active torch dispatch modes (one assumed where torch does not say)
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 1)
_function_modes = getattr(torch._C, "_len_torch_function_stack", lambda: 1)


def _watched():
    """Whether a torch function mode, other than a default device, would see the registered ops' calls."""
    modes = getattr(torch.overrides, "_get_current_function_mode_stack", lambda: [None])()
    return any(type(m) is not DeviceContext for m in modes)


def _plain_eager(*tensors):
    """True when the call runs eagerly on plain tensors: no torch.compile
    trace, no dispatch mode (fake tensors, functionalization), no function mode
    that would see the call, and tensors or parameters proper. The host module then takes it, without the registered
    ops' dispatch and Python between the launches; the registered ops serve
    the rest (the module itself looks at the tensors it is given)."""
    if torch.compiler.is_compiling() or _dispatch_modes() > 0 or (_function_modes() > 0 and _watched()):
        return False
    return all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in tensors)


def unified_memory(r, v, g, w):
    """r: (B,T,M) read addresses, v: (B,T,D) values, g: scalar log decay, w: (M,) prior mass.
    Returns (q fp32, fast in v's dtype) (kernel.py:236-238)."""
    if _plain_eager():
        out = nat.host().memory(r, v, g, w)
        if out is not None:
            return out
    _check_fm(r, v, g, w)
    q, fast, _ = fm_fwd(r, v, g, w)
    return q, fast


class UnifiedMemory:
    """The reference's autograd Function (kernel.py:199-233) as a call
    surface: apply(r, v, g, w) is unified_memory, whose backward is the
    registered ulm::fm_bwd. The forward keeps one opaque buffer of what the
    backward needs (bf16 operand tiles of q, k and v, score tiles and the
    per-chunk evidence checkpoints that stand in for the full c tensor); v is
    passed in its own dtype and cast to bf16 for the products inside
    (kernel.py:205)."""

    @staticmethod
    def apply(r, v, g, w):
        return unified_memory(r, v, g, w)


def la(a, b, c, g, reverse=False, split=False):
    """o_t = sum_{s<=t} lam^(t-s) (a_t . b_s) c_s (s>=t when reverse), fp32 output.
    The chunked building block (kernel.py:183-196); a, b (B,T,K), c (B,T,V).
    split carries the decayed state-update operand as a bf16 hi + lo pair."""
    nat.require_device(a, b, c, g)
    a16, b16, c16 = (x.to(torch.bfloat16).contiguous() for x in (a, b, c))
    B, T, K = a16.shape
    V = c16.shape[-1]
    if b16.shape != a16.shape or c16.shape[:2] != a16.shape[:2]:
        raise ValueError("la: a, b must be (B,T,K) and c (B,T,V)")
    g1 = g.float().reshape(1).contiguous()
    out = torch.empty(B, T, V, device=a.device, dtype=torch.float32)
    ws_bytes = nat.lib().ulm_la_workspace_bytes(B, T, K, V)
    ws = torch.empty(max(ws_bytes, 1), device=a.device, dtype=torch.uint8)
    call("ulm_la", ptr(a16), ptr(b16), ptr(c16), ptr(g1), ptr(out), B, T, K, V, int(reverse), int(split), ptr(ws),
         ws_bytes, nat.stream_of(a))
    return out


# ---------------------------------------------------------------------------
# relu^2 slot address (model.py:70-72)

@torch.library.custom_op("ulm::addr_fwd", mutates_args=())
def addr_fwd(pre: Tensor, bias: Optional[Tensor], log_eps: Tensor) -> tuple[Tensor, Tensor]:
    """(r fp32 shaped like pre, denom (M,) fp32): ulm_addr_fwd."""
    A = pre.shape[-1]
    pre_c = pre.contiguous()
    b32 = bias.float().contiguous() if bias is not None else None
    le = log_eps.float().reshape(1).contiguous()
    M = pre_c.numel() // A
    r = torch.empty(pre.shape, device=pre.device, dtype=torch.float32)
    denom = torch.empty(M, device=pre.device, dtype=torch.float32)
    call("ulm_addr_fwd", ptr(pre_c), nat.dtype_code(pre.dtype), ptr(b32), ptr(le), ptr(r), ptr(denom), M, A,
         nat.stream_of(pre))
    return r, denom


@addr_fwd.register_fake
def _addr_fwd_fake(pre, bias, log_eps):
    return pre.new_empty(pre.shape, dtype=torch.float32), pre.new_empty(pre.numel() // pre.shape[-1],
                                                                        dtype=torch.float32)


@torch.library.custom_op("ulm::addr_bwd", mutates_args=())
def addr_bwd(pre: Tensor, bias: Optional[Tensor], log_eps: Tensor, r: Tensor, denom: Tensor,
             dr: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """(dpre in pre's dtype, dbias (A,) fp32 or (0,) without a bias, dlog_eps (1,)): ulm_addr_bwd."""
    A = pre.shape[-1]
    pre_c = pre.contiguous()
    M = pre_c.numel() // A
    b32 = bias.float().contiguous() if bias is not None else None
    le = log_eps.float().reshape(1).contiguous()
    dr = dr.float().contiguous()
    dpre = torch.empty_like(pre_c)
    dbias = torch.empty(A if bias is not None else 0, device=pre.device, dtype=torch.float32)
    dle = torch.empty(1, device=pre.device, dtype=torch.float32)
    ws_bytes = nat.lib().ulm_addr_bwd_workspace_bytes(M, A)
    ws = torch.empty(ws_bytes, device=pre.device, dtype=torch.uint8)
    call("ulm_addr_bwd", ptr(pre_c), nat.dtype_code(pre.dtype), ptr(b32), ptr(le), ptr(r.contiguous()),
         ptr(denom), ptr(dr), ptr(dpre), ptr(dbias if bias is not None else None), ptr(dle), ptr(ws), ws_bytes,
         M, A, nat.stream_of(pre))
    return dpre, dbias, dle


@addr_bwd.register_fake
def _addr_bwd_fake(pre, bias, log_eps, r, denom, dr):
    A = pre.shape[-1]
    return (torch.empty_like(pre, memory_format=torch.contiguous_format),
            pre.new_empty(A if bias is not None else 0, dtype=torch.float32), pre.new_empty(1, dtype=torch.float32))


def _addr_setup(ctx, inputs, output):
    pre, bias, log_eps = inputs
    r, denom = output
    ctx.save_for_backward(pre, bias, log_eps, r, denom)
    ctx.mark_non_differentiable(denom)
    ctx.set_materialize_grads(False)


def _addr_backward(ctx, dr, _ddenom):
    if dr is None:
        return None, None, None
    pre, bias, log_eps, r, denom = ctx.saved_tensors
    dpre, dbias, dle = addr_bwd(pre, bias, log_eps, r, denom, dr)
    return dpre, (dbias if bias is not None else None), dle.reshape(log_eps.shape)


torch.library.register_autograd("ulm::addr_fwd", _addr_backward, setup_context=_addr_setup)


def relu2_address(pre, bias, log_eps):
    """The slot address of model.py:70-72 from pre = K u (the bias added in fp32
    inside): r = z / (exp(clamp(log_eps,-10,10)) + sum_a z), z = relu(pre + bias)^2."""
    _check_float("pre", pre)
    if pre.dim() < 1 or pre.numel() == 0:
        raise ValueError(f"pre must be non-empty (..., A), got {tuple(pre.shape)}")
    A = pre.shape[-1]
    if bias is not None and bias.shape != (A,):
        raise ValueError(f"bias must have shape ({A},), got {tuple(bias.shape)}")
    if log_eps.numel() != 1:
        raise ValueError("log_eps must hold one scalar")
    nat.dtype_code(pre.dtype)
    nat.require_device(pre, bias, log_eps)
    return addr_fwd(pre, bias, log_eps)[0]


# ---------------------------------------------------------------------------
# UnifiedBlock.forward (model.py:77-85) with the fast memory and its
# elementwise ends fused; the GEMMs are plain library GEMMs (hipBLASLt through
# torch.mm) with fp32 accumulation

# clamp range of a block's log prior mass, w = exp(clamp(log_w, -7, 12)) (model.py:75)
LOG_W_MIN, LOG_W_MAX = -7.0, 12.0


def _mm(a, b, out_dtype):
    """a @ b, written in out_dtype straight from the fp32 accumulator."""
    return torch.mm(a, b) if a.dtype == out_dtype else torch.mm(a, b, out_dtype=out_dtype)


def _wgrad(a, b):
    """a^T b in fp32 for a (K, N1), b (K, N2) with K the token dimension: the
    split-K MFMA kernel for bf16 operands whose widths are multiples of 8,
    the library GEMM otherwise."""
    K, N1 = a.shape
    N2 = b.shape[1]
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16 or N1 % 8 or N2 % 8:
        return _mm(a.t(), b, torch.float32)
    a, b = a.contiguous(), b.contiguous()
    c = torch.empty(N1, N2, device=a.device, dtype=torch.float32)
    ws_bytes = nat.lib().ulm_wgrad_workspace_bytes(K, N1, N2)
    ws = torch.empty(max(ws_bytes, 1), device=a.device, dtype=torch.uint8)
    call("ulm_wgrad", ptr(a), ptr(b), ptr(c), K, N1, N2, ptr(ws), ws_bytes, nat.stream_of(a))
    return c


def _addmm_(c, a, b):
    """c += a @ b in place, c fp32, accumulated in the GEMM's epilogue."""
    if a.dtype == c.dtype:
        return torch.addmm(c, a, b, out=c)
    return torch.addmm(c, a, b, out_dtype=c.dtype, out=c)


# One UnifiedBlock (model.py:77-85) as two registered ops:
#
#     h, u   = RMSNorm(x), causal conv(h)               ulm_norm_conv_fwd
#     pre, v = u K^T, h W_v^T                            GEMMs in cdt
#     denom  = the relu^2 address's row sums of pre + b  ulm_addr_fwd (r not written)
#     g, w   = -exp(log_rate), exp(clamp(log_w))         ulm_block_params
#     wq, y  = w q, x + fast                             ulm_block_fm_fwd (r formed from pre)
#     out    = y + wq mu^T                               GEMM accumulating into y
#
# cdt is the GEMM operand dtype: bf16 under bf16 autocast (the reference's
# training configuration, train.py), fp32 otherwise. x is the fp32 residual
# stream; every gradient is returned in fp32. The forward's extra outputs are
# what the backward reads (the normalised input, the conv output, the key
# GEMM's output, the address denominators, g and w, the fast memory's saved
# buffer and w q).

_BLOCK_SAVED = 9   # outputs of block_fwd past `out`


@torch.library.custom_op("ulm::block_fwd", mutates_args=())
def block_fwd(x: Tensor, norm_w: Tensor, conv_w: Tensor, key_w: Tensor, key_b: Optional[Tensor], log_eps: Tensor,
              val_w: Tensor, mu_w: Tensor, log_rate: Tensor, log_w: Tensor, norm_eps: float,
              cdt: torch.dtype) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(out, rstd, h, u, pre, denom, g, w, saved, wq)."""
    # the GEMM dtypes are explicit: autocast must not re-cast them
    with torch.autocast("cuda", enabled=False):
        return _block_fwd_impl(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt)


def _block_fwd_impl(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt):
    B, T, D = x.shape
    A = key_w.shape[0]
    Kc = conv_w.shape[-1]
    M = B * T
    dev = x.device
    s = nat.stream_of(x)
    cd = nat.dtype_code(cdt)
    f32 = torch.float32
    x32 = x.contiguous()
    nw = norm_w.float().contiguous()
    cw = conv_w.float().reshape(D, Kc).contiguous()
    h = torch.empty(B, T, D, device=dev, dtype=cdt)
    u = torch.empty(B, T, D, device=dev, dtype=cdt)
    rstd = torch.empty(B, T, device=dev, dtype=f32)
    call("ulm_norm_conv_fwd", ptr(x32), nat.ULM_F32, ptr(nw), ptr(cw), Kc, float(norm_eps), ptr(h), cd, ptr(u), cd,
         ptr(rstd), B, T, D, s)
    kw, vw, mw = (t.to(cdt).contiguous() for t in (key_w, val_w, mu_w))
    pre = torch.mm(u.view(M, D), kw.t())
    v = torch.mm(h.view(M, D), vw.t())
    b32 = key_b.float().contiguous() if key_b is not None else None
    le = log_eps.float().reshape(1).contiguous()
    denom = torch.empty(M, device=dev, dtype=f32)
    # r itself is never written: the fast memory forms it from pre, bias and denom
    call("ulm_addr_fwd", ptr(pre), cd, ptr(b32), ptr(le), None, ptr(denom), M, A, s)
    lr = log_rate.float().reshape(1).contiguous()
    lw = log_w.float().contiguous()
    g1 = torch.empty(1, device=dev, dtype=f32)
    w32 = torch.empty(A, device=dev, dtype=f32)
    call("ulm_block_params", ptr(lr), ptr(lw), LOG_W_MIN, LOG_W_MAX, A, ptr(g1), ptr(w32), s)
    saved_bytes = nat.lib().ulm_fm_saved_bytes(B, T, A, D, cd)
    saved = torch.empty(saved_bytes, device=dev, dtype=torch.uint8)
    ws_bytes = nat.lib().ulm_block_fm_fwd_workspace_bytes(B, T, A, D)
    ws = torch.empty(max(ws_bytes, 1), device=dev, dtype=torch.uint8)
    qw = torch.empty(M, A, device=dev, dtype=cdt)
    y = torch.empty(M, D, device=dev, dtype=f32)
    call("ulm_block_fm_fwd", ptr(pre), cd, ptr(b32), ptr(denom), ptr(v), cd, ptr(g1), ptr(w32), ptr(qw), cd,
         ptr(x32), ptr(y), ptr(saved), saved_bytes, ptr(ws), ws_bytes, B, T, A, D, s)
    del ws, v
    out = _addmm_(y, qw, mw.t())
    return out.view(B, T, D), rstd, h, u, pre, denom, g1, w32, saved, qw


@block_fwd.register_fake
def _block_fwd_fake(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt):
    B, T, D = x.shape
    A = key_w.shape[0]
    M = B * T
    f32 = torch.float32
    saved_bytes = nat.lib().ulm_fm_saved_bytes(B, T, A, D, nat.dtype_code(cdt))
    e = x.new_empty
    return (e(B, T, D, dtype=f32), e(B, T, dtype=f32), e(B, T, D, dtype=cdt), e(B, T, D, dtype=cdt),
            e(M, A, dtype=cdt), e(M, dtype=f32), e(1, dtype=f32), e(A, dtype=f32), e(saved_bytes, dtype=torch.uint8),
            e(M, A, dtype=cdt))


@torch.library.custom_op("ulm::block_bwd", mutates_args=())
def block_bwd(dout: Tensor, x: Tensor, norm_w: Tensor, conv_w: Tensor, key_w: Tensor, key_b: Optional[Tensor],
              log_eps: Tensor, val_w: Tensor, mu_w: Tensor, log_rate: Tensor, log_w: Tensor, rstd: Tensor, h: Tensor,
              u: Tensor, pre: Tensor, denom: Tensor, g1: Tensor, w32: Tensor, saved: Tensor, qw: Tensor,
              cdt: torch.dtype) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor,
                                         Tensor]:
    """(dx, dnorm_w, dconv_w, dkey_w, dkey_b ((0,) without a bias), dlog_eps,
    dval_w, dmu_w, dlog_rate, dlog_w), all fp32."""
    with torch.autocast("cuda", enabled=False):
        return _block_bwd_impl(dout, x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, rstd, h,
                               u, pre, denom, g1, w32, saved, qw, cdt)


def _block_bwd_impl(dout, x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, rstd, h, u, pre,
                    denom, g1, w32, saved, qw, cdt):
    B, T, D = x.shape
    A = key_w.shape[0]
    Kc = conv_w.shape[-1]
    M = B * T
    dev = x.device
    s = nat.stream_of(x)
    cd = nat.dtype_code(cdt)
    f32 = torch.float32
    x32 = x.contiguous()
    nw = norm_w.float().contiguous()
    cw = conv_w.float().reshape(D, Kc).contiguous()
    kw, vw, mw = (t.to(cdt).contiguous() for t in (key_w, val_w, mu_w))
    b32 = key_b.float().contiguous() if key_b is not None else None
    le = log_eps.float().reshape(1).contiguous()
    lr = log_rate.float().reshape(1).contiguous()
    lw = log_w.float().contiguous()
    dout = dout.float().contiguous()
    if cdt == f32:
        d16 = dout
    else:
        d16 = torch.empty(B, T, D, device=dev, dtype=cdt)
        call("ulm_cast", ptr(dout), nat.ULM_F32, ptr(d16), cd, M * D, s)
    d2 = d16.view(M, D)
    dqw = torch.mm(d2, mw)                       # d(w q) = dout mu
    dmu = _wgrad(d2, qw)
    dr = torch.empty(M, A, device=dev, dtype=f32)
    dv = torch.empty(M, D, device=dev, dtype=cdt)
    dg = torch.empty(1, device=dev, dtype=f32)
    dw = torch.empty(A, device=dev, dtype=f32)
    ws_bytes = nat.lib().ulm_fm_bwd_workspace_bytes(B, T, A, D, cd, saved.numel(), cd)
    ws = torch.empty(max(ws_bytes, 1), device=dev, dtype=torch.uint8)
    call("ulm_block_fm_bwd", ptr(pre), cd, ptr(b32), ptr(denom), ptr(g1), ptr(w32), ptr(saved), saved.numel(), cd,
         ptr(d16), cd, ptr(dqw), cd, ptr(dr), ptr(dv), cd, ptr(dg), ptr(dw), ptr(ws), ws_bytes, B, T, A, D, s)
    del ws, dqw
    dlr = torch.empty(1, device=dev, dtype=f32)
    dlw = torch.empty(A, device=dev, dtype=f32)
    call("ulm_block_params_bwd", ptr(lr), ptr(lw), LOG_W_MIN, LOG_W_MAX, ptr(dg), ptr(dw), A, ptr(dlr), ptr(dlw), s)
    dpre = torch.empty_like(pre)
    dbias = torch.empty(A if key_b is not None else 0, device=dev, dtype=f32)
    dle = torch.empty(1, device=dev, dtype=f32)
    ws_bytes = nat.lib().ulm_addr_bwd_workspace_bytes(M, A)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    call("ulm_addr_bwd", ptr(pre), cd, ptr(b32), ptr(le), None, ptr(denom), ptr(dr), ptr(dpre),
         ptr(dbias if key_b is not None else None), ptr(dle), ptr(ws), ws_bytes, M, A, s)
    del ws, dr
    du = _mm(dpre, kw, f32)
    dkey = _wgrad(dpre, u.view(M, D))
    dhv = _mm(dv, vw, f32)
    dval = _wgrad(dv, h.view(M, D))
    dx = torch.empty(B, T, D, device=dev, dtype=f32)
    dnw = torch.empty(D, device=dev, dtype=f32)
    dcw = torch.empty(D, Kc, device=dev, dtype=f32)
    ws_bytes = nat.lib().ulm_norm_conv_bwd_workspace_bytes(B, T, D, Kc)
    if ws_bytes == 0:
        raise ValueError(f"ulm_norm_conv_bwd: unsupported D={D}")
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    call("ulm_norm_conv_bwd", ptr(x32), nat.ULM_F32, ptr(rstd), ptr(nw), ptr(cw), Kc, ptr(du), nat.ULM_F32, ptr(dhv),
         nat.ULM_F32, ptr(dout), ptr(dx), ptr(dnw), ptr(dcw), ptr(ws), ws_bytes, B, T, D, s)
    return (dx, dnw, dcw.view(conv_w.shape), dkey, dbias, dle.reshape(log_eps.shape), dval, dmu,
            dlr.reshape(log_rate.shape), dlw)


@block_bwd.register_fake
def _block_bwd_fake(dout, x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, rstd, h, u, pre,
                    denom, g1, w32, saved, qw, cdt):
    f32 = torch.float32
    A = key_w.shape[0]
    e = x.new_empty
    return (e(x.shape, dtype=f32), e(norm_w.shape, dtype=f32), e(conv_w.shape, dtype=f32), e(key_w.shape, dtype=f32),
            e(A if key_b is not None else 0, dtype=f32), e(log_eps.shape, dtype=f32), e(val_w.shape, dtype=f32),
            e(mu_w.shape, dtype=f32), e(log_rate.shape, dtype=f32), e(log_w.shape, dtype=f32))


def _block_setup(ctx, inputs, output):
    x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt = inputs
    ctx.save_for_backward(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, *output[1:])
    ctx.cdt = cdt
    ctx.mark_non_differentiable(*output[1:])
    # the extra outputs never get gradients: no zero-filled stand-ins for them
    ctx.set_materialize_grads(False)


def _block_backward(ctx, dout, *_unused):
    if dout is None:
        return (None,) * 12
    saved = ctx.saved_tensors
    key_b = saved[4]
    dx, dnw, dcw, dkey, dbias, dle, dval, dmu, dlr, dlw = block_bwd(dout, *saved, ctx.cdt)
    return dx, dnw, dcw, dkey, (dbias if key_b is not None else None), dle, dval, dmu, dlr, dlw, None, None


torch.library.register_autograd("ulm::block_fwd", _block_backward, setup_context=_block_setup)


def block_eager(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt):
    """unified_block of a plain eager call on the host module, or None."""
    if not _plain_eager():
        return None
    return nat.host().block(norm_eps, cdt, x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w)


def unified_block(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps,
                  cdt=torch.float32):
    """x + mu(w q) + fast of one UnifiedBlock (model.py:77-85) in one fused
    forward and backward. x (B, T, D) fp32; key_w (A, D), mu_w (D, A),
    val_w (D, D), conv_w (D, 1, Kc); log_rate (a scalar) and log_w (A,) are the
    block's parameters: g = -exp(log_rate), w = exp(clamp(log_w, LOG_W_MIN,
    LOG_W_MAX)) (model.py:75, 84) are formed, and differentiated, natively."""
    out = block_eager(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, float(norm_eps), cdt)
    if out is not None:
        return out
    if x.dim() != 3 or x.dtype != torch.float32:
        raise ValueError(f"x must be (B, T, D) fp32, got {tuple(x.shape)} {x.dtype}")
    B, T, D = x.shape
    A = key_w.shape[0]
    if B == 0 or T == 0 or D == 0:
        raise ValueError(f"empty input {tuple(x.shape)}")
    if key_w.shape != (A, D) or mu_w.shape != (D, A) or val_w.shape != (D, D) or log_w.shape != (A,):
        raise ValueError("block weights disagree with x: key (A, D), mu (D, A), val (D, D), log_w (A,)")
    if log_rate.numel() != 1:
        raise ValueError(f"log_rate must hold one value, got {tuple(log_rate.shape)}")
    if conv_w.numel() % D or not 1 <= conv_w.shape[-1] <= 8:
        raise ValueError(f"conv_w must be (D, 1, Kc) with 1 <= Kc <= 8, got {tuple(conv_w.shape)}")
    if cdt not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported GEMM dtype {cdt}")
    nat.require_device(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w)
    return block_fwd(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, float(norm_eps), cdt)[0]


# ---------------------------------------------------------------------------
# per-token decode (model.py:96-111), N sequences at once, fp32

def block_prefill_eager(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps, cdt):
    """block_prefill of a plain eager call on the host module, or None: (out,
    S, c, r_prev, the conv window (B, D, taps - 1) fp32, g, w)."""
    if not _plain_eager():
        return None
    return nat.host().prefill(norm_eps, cdt, x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w)


@torch.no_grad()
def block_prefill(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w, norm_eps,
                  cdt=torch.float32):
    """UnifiedBlock.forward over a prompt (no autograd), fused as in
    block_fwd, plus what decoding continues from: returns (out, S, c,
    r_prev, h) with S (B, D, A) and c (B, A) the fast-memory state after the
    last position (as fm_prefill), r_prev (B, A) fp32 the address at that
    position and h (B, T, D) the normalised input in cdt (its last positions
    fill the conv window). log_rate and log_w are the block's parameters, as
    for unified_block."""
    if x.dim() != 3 or x.dtype != torch.float32:
        raise ValueError(f"x must be (B, T, D) fp32, got {tuple(x.shape)} {x.dtype}")
    B, T, D = x.shape
    A = key_w.shape[0]
    Kc = conv_w.shape[-1]
    M = B * T
    nat.require_device(x, norm_w, conv_w, key_w, key_b, log_eps, val_w, mu_w, log_rate, log_w)
    cd = nat.dtype_code(cdt)
    ws_bytes = nat.lib().ulm_block_fm_prefill_workspace_bytes(B, T, A, D, cd)
    if ws_bytes == 0:
        raise ValueError(f"block_prefill: unsupported sizes B={B} T={T} A={A} D={D}")
    dev = x.device
    s = nat.stream_of(x)
    f32 = torch.float32
    x32 = x.contiguous()
    nw = norm_w.float().contiguous()
    cw = conv_w.float().reshape(D, Kc).contiguous()
    h = torch.empty(B, T, D, device=dev, dtype=cdt)
    u = torch.empty(B, T, D, device=dev, dtype=cdt)
    rstd = torch.empty(B, T, device=dev, dtype=f32)
    call("ulm_norm_conv_fwd", ptr(x32), nat.ULM_F32, ptr(nw), ptr(cw), Kc, float(norm_eps), ptr(h), cd, ptr(u), cd,
         ptr(rstd), B, T, D, s)
    kw, vw, mw = (t.to(cdt).contiguous() for t in (key_w, val_w, mu_w))
    pre = torch.mm(u.view(M, D), kw.t())
    v = torch.mm(h.view(M, D), vw.t())
    del u
    b32 = key_b.float().contiguous() if key_b is not None else None
    le = log_eps.float().reshape(1).contiguous()
    denom = torch.empty(M, device=dev, dtype=f32)
    call("ulm_addr_fwd", ptr(pre), cd, ptr(b32), ptr(le), None, ptr(denom), M, A, s)
    lr = log_rate.float().reshape(1).contiguous()
    lw = log_w.float().contiguous()
    g1 = torch.empty(1, device=dev, dtype=f32)
    w32 = torch.empty(A, device=dev, dtype=f32)
    call("ulm_block_params", ptr(lr), ptr(lw), LOG_W_MIN, LOG_W_MAX, A, ptr(g1), ptr(w32), s)
    qw = torch.empty(M, A, device=dev, dtype=cdt)
    y = torch.empty(M, D, device=dev, dtype=f32)
    S = torch.empty(B, D, A, device=dev, dtype=f32)
    c = torch.empty(B, A, device=dev, dtype=f32)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    call("ulm_block_fm_prefill", ptr(pre), cd, ptr(b32), ptr(denom), ptr(v), cd, ptr(g1), ptr(w32), ptr(qw), cd,
         ptr(x32), ptr(y), ptr(S), ptr(c), ptr(ws), ws_bytes, B, T, A, D, s)
    del ws, v
    out = _addmm_(y, qw, mw.t())
    # the address at the last position, the decode state's r_prev
    pre_last = pre.view(B, T, A)[:, -1].contiguous()
    r_prev = torch.empty(B, A, device=dev, dtype=f32)
    dn_last = torch.empty(B, device=dev, dtype=f32)
    call("ulm_addr_fwd", ptr(pre_last), cd, ptr(b32), ptr(le), ptr(r_prev), ptr(dn_last), B, A, s)
    return out.view(B, T, D), S, c, r_prev, h


def fm_prefill(r, v, g, w):
    """The forward of unified_memory (no autograd) plus the decode state after
    the last position: returns (q, fast, S, c) with S (B, D, A) fp32 =
    sum_s lam^(T-1-s) v_s k_s^T and c (B, A) fp32 = w + sum_s lam^(T-1-s) k_s,
    the state UnifiedBlock.step carries (model.py:88-111)."""
    _check_fm(r, v, g, w)
    B, T, A = r.shape
    D = v.shape[-1]
    r32 = r.float().contiguous()
    vc = v.contiguous()
    g1 = g.float().reshape(1).contiguous()
    w32 = w.float().contiguous()
    vdt = nat.dtype_code(v.dtype)
    ws_bytes = nat.lib().ulm_fm_prefill_workspace_bytes(B, T, A, D, vdt, vdt)
    if ws_bytes == 0:
        raise RuntimeError(f"fm_prefill: unsupported sizes B={B} T={T} A={A} D={D}")
    q = torch.empty_like(r32)
    fast = torch.empty(B, T, D, device=r.device, dtype=v.dtype)
    S = torch.empty(B, D, A, device=r.device, dtype=torch.float32)
    c = torch.empty(B, A, device=r.device, dtype=torch.float32)
    ws = torch.empty(ws_bytes, device=r.device, dtype=torch.uint8)
    call("ulm_fm_prefill", ptr(r32), ptr(vc), vdt, ptr(g1), ptr(w32), ptr(q), ptr(fast), vdt, ptr(S), ptr(c), ptr(ws),
         ws_bytes, B, T, A, D, nat.stream_of(r))
    return q, fast, S, c


def matrix_copies(device, *mats):
    """Contiguous fp32 copies of matrices on `device`, one allocation and one
    launch: 9 us of a 117-position prompt's 154 for a block's three (17 by way of
    torch.cat in Python, which serves tensors the host module leaves alone)."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if device.type == "cuda" and all(m.device == device for m in mats) and _plain_eager():
        out = nat.host().copies(*mats)
        if out is not None:
            return out
    flat = torch.cat([m.detach().to(device=device, dtype=torch.float32).reshape(-1) for m in mats])
    return [t.view(m.shape) for t, m in zip(flat.split([m.numel() for m in mats]), mats)]


def _f32c(t):
    if t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError("decode tensors must be contiguous float32")
    return t


def decode_pre(x, norm_w, conv_w, conv_buf, norm_eps):
    """h = RMSNorm(x), u = causal conv over [conv_buf, h]; conv_buf shifted in place."""
    N, D = x.shape
    Kc = conv_w.shape[-1]
    nat.require_device(x, norm_w, conv_w, conv_buf)
    h = torch.empty_like(x)
    u = torch.empty_like(x)
    call("ulm_decode_pre", ptr(_f32c(x)), ptr(_f32c(norm_w)), ptr(_f32c(conv_w)), ptr(_f32c(conv_buf)), ptr(h), ptr(u),
         N, D, Kc, float(norm_eps), nat.stream_of(x))
    return h, u


def rms_norm(x, weight, eps):
    """RMSNorm of a decode position's x (N, D) in one launch (ulm_decode_pre
    with a conv of one tap, whose output is not used), or None for other
    dtypes and layouts; no autograd."""
    if (not _plain_eager(x, weight) or x.dim() != 2 or x.shape[1:] != weight.shape or x.numel() == 0
            or not (x.is_cuda and x.dtype == weight.dtype == torch.float32 and x.device == weight.device)
            or not (x.is_contiguous() and weight.is_contiguous())):
        return None
    h, u = torch.empty_like(x), torch.empty_like(x)
    call("ulm_decode_pre", ptr(x), ptr(weight), ptr(weight), None, ptr(h), ptr(u), x.shape[0], x.shape[1], 1, float(eps),
         nat.stream_of(x))
    return h


def decode_addr(pre, bias, log_eps, w, g, r_prev, c):
    """r = relu^2 address, c <- lam c + (1-lam) w + r_prev (in place), q = r / c.
    Returns (r, q, w*q)."""
    N, A = pre.shape
    nat.require_device(pre, bias, log_eps, w, g, r_prev, c)
    r = torch.empty_like(pre)
    q = torch.empty_like(pre)
    wq = torch.empty_like(pre)
    call("ulm_decode_addr", ptr(_f32c(pre)), ptr(None if bias is None else _f32c(bias)), ptr(_f32c(log_eps)),
         ptr(_f32c(w)), ptr(_f32c(g)), ptr(_f32c(r_prev)), ptr(_f32c(c)), ptr(r), ptr(q), ptr(wq), N, A,
         nat.stream_of(pre))
    return r, q, wq


def decode_state(S, v, r_prev, q, g, x, ymu, out=None):
    """S <- lam S + v r_prev^T (in place); returns x + S q + ymu."""
    N, D, A = S.shape
    nat.require_device(S, v, r_prev, q, g, x, ymu)
    out = torch.empty_like(x) if out is None else out
    call("ulm_decode_state", ptr(_f32c(S)), ptr(_f32c(v)), ptr(_f32c(r_prev)), ptr(_f32c(q)), ptr(_f32c(g)),
         ptr(_f32c(x)), ptr(_f32c(ymu)), ptr(out), N, D, A, nat.stream_of(S))
    return out


def decode_addr_deferred(pre, bias, log_eps, w, g, r_prev, c, pr, slot, dots):
    """decode_addr for a deferred state: also appends r_prev as pending key
    `slot` of pr (J,N,A) and, with dots, returns the read-out weights
    cj (slot+1, N) of the terms 0 .. slot. Returns (r, q, w*q, cj or None)."""
    N, A = pre.shape
    nat.require_device(pre, bias, log_eps, w, g, r_prev, c, pr)
    r = torch.empty_like(pre)
    q = torch.empty_like(pre)
    wq = torch.empty_like(pre)
    cj = torch.empty(slot + 1, N, device=pre.device, dtype=torch.float32) if dots else None
    call("ulm_decode_addr_deferred", ptr(_f32c(pre)), ptr(None if bias is None else _f32c(bias)), ptr(_f32c(log_eps)),
         ptr(_f32c(w)), ptr(_f32c(g)), ptr(_f32c(r_prev)), ptr(_f32c(c)), ptr(r), ptr(q), ptr(wq), ptr(_f32c(pr)),
         slot, ptr(cj), N, A, nat.stream_of(pre))
    return r, q, wq, cj


def decode_step(x, states, norm_eps):
    """One position of consecutive blocks in two launches
    per block (ulm_decode_step): x (N, D) fp32, states the blocks' deferred
    decode states (dicts of buf, S, c, r_prev, pv and pr, the pending count
    "np" and the parameters "params"), norm_eps their norms' epsilons. The
    states are updated in place. Returns the last block's output, or None,
    with nothing touched, for a call this form does not take (sizes at which
    the per-kernel form is the faster one, other dtypes or layouts, tensors that disagree with each other): the
    per-kernel form serves those, or refuses them."""
    return nat.host().decode_step(x, states, norm_eps) if _plain_eager() else None


def decode_deferred(S, pv, pr, m, flush, q, g, x, ymu, cj=None):
    """One position on a deferred state (S_base, the first m of the pending
    write terms pv (J,N,D), pr (J,N,A), the newest term already appended):
    with flush, S_base <- S_t in place; else S_base is only read, with the
    terms' read-out weights cj (m,N) (formed here by ulm_decode_dots when not
    given). Returns x + S_t q + ymu."""
    N, D, A = S.shape
    nat.require_device(S, pv, pr, q, g, x, ymu)
    out = torch.empty_like(x)
    st = nat.stream_of(S)
    if flush:
        call("ulm_decode_flush", ptr(_f32c(S)), ptr(_f32c(pv)), ptr(_f32c(pr)), m, ptr(_f32c(q)), ptr(_f32c(g)),
             ptr(_f32c(x)), ptr(_f32c(ymu)), ptr(out), N, D, A, st)
    else:
        if cj is None:
            cj = torch.empty(m, N, device=S.device, dtype=torch.float32)
            call("ulm_decode_dots", ptr(_f32c(pr)), ptr(_f32c(q)), ptr(cj), m, N, A, st)
        call("ulm_decode_read", ptr(_f32c(S)), ptr(_f32c(pv)), ptr(_f32c(cj)), m, ptr(_f32c(q)), ptr(_f32c(g)),
             ptr(_f32c(x)), ptr(_f32c(ymu)), ptr(out), N, D, A, st)
    return out


# ---------------------------------------------------------------------------
# log probabilities of given tokens (F.cross_entropy over the logits,
# model.py:160-161), with each row's entropy and its largest entries

TokenLogprobs = namedtuple("TokenLogprobs", "logprob entropy top_logprobs top_tokens")
MAX_TOP = 64   # ulm_token_logprobs_max_top()


def _int_tokens(tokens):
    """Token ids as the kernels read them."""
    return tokens.to(torch.int64).contiguous()


def _rows(logits):
    """(tensor, inner, outer stride, row stride): the rows of (..., V) logits as
    the kernels address them, without a copy where the last dimension is dense
    and the leading ones collapse into two."""
    dims = [[n, st] for n, st in zip(logits.shape[:-1], logits.stride()[:-1]) if n != 1]
    groups = []
    for n, st in dims:
        if groups and groups[-1][1] == n * st:
            groups[-1] = [groups[-1][0] * n, st]
        else:
            groups.append([n, st])
    V = logits.shape[-1]
    if len(groups) > 2 or (V > 1 and logits.stride(-1) != 1):
        return logits.contiguous(), max(1, logits.numel() // V), 0, V
    if len(groups) == 2:
        return logits, groups[1][0], groups[0][1], groups[1][1]
    return (logits, groups[0][0], 0, groups[0][1]) if groups else (logits, 1, 0, V)


@torch.library.custom_op("ulm::token_logprobs", mutates_args=())
def token_logprobs_fwd(logits: Tensor, tokens: Tensor, top: int,
                       ignore_index: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(logprob, entropy, top_logprobs, top_tokens, stats (..., 2)): ulm_token_logprobs."""
    lead, V = logits.shape[:-1], logits.shape[-1]
    f32 = dict(device=logits.device, dtype=torch.float32)
    logprob, entropy = torch.empty(lead, **f32), torch.empty(lead, **f32)
    top_logprobs = torch.empty(*lead, top, **f32)
    top_tokens = torch.empty(*lead, top, device=logits.device, dtype=torch.int64)
    stats = torch.empty(*lead, 2, **f32)
    rows = logprob.numel()
    if rows:
        with torch.cuda.device(logits.device):
            x, inner, outer_stride, row_stride = _rows(logits)
            tok = _int_tokens(tokens)
            ws_bytes = nat.lib().ulm_token_logprobs_workspace_bytes(rows, V, top, nat.dtype_code(logits.dtype))
            ws = torch.empty(max(ws_bytes, 1), device=logits.device, dtype=torch.uint8)
            call("ulm_token_logprobs", ptr(x), nat.dtype_code(logits.dtype), ptr(tok), rows, inner, outer_stride,
                 row_stride, V, top, ignore_index, ptr(logprob), ptr(entropy), ptr(top_logprobs), ptr(top_tokens),
                 ptr(stats), ptr(ws), ws_bytes, nat.stream_of(logits))
    return logprob, entropy, top_logprobs, top_tokens, stats


@token_logprobs_fwd.register_fake
def _token_logprobs_fake(logits, tokens, top, ignore_index):
    lead = logits.shape[:-1]
    e = lambda *shape, dtype=torch.float32: logits.new_empty(*shape, dtype=dtype)  # noqa: E731
    return e(lead), e(lead), e((*lead, top)), e((*lead, top), dtype=torch.int64), e((*lead, 2))


@torch.library.custom_op("ulm::token_logprobs_bwd", mutates_args=())
def token_logprobs_bwd(logits: Tensor, tokens: Tensor, top: int, ignore_index: int, stats: Tensor, entropy: Tensor,
                       top_tokens: Tensor, dlogprob: Optional[Tensor], dentropy: Optional[Tensor],
                       dtop: Optional[Tensor]) -> Tensor:
    """The logits' gradient in their dtype, dense: ulm_token_logprobs_bwd."""
    V = logits.shape[-1]
    out = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    rows = out.numel() // V
    if rows:
        with torch.cuda.device(logits.device):
            x, inner, outer_stride, row_stride = _rows(logits)
            tok = _int_tokens(tokens)
            up = [None if t is None or t.numel() == 0 else t.float().contiguous() for t in (dlogprob, dentropy, dtop)]
            call("ulm_token_logprobs_bwd", ptr(x), nat.dtype_code(logits.dtype), ptr(tok), rows, inner, outer_stride,
                 row_stride, V, top, ignore_index, ptr(stats.contiguous()), ptr(entropy.contiguous()),
                 ptr(top_tokens.contiguous()), *map(ptr, up), ptr(out), nat.stream_of(logits))
    return out


@token_logprobs_bwd.register_fake
def _token_logprobs_bwd_fake(logits, tokens, top, ignore_index, stats, entropy, top_tokens, dlogprob, dentropy, dtop):
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _token_logprobs_setup(ctx, inputs, output):
    logits, tokens, ctx.top, ctx.ignore_index = inputs
    _, entropy, _, top_tokens, stats = output
    ctx.save_for_backward(logits, tokens, stats, entropy, top_tokens)
    ctx.mark_non_differentiable(top_tokens, stats)
    ctx.set_materialize_grads(False)


def _token_logprobs_backward(ctx, dlogprob, dentropy, dtop, _dtokens, _dstats):
    if dlogprob is None and dentropy is None and dtop is None:
        return None, None, None, None
    logits, tokens, stats, entropy, top_tokens = ctx.saved_tensors
    dx = token_logprobs_bwd(logits, tokens, ctx.top, ctx.ignore_index, stats, entropy, top_tokens, dlogprob, dentropy,
                            dtop)
    return dx, None, None, None


torch.library.register_autograd("ulm::token_logprobs", _token_logprobs_backward, setup_context=_token_logprobs_setup)


def _check_capture(leaf):
    """What the host module refuses of a call that is being captured, for the calls it does not take."""
    if not torch.compiler.is_compiling() and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        nat.host().check_capture(leaf)


def _check_tokens(tokens):
    if not isinstance(tokens, torch.Tensor):
        raise TypeError("tokens must be a tensor")
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise TypeError(f"tokens must be an integer tensor, got {tokens.dtype}")


def token_logprobs(logits, tokens, top=0, ignore_index=-1):
    """Log probabilities of `tokens` (...) under `logits` (..., V), as TokenLogprobs:

      logprob      (...)      x_t - ln sum_i exp(x_i), t the token; 0, without a gradient, where t is
                              ignore_index (F.cross_entropy's, -1 as in UnifiedLM.forward); NaN for any
                              other token outside [0, V)
      entropy      (...)      -sum_i p_i ln p_i
      top_logprobs (..., top) the `top` most likely tokens' log probabilities (at most 64),
      top_tokens   (..., top) and those tokens, the lower first on ties

    fp32 from fp32, bf16 or fp16 logits, differentiable in them through the first three (dlogits in the
    logits' dtype). Masked logits (-inf, or any large negative number) have probability 0; a row of -inf
    alone has logprob and top_logprobs -inf, entropy 0 and no gradient. Equal calls give equal bits; a row's
    last bits may differ between calls of up to 512 rows and of more, which share a row among more or fewer
    threads. Any view whose last dimension is dense is read in
    place (logits[:, :-1], say). The loss of a training step is -logprob summed over the tokens
    that count."""
    if _plain_eager():
        out = nat.host().token_logprobs(logits, tokens, top, ignore_index)
        if out is not None:
            return TokenLogprobs._make(out)
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a tensor")
    _check_float("logits", logits)
    _check_tokens(tokens)
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be (..., V), got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} must have the logits' leading shape, {tuple(logits.shape)}")
    V = logits.shape[-1]
    top, ignore_index = operator.index(top), operator.index(ignore_index)
    if not 0 <= top <= min(V, MAX_TOP):
        raise ValueError(f"top must be between 0 and {min(V, MAX_TOP)}, got {top}")
    if V > 1 << 30 or (top and V > 1 << 22):
        raise ValueError(f"at most 2^30 columns, 2^22 with alternatives, got {V}")
    nat.dtype_code(logits.dtype)
    nat.require_device(logits, tokens)
    _check_capture(logits)
    return TokenLogprobs(*token_logprobs_fwd(logits, tokens, top, ignore_index)[:4])


# ---------------------------------------------------------------------------
# embedding lookup with scaling (nn.Embedding, model.py:117, 150)

@torch.library.custom_op("ulm::embed_fwd", mutates_args=())
def embed_fwd(weight: Tensor, tokens: Tensor, scale: float) -> Tensor:
    """scale W[tokens] (..., D) in the weight's dtype: ulm_embed_fwd."""
    V, D = weight.shape
    out = torch.empty(*tokens.shape, D, device=weight.device, dtype=weight.dtype)
    if tokens.numel():
        with torch.cuda.device(weight.device):
            w, tok = weight.contiguous(), _int_tokens(tokens)
            call("ulm_embed_fwd", ptr(w), nat.dtype_code(weight.dtype), ptr(tok), tok.numel(), V, D, scale, ptr(out),
                 nat.stream_of(weight))
    return out


@embed_fwd.register_fake
def _embed_fwd_fake(weight, tokens, scale):
    return weight.new_empty(*tokens.shape, weight.shape[1])


@torch.library.custom_op("ulm::embed_bwd", mutates_args=())
def embed_bwd(dout: Tensor, tokens: Tensor, V: int, scale: float) -> Tensor:
    """The weight's gradient (V, D) in dout's dtype: ulm_embed_bwd."""
    D = dout.shape[-1]
    dw = torch.empty(V, D, device=dout.device, dtype=dout.dtype)
    if not tokens.numel():
        return dw.zero_()
    with torch.cuda.device(dout.device):
        d, tok = dout.contiguous(), _int_tokens(tokens)
        ws_bytes = nat.lib().ulm_embed_bwd_workspace_bytes(tok.numel(), V, D)
        ws = torch.empty(max(ws_bytes, 1), device=dout.device, dtype=torch.uint8)
        call("ulm_embed_bwd", ptr(d), nat.dtype_code(dout.dtype), ptr(tok), tok.numel(), V, D, scale, ptr(dw), ptr(ws),
             ws_bytes, nat.stream_of(dout))
    return dw


@embed_bwd.register_fake
def _embed_bwd_fake(dout, tokens, V, scale):
    return dout.new_empty(V, dout.shape[-1])


def _embed_setup(ctx, inputs, output):
    weight, tokens, ctx.scale = inputs
    ctx.V, ctx.dtype = weight.shape[0], weight.dtype
    ctx.save_for_backward(tokens)
    ctx.set_materialize_grads(False)


def _embed_backward(ctx, dout):
    if dout is None:
        return None, None, None
    tokens, = ctx.saved_tensors
    return embed_bwd(dout.to(ctx.dtype), tokens, ctx.V, ctx.scale), None, None


torch.library.register_autograd("ulm::embed_fwd", _embed_backward, setup_context=_embed_setup)


def embedding(weight, tokens, scale=1.0):
    """scale * weight[tokens]: weight (V, D) fp32, bf16 or fp16, tokens (...) integer, the result
    (..., D) in the weight's dtype, multiplied in fp32 and rounded from it. A token outside [0, V) gives a row of NaN.
    The weight's gradient is dense, in its dtype: each row the fp32 sum of its tokens' gradients in
    an order that the tokens alone fix, so that equal inputs give equal bits; tokens outside [0, V) add
    nothing."""
    if _plain_eager():
        out = nat.host().embedding(weight, tokens, scale)
        if out is not None:
            return out
    if not isinstance(weight, torch.Tensor):
        raise TypeError("weight must be a tensor")
    if isinstance(scale, torch.Tensor):
        raise TypeError("scale must be a number")
    _check_float("weight", weight)
    _check_tokens(tokens)
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be a non-empty (V, D), got {tuple(weight.shape)}")
    if weight.shape[0] > 1 << 28 or weight.shape[1] > 1 << 20 or tokens.numel() > 1 << 30:
        raise ValueError(f"weight at most 2^28 x 2^20 and 2^30 tokens, got {tuple(weight.shape)} and {tokens.numel()}")
    nat.dtype_code(weight.dtype)
    nat.require_device(weight, tokens)
    _check_capture(weight)
    return embed_fwd(weight, tokens, float(scale))


# ---------------------------------------------------------------------------
# the gradients' global norm and clipping (train.py, before the optimizer's step)

def _norm_type(norm_type):
    code = nat.NORM_TYPES.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return code


def _check_grads(grads, what="gradient"):
    """The tensors of a norm: a tensor or an iterable of them, on one device, of the three types."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    for t in grads:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"every {what} must be a tensor, got {type(t).__name__}")
        if t.layout != torch.strided:
            raise TypeError(f"every {what} must be strided, got {t.layout}")
        nat.dtype_code(t.dtype)
    nat.require_device(*grads)
    return grads


def _dense(t):
    """Whether t's elements fill one region of memory, each once."""
    if t.is_contiguous():
        return True
    want = 1
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _table(pairs):
    table = (nat.Grad * max(1, len(pairs)))()
    for g, (src, dst) in zip(table, pairs):
        g.src, g.numel, g.src_dtype = src.data_ptr(), src.numel(), nat.dtype_code(src.dtype)
        if dst is not None:
            g.dst, g.dst_dtype = dst.data_ptr(), nat.dtype_code(dst.dtype)
    return table


def _run_norm(entry, pairs, device, norm_type, *bound):
    norm = torch.empty((), device=device, dtype=torch.float32)
    table = _table(pairs)
    ws_bytes = nat.lib().ulm_grad_norm_workspace_bytes(table, len(pairs))
    ws = torch.empty(ws_bytes, device=device, dtype=torch.uint8)
    call(entry, table, len(pairs), _norm_type(norm_type), *bound, ptr(norm), ptr(ws), ws_bytes, nat.stream_of(norm))
    return norm


@torch.library.custom_op("ulm::grad_norm", mutates_args=())
def _grad_norm_op(grads: list[Tensor], norm_type: float) -> Tensor:
    """ulm_grad_norm over at least one tensor."""
    with torch.cuda.device(grads[0].device):
        return _run_norm("ulm_grad_norm", [(t if _dense(t) else t.contiguous(), None) for t in grads],
                         grads[0].device, norm_type)


@_grad_norm_op.register_fake
def _grad_norm_fake(grads, norm_type):
    return grads[0].new_empty((), dtype=torch.float32)


def _check_regions(grads, out):
    """Refuses results whose memory, from the first element to the last, overlaps
    another result's or another gradient's."""
    spans = []
    for g, o in zip(grads, out):
        if o.numel() == 0:
            continue
        if any(st == 0 and n > 1 for n, st in zip(o.shape, o.stride())):
            raise ValueError("a result's elements share memory")
        span = lambda t: (t.data_ptr(), t.data_ptr() + t.element_size() * (  # noqa: E731
            1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))))
        spans.append((*span(o), True))
        if g is not o and (g.data_ptr() != o.data_ptr() or g.dtype != o.dtype or g.stride() != o.stride()):
            spans.append((*span(g), False))
    written = read = 0
    for start, end, is_out in sorted(spans):
        if start < written or (is_out and start < read):
            raise ValueError("results must not share memory with each other or with other gradients")
        written = max(written, end) if is_out else written
        read = max(read, end)


def _clip_impl(grads, out, max_norm, norm_type):
    _check_regions(grads, out)
    with torch.cuda.device(grads[0].device):
        pairs, late = [], []
        for g, o in zip(grads, out):
            if _dense(o) and g.stride() == o.stride():
                pairs.append((g, o))
                continue
            src = g.contiguous()
            dst = o if o.is_contiguous() else torch.empty_like(o, memory_format=torch.contiguous_format)
            if dst is not o:
                late.append((o, dst))
            pairs.append((src, dst))
        norm = _run_norm("ulm_clip_grads", pairs, grads[0].device, norm_type, max_norm)
        for o, dst in late:
            o.copy_(dst)
    return norm


@torch.library.custom_op("ulm::clip_grads", mutates_args={"out"})
def _clip_op(grads: list[Tensor], out: list[Tensor], max_norm: float, norm_type: float) -> Tensor:
    """ulm_clip_grads over at least one tensor, into `out`; returns the norm."""
    return _clip_impl(grads, out, max_norm, norm_type)


@torch.library.custom_op("ulm::clip_grads_", mutates_args={"grads"})
def _clip_op_(grads: list[Tensor], max_norm: float, norm_type: float) -> Tensor:
    """ulm_clip_grads over at least one tensor, in place; returns the norm."""
    return _clip_impl(grads, grads, max_norm, norm_type)


@_clip_op.register_fake
def _clip_fake(grads, out, max_norm, norm_type):
    return grads[0].new_empty((), dtype=torch.float32)


@_clip_op_.register_fake
def _clip_fake_(grads, max_norm, norm_type):
    return grads[0].new_empty((), dtype=torch.float32)


@torch.no_grad()
def grad_norm(grads, norm_type=2.0):
    """The norm of all elements of `grads` (a tensor or an iterable of them) taken together, a 0-d fp32
    tensor: the root of the sum of squares, summed in double, or with norm_type inf the largest |g|."""
    if _plain_eager():
        out = nat.host().grad_norm(grads, norm_type)
        if out is not None:
            return out
    _norm_type(norm_type)
    grads = _check_grads(grads)
    return _grad_norm_op(grads, float(norm_type)) if grads else torch.zeros(())


@torch.no_grad()
def clip_grads(grads, max_norm, out=None, norm_type=2.0):
    """(norm, clipped): the norm of all `grads` (grad_norm) and every gradient times
    min(1, max_norm / (norm + 1e-6)), in fp32 and rounded once to the result's dtype. `out` is a list of
    tensors of the gradients' shapes to write, each of the three types (gradients in bf16 clipped into
    the optimizer's fp32 buffers, say); out = grads clips in place, leaving the gradients as they
    are where the norm is within the bound; None makes new tensors of the gradients' dtypes.
    Nothing waits for the GPU. A NaN among the gradients makes the norm and all of them NaN.
    Results share no memory, from their first to their last elements, with each other or with
    another gradient."""
    if _plain_eager():
        done = nat.host().clip_grads(grads, max_norm, out, norm_type)
        if done is not None:
            return done
    _norm_type(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    in_place = out is grads
    grads = _check_grads(grads)
    if out is None:
        out = [torch.empty_like(t) for t in grads]
    else:
        out = grads if in_place else _check_grads(out, "result")
    if len(out) != len(grads) or any(o.shape != g.shape for o, g in zip(out, grads)):
        raise ValueError("out must hold a tensor of each gradient's shape")
    if not grads:
        return torch.zeros(()), out
    nat.require_device(*grads, *out)
    if in_place:
        return _clip_op_(grads, max_norm, float(norm_type)), out
    return _clip_op(grads, out, max_norm, float(norm_type)), out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """The gradients of `parameters` (a tensor or an iterable; those without one are passed over) clipped
    in place to a joint norm of max_norm (clip_grads); returns the norm they had. With
    error_if_nonfinite, a norm that is not finite raises before anything is changed (this waits for the GPU)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if error_if_nonfinite:
        norm = grad_norm([p.grad for p in parameters if p.grad is not None], norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the gradients' norm is {norm.item()}; nothing was clipped")
    if _plain_eager():
        norm = nat.host().clip_parameters(parameters, max_norm, norm_type)
        if norm is not None:
            return norm
    grads = [p.grad for p in parameters if p.grad is not None]
    return clip_grads(grads, max_norm, out=grads, norm_type=norm_type)[0]
