"""The two ends of a training, scoring or decoding step, as timed cases.

Six kinds, by what a program has done:

  score   token_logprobs, forward only: given tokens' log probabilities, entropies and alternatives
  loss    token_logprobs, forward and backward: the training loss's outputs and the logits' gradient
  lookup  embedding, forward only: the inputs of a decode position
  embed   embedding, forward and backward: the rows of a training batch and the weight's gradient
  clip    clip_grads of a whole model's gradients into buffers of their own
  keep    clip_grad_norm_ of a whole model's gradients whose norm is below the bound

`own` false computes the plain form in elementary torch operations, true calls the package.
"""
import math
import os
import sys

import numpy as np
import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unifiedlm.c_amd")

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -1
TAPS = 4
CLIP_EPS = 1e-6   # added to the norm before the bound is divided by it


def listed():
    return [
        # one user's decode position: the chosen token's log probability and five alternatives
        dict(name="score-1", kind="score", B=1, T=1, V=32000, dtype="fp32", top=5, masked=0.0, ahead=False),
        # a batch of decode positions with twenty alternatives each
        dict(name="score-256", kind="score", B=256, T=1, V=32000, dtype="fp32", top=20, masked=0.0, ahead=False),
        # prompts scored by their own next tokens: rows of a (B, T, V) tensor without its last positions
        dict(name="score-prompts", kind="score", B=16, T=1024, V=32000, dtype="bf16", top=0, masked=0.0, ahead=True),
        # a large vocabulary, a part of it masked away
        dict(name="score-large-vocab", kind="score", B=4, T=128, V=131072, dtype="bf16", top=10, masked=0.3, ahead=False),
        # the loss of the 110M shape's training batch under bf16 autocast
        dict(name="loss-110M", kind="loss", B=16, T=1024, V=32000, dtype="bf16", top=0, masked=0.0, ahead=False,
             entropy=False),
        # a small ragged batch with an odd vocabulary, an entropy bonus and a loss on the alternatives
        dict(name="loss-ragged", kind="loss", B=3, T=331, V=31999, dtype="fp16", top=8, masked=0.1, ahead=False,
             entropy=True),
        # a batch of decode positions
        dict(name="lookup-256", kind="lookup", N=256, V=32000, D=768, dtype="fp32", scaled=False, skew=1.0),
        # the 110M shape's training batch: text's skewed token frequencies
        dict(name="embed-110M", kind="embed", N=16384, V=32000, D=768, dtype="fp32", scaled=False, skew=1.0),
        # many short ragged rows, odd widths, the rows scaled by sqrt(D)
        dict(name="embed-ragged", kind="embed", N=3241, V=4099, D=289, dtype="bf16", scaled=True, skew=1.0),
        # the smallest model in use: launches and latency
        dict(name="keep-260K", kind="keep", L=5, D=64, A=128, V=512, src="fp32", dst="fp32"),
        # the default model's gradients in bf16, clipped into fp32 for the optimizer
        dict(name="clip-15M", kind="clip", L=12, D=288, A=712, V=32000, src="bf16", dst="fp32"),
        # the 110M shape's gradients
        dict(name="clip-110M", kind="clip", L=12, D=768, A=3072, V=32000, src="fp32", dst="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "score", "loss", "loss", "lookup", "embed", "embed", "clip", "keep"])
    if kind in ("score", "loss"):
        V = _log_int(rng, 200, 131072)
        top = rng.choice([0, 0, 1, 5, rng.randint(2, 32)])
        most = 16384 * 32000 // (8 if top else 1)   # alternatives cost the plain form a sort
        rows = _log_int(rng, 1, max(1, min(16384, most // V)))
        B = min(rows, _log_int(rng, 1, 32))
        T = max(1, rows // B)
        dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        if dtype == "fp32":   # twice the bytes
            T = max(1, T // 2)
        case = dict(kind=kind, B=B, T=T, V=V, dtype=dtype, top=top,
                    masked=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]), ahead=T > 1 and rng.random() < 0.4)
        return case if kind == "score" else dict(case, entropy=rng.random() < 0.4)
    if kind in ("lookup", "embed"):
        D = _log_int(rng, 16, 768)
        N = _log_int(rng, 1, 512) if kind == "lookup" else _log_int(rng, 16, 16384)
        return dict(kind=kind, N=N, V=_log_int(rng, 100, 32000), D=D, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    scaled=rng.random() < 0.5, skew=round(rng.uniform(0.0, 1.3), 2))
    return dict(kind=kind, L=rng.randint(1, 12), D=_log_int(rng, 48, 768), A=_log_int(rng, 64, 2048),
                V=_log_int(rng, 256, 32000), src=rng.choice(["fp32", "fp32", "bf16", "fp16"]), dst="fp32")


# ---- inputs, from the seed alone

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)


def _logit_inputs(case, seed):
    """Logits (B, T, V) as a trained model gives them, the tokens scored, and upstream gradients.

    A row is normal noise with a handful of likely tokens well above it; the token scored is one
    of those more often than not, and one row in twenty belongs to padding."""
    gen = _gen(seed)
    B, T, V, dt = case["B"], case["T"], case["V"], DTYPES[case["dtype"]]
    full = T + 1 if case["ahead"] else T
    logits = torch.empty(B, full, V, device=DEV, dtype=dt)
    rows = logits.view(B * full, V)
    n_likely = min(8, V)
    likely = torch.randint(0, V, (B * full, n_likely), generator=gen, device=DEV)
    lift = 4.0 + 5.0 * torch.rand(B * full, n_likely, generator=gen, device=DEV)
    hidden = None
    if case["masked"]:   # tokens that no row may take
        hidden = torch.rand(V, generator=gen, device=DEV) < case["masked"]
        hidden[: V // 4 + 1] = False
    at_once = max(1, (1 << 27) // V)
    for i in range(0, B * full, at_once):
        x = torch.randn(min(at_once, B * full - i), V, generator=gen, device=DEV).mul_(1.5)
        x.scatter_add_(1, likely[i:i + at_once], lift[i:i + at_once])
        if hidden is not None:
            x.masked_fill_(hidden, -math.inf)
        rows[i:i + at_once] = x
    allowed = torch.arange(V, device=DEV) if hidden is None else torch.nonzero(~hidden).flatten()
    tokens = allowed[torch.randint(0, allowed.numel(), (B * full,), generator=gen, device=DEV)]
    take = torch.rand(B * full, generator=gen, device=DEV) < 0.7
    if hidden is not None:
        take &= ~hidden[likely[:, 0]]
    tokens = torch.where(take, likely[:, 0], tokens)
    if B * full > 1:
        tokens[torch.rand(B * full, generator=gen, device=DEV) < 0.05] = IGNORE
    tokens = tokens.view(B, full)
    if case["ahead"]:
        tokens = torch.cat([tokens[:, 1:], tokens[:, :1]], 1)[:, :-1].contiguous()
    up = None
    if case["kind"] == "loss":
        # the mean over the tokens that count; in fp16 scaled up, as such training does
        each = (1024.0 if dt == torch.float16 else 1.0) / max(1, int((tokens != IGNORE).sum()))
        up = [torch.full((B, T), -each, device=DEV), None, None]
        if case["entropy"]:
            up[1] = torch.full((B, T), -0.01 * each, device=DEV)
        if case["top"]:
            up[2] = torch.randn(B, T, case["top"], generator=gen, device=DEV).mul_(0.1 * each)
    return logits[:, :T], tokens, up


def _frequencies(case):
    """Token frequencies falling with the rank's power `skew`."""
    f = 1.0 / (np.arange(case["V"]) + 2.7) ** case["skew"]
    return f / f.sum()


def _embed_inputs(case, seed):
    gen = _gen(seed)
    N, V, D, dt = case["N"], case["V"], case["D"], DTYPES[case["dtype"]]
    cdf = torch.from_numpy(np.cumsum(_frequencies(case))).to(DEV)
    rank = torch.searchsorted(cdf, torch.rand(N, generator=gen, device=DEV, dtype=torch.float64)).clamp_(max=V - 1)
    tokens = torch.randperm(V, generator=gen, device=DEV)[rank]
    weight = torch.randn(V, D, generator=gen, device=DEV).mul_(0.02).to(dt)
    dout = torch.randn(N, D, generator=gen, device=DEV).to(dt) if case["kind"] == "embed" else None
    return weight, tokens, dout, math.sqrt(D) if case["scaled"] else 1.0


def _shapes(case):
    """A model's parameters: the tied embedding, the final norm, and nine tensors a block."""
    L, D, A, V = (case[k] for k in "LDAV")
    return [(V, D), (D,)] + [s for _ in range(L) for s in
                             ((D,), (D, 1, TAPS), (A, D), (A,), (D, A), (D, D), (A,), (), ())]


def _clip_inputs(case, seed):
    """Gradients whose sizes differ by orders of magnitude from tensor to tensor, and the bound on their norm:
    a third of it (clip) or three times it (keep), from the sizes alone."""
    gen = _gen(seed)
    grads, total = [], 0.0
    for i, s in enumerate(_shapes(case)):
        std = 10.0 ** (-1 - i % 4)
        grads.append(torch.randn(s, generator=gen, device=DEV).mul_(std).to(DTYPES[case["src"]]))
        total += math.prod(s) * std * std
    return grads, math.sqrt(total) * (3.0 if case["kind"] == "keep" else 1.0 / 3.0)


def _flat(shapes, dtype):
    """One buffer and its views, tensor after tensor: what a program that reduces gradients in buckets keeps."""
    flat = torch.zeros(sum(math.prod(s) for s in shapes), device=DEV, dtype=dtype)
    return flat, [t.view(s) for t, s in zip(flat.split([math.prod(s) for s in shapes]), shapes)]


def prepare(case, seed):
    kind = case["kind"]
    state = dict(kind=kind)
    if kind in ("score", "loss"):
        logits, tokens, up = _logit_inputs(case, seed)
        if kind == "loss":
            logits = logits.detach().requires_grad_(True)
        state.update(logits=logits, tokens=tokens, top=case["top"], up=up)
    elif kind in ("lookup", "embed"):
        weight, tokens, dout, scale = _embed_inputs(case, seed)
        state.update(weight=weight.requires_grad_(kind == "embed"), tokens=tokens, dout=dout, scale=scale)
    else:
        grads, bound = _clip_inputs(case, seed)
        state.update(bound=bound)
        if kind == "keep":   # parameters of no use here but for the gradients they hold, views of a bucket
            state["flat"], views = _flat(_shapes(case), DTYPES[case["src"]])
            state["params"] = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
            for p, v, g in zip(state["params"], views, grads):
                p.grad = v.copy_(g)
        else:   # gradients as the backward allocated them, an optimizer's flat buffer
            state["grads"] = grads
            state["flat"], state["out"] = _flat(_shapes(case), DTYPES[case["dst"]])
    return state


# ---- one pass

def _named(outs, **more):
    return dict({k: t for k, t in zip(("logprob", "entropy", "top_logprobs", "top_tokens"), outs)}, **more)


def _plain_logprobs(logits, tokens, top, up):
    """The four outputs and, with `up`, the logits' gradient."""
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    logs = torch.log(s)
    valid = tokens != IGNORE
    at = tokens.clamp(min=0)[..., None]
    logprob = torch.where(valid, (d.gather(-1, at) - logs)[..., 0], 0.0)
    masked = d == -math.inf
    entropy = logs[..., 0] - (e * d.masked_fill(masked, 0.0)).sum(-1) / s[..., 0]
    if top:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
    else:
        ids = torch.empty(*tokens.shape, 0, device=x.device, dtype=torch.int64)
    top_logprobs = d.gather(-1, ids) - logs
    if up is None:
        return (logprob, entropy, top_logprobs, ids), None
    a, h, c = up
    a = torch.where(valid, a, 0.0)[..., None]
    p = e / s
    dx = -p * (a if c is None else a + c.sum(-1, keepdim=True))
    if h is not None:
        dx -= h[..., None] * p * ((d - logs).masked_fill(masked, 0.0) + entropy[..., None])
    dx.scatter_add_(-1, at, a)
    if c is not None:
        dx.scatter_add_(-1, ids, c)
    return (logprob, entropy, top_logprobs, ids), dx.to(logits.dtype)


def _plain_norm(grads):
    return torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()


@torch.no_grad()
def _plain(state):
    kind = state["kind"]
    if kind in ("score", "loss"):
        outs, dx = _plain_logprobs(state["logits"], state["tokens"], state["top"], state["up"])
        return _named(outs) if dx is None else _named(outs, dlogits=dx)
    if kind in ("lookup", "embed"):
        weight, tokens, dout = state["weight"], state["tokens"], state["dout"]
        out = (weight[tokens].float() * state["scale"]).to(weight.dtype)
        if dout is None:
            return dict(out=out)
        dw = torch.zeros(weight.shape, device=weight.device).index_add_(0, tokens, dout.float())
        return dict(out=out, dweight=(dw * state["scale"]).to(weight.dtype))
    grads = [p.grad for p in state["params"]] if kind == "keep" else state["grads"]
    norm = _plain_norm(grads)
    coef = (state["bound"] / (norm + CLIP_EPS)).clamp(max=1.0)
    out = grads if kind == "keep" else state["out"]
    for o, g in zip(out, grads):
        o.copy_(g.float() * coef)
    return dict(norm=norm, grads=state["flat"])


def run(state):
    if not own:
        return _plain(state)
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import kernel
    kind = state["kind"]
    if kind == "score":
        return _named(kernel.token_logprobs(state["logits"], state["tokens"], state["top"]))
    if kind == "loss":
        outs = kernel.token_logprobs(state["logits"], state["tokens"], state["top"])
        used = [(o, u) for o, u in zip(outs, state["up"]) if u is not None]
        dx, = torch.autograd.grad([o for o, _ in used], [state["logits"]], [u for _, u in used])
        return _named([o.detach() for o in outs], dlogits=dx)
    if kind == "lookup":
        return dict(out=kernel.embedding(state["weight"], state["tokens"], state["scale"]))
    if kind == "embed":
        out = kernel.embedding(state["weight"], state["tokens"], state["scale"])
        dw, = torch.autograd.grad([out], [state["weight"]], [state["dout"]])
        return dict(out=out.detach(), dweight=dw)
    if kind == "keep":
        norm = kernel.clip_grad_norm_(state["params"], state["bound"])
        return dict(norm=norm, grads=state["flat"])
    norm, _ = kernel.clip_grads(state["grads"], state["bound"], out=state["out"])
    return dict(norm=norm, grads=state["flat"])


# ---- what one pass cannot do without

def work(case):
    kind = case["kind"]
    if kind in ("score", "loss"):
        rows, V, b = case["B"] * case["T"], case["V"], 4 if case["dtype"] == "fp32" else 2
        # the logits, the tokens; log probability, entropy, alternatives
        bytes_ = rows * (V * b + 8 + 8 + 12 * case["top"])
        flops = rows * V * 7
        if kind == "loss":   # the logits' gradient and the upstream ones
            bytes_ += rows * (V * b + 4 + 4 * case["entropy"] + 4 * case["top"])
            flops += rows * V * (6 if case["entropy"] else 4)
        return {"bytes": bytes_, "flops": flops}
    if kind in ("lookup", "embed"):
        N, V, D, b = case["N"], case["V"], case["D"], 4 if case["dtype"] == "fp32" else 2
        rows = float(-np.expm1(N * np.log1p(-_frequencies(case))).sum()) if V > 1 else 1.0   # distinct tokens expected
        bytes_, flops = rows * D * b + N * D * b + 8 * N, N * D * case["scaled"]
        if kind == "embed":
            bytes_, flops = bytes_ + N * D * b + V * D * b, flops + N * D + rows * D * case["scaled"]
        return {"bytes": int(bytes_), "flops": int(flops)}
    n = sum(math.prod(s) for s in _shapes(case))
    src, dst = (4 if case[k] == "fp32" else 2 for k in ("src", "dst"))
    return {"bytes": n * src + (n * dst if kind == "clip" else 0) + 4, "flops": n * (3 if kind == "clip" else 2)}


# ---- the same outputs in 64 bits

def _exact_rows(x, tokens, top, up):
    """One block of rows (n, V): log-softmax by torch.logsumexp, the alternatives by value and index."""
    x = x.double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(-1)
    keep = (tokens != IGNORE).double()
    at = torch.where(tokens == IGNORE, 0, tokens)
    lp = logp[torch.arange(x.shape[0], device=x.device), at]
    outs = [torch.where(tokens == IGNORE, 0.0, lp), H]
    left, ids = x.clone(), []
    for _ in range(top):   # argmax by the first of the largest, then taken out
        best = (left == left.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1)
        ids.append(best)
        left[torch.arange(x.shape[0], device=x.device), best] = -math.inf
    ids = torch.stack(ids, -1) if top else torch.empty(x.shape[0], 0, device=x.device, dtype=torch.int64)
    outs += [torch.gather(logp, -1, ids), ids]
    if up is None:
        return outs
    a, h, c = up
    dx = torch.zeros_like(x)
    onehot = torch.arange(x.shape[1], device=x.device)
    dx += (a.double() * keep)[:, None] * ((onehot == at[:, None]).double() - p)
    if h is not None:
        dx -= h.double()[:, None] * (plogp + p * H[:, None])
    for j in range(top if c is not None else 0):
        dx += c[:, j, None].double() * ((onehot == ids[:, j, None]).double() - p)
    return outs + [dx]


@torch.no_grad()
def exact(case, seed):
    kind = case["kind"]
    if kind in ("score", "loss"):
        logits, tokens, up = _logit_inputs(case, seed)
        B, T, V = logits.shape
        flat = [None if u is None else u.reshape(B * T, *u.shape[2:]) for u in up or ()]
        rows, tok = logits.reshape(B * T, V), tokens.reshape(B * T)
        parts, n = [], max(1, (1 << 26) // V)
        for i in range(0, B * T, n):
            parts.append(_exact_rows(rows[i:i + n], tok[i:i + n], case["top"],
                                     None if up is None else [None if u is None else u[i:i + n] for u in flat]))
        outs = [torch.cat(t).view(B, T, *t[0].shape[1:]) for t in zip(*parts)]
        return _named(outs[:4]) if up is None else _named(outs[:4], dlogits=outs[4])
    if kind in ("lookup", "embed"):
        weight, tokens, dout, scale = _embed_inputs(case, seed)
        out = weight.double().index_select(0, tokens) * scale
        if dout is None:
            return dict(out=out)
        dw = torch.zeros(weight.shape, device=DEV, dtype=torch.float64)
        dw.index_put_((tokens,), dout.double() * scale, accumulate=True)
        return dict(out=out, dweight=dw)
    grads, bound = _clip_inputs(case, seed)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    coef = min(1.0, bound / (norm + CLIP_EPS))
    return dict(norm=torch.tensor(norm, device=DEV, dtype=torch.float64),
                grads=torch.cat([g.double().flatten() * coef for g in grads]))
