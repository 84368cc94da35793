"""Drawing tokens from logits and learning from a teacher's logits, as timed cases.

Three kinds, by what a program has done:

  draw   sample_tokens: one token for every row, from temperature, top-k, top-p, min-p and a given random number
  match  distillation, forward only: how far a student is from a teacher's top logits (validation)
  teach  distillation, forward and backward: the training loss's outputs and the logits' gradient

`own` false computes the plain form in elementary torch operations, true calls the package.
"""
import math
import os
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unifiedlm.c_amd")

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ABSENT = -1   # a teacher's entry, or a token, that does not count


def listed():
    return [
        # one user's decode position with the usual nucleus
        dict(name="draw-1", kind="draw", rows=1, V=32000, dtype="fp32", T=0.8, k=0, p=0.9, m=0.0, each=False, masked=0.0),
        # the smallest model's few users, everything below a twentieth of the likeliest token left out
        dict(name="draw-260K", kind="draw", rows=8, V=512, dtype="fp32", T=1.0, k=0, p=1.0, m=0.05, each=False, masked=0.0),
        # a batch of decode positions, every user with settings of their own, some of them greedy
        dict(name="draw-256", kind="draw", rows=256, V=32000, dtype="fp32", T=0.9, k=50, p=0.95, m=0.02, each=True,
             masked=0.0),
        # draws from the model's distribution itself, as exploration in training takes them
        dict(name="draw-unfiltered", kind="draw", rows=200, V=31999, dtype="bf16", T=1.0, k=0, p=1.0, m=0.0, each=False,
             masked=0.0),
        # a large vocabulary, a part of it masked away
        dict(name="draw-large-vocab", kind="draw", rows=512, V=131072, dtype="bf16", T=0.7, k=40, p=0.95, m=0.0,
             each=False, masked=0.3),
        # rollouts: many continuations of many prompts, position by position
        dict(name="draw-rollouts", kind="draw", rows=4096, V=32000, dtype="fp32", T=1.0, k=0, p=0.95, m=0.0, each=False,
             masked=0.0),
        # a validation batch against stored top tokens
        dict(name="match-8K", kind="match", B=8, T=1024, V=32000, dtype="bf16", K=64, tau=1.0, labels=False, rest=False,
             absent=0.0),
        # the smallest model's batch
        dict(name="teach-260K", kind="teach", B=4, T=64, V=512, dtype="fp32", K=16, tau=2.0, labels=False, rest=False,
             absent=0.0),
        # the default model's batch in fp32: teacher and text together, the teacher's remaining mass as one more token
        dict(name="teach-15M", kind="teach", B=8, T=256, V=32000, dtype="fp32", K=32, tau=1.0, labels=True, rest=True,
             absent=0.0),
        # a small ragged batch, an odd vocabulary, teacher's lists of different lengths
        dict(name="teach-ragged", kind="teach", B=3, T=331, V=31999, dtype="fp16", K=50, tau=1.5, labels=False, rest=True,
             absent=0.3),
        # the 110M shape's training batch under bf16 autocast, softened by a temperature, with the text's own loss
        dict(name="teach-110M", kind="teach", B=16, T=1024, V=32000, dtype="bf16", K=64, tau=2.0, labels=True, rest=False,
             absent=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["draw", "draw", "draw", "match", "teach", "teach"])
    V = _log_int(rng, 200, 131072)
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if kind == "draw":
        rows = _log_int(rng, 1, max(1, min(4096, 4096 * 32000 // 4 // V)))   # the plain form sorts
        k = rng.choice([0, 0, 1, 40, _log_int(rng, 2, 2000)])
        return dict(kind=kind, rows=rows, V=V, dtype=dtype, T=round(rng.uniform(0.3, 1.6), 2), k=min(k, V),
                    p=rng.choice([1.0, 0.9, round(rng.uniform(0.3, 0.99), 3)]),
                    m=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.3), 3)]), each=rng.random() < 0.4,
                    masked=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]))
    rows = _log_int(rng, 1, max(1, min(16384, 16384 * 32000 // (4 if dtype == "fp32" else 2) // V)))
    B = min(rows, _log_int(rng, 1, 32))
    return dict(kind=kind, B=B, T=max(1, rows // B), V=V, dtype=dtype, K=min(_log_int(rng, 1, 200), V // 2),
                tau=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)]), labels=rng.random() < 0.5,
                rest=rng.random() < 0.4, absent=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]))


# ---- inputs, from the seed alone

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 2 + 1)


def _logits(rows, V, dtype, gen, likely, lift, hidden=None):
    """Rows as a trained model gives them: normal noise, the tokens `likely` lifted above it."""
    out = torch.empty(rows, V, device=DEV, dtype=dtype)
    at_once = max(1, (1 << 27) // V)
    for i in range(0, rows, at_once):
        x = torch.randn(min(at_once, rows - i), V, generator=gen, device=DEV).mul_(1.5)
        x.scatter_add_(1, likely[i:i + at_once], lift[i:i + at_once])
        if hidden is not None:
            x.masked_fill_(hidden, -math.inf)
        out[i:i + at_once] = x
    return out


def _draw_inputs(case, seed):
    """Logits (rows, V), random numbers and the settings: one for all, or a row's own."""
    gen = _gen(seed)
    rows, V = case["rows"], case["V"]
    n = min(8, V)
    likely = torch.randint(0, V, (rows, n), generator=gen, device=DEV)
    lift = 4.0 + 5.0 * torch.rand(rows, n, generator=gen, device=DEV)
    hidden = None
    if case["masked"]:   # tokens that no row may take
        hidden = torch.rand(V, generator=gen, device=DEV) < case["masked"]
        hidden[: V // 4 + 1] = False
    logits = _logits(rows, V, DTYPES[case["dtype"]], gen, likely, lift, hidden)
    u = torch.rand(rows, generator=gen, device=DEV)
    T, k, p, m = case["T"], case["k"], case["p"], case["m"]
    if case["each"]:
        f = lambda: torch.rand(rows, generator=gen, device=DEV)  # noqa: E731
        some = lambda share, yes, no: torch.where(f() < share, yes, torch.full((rows,), no, device=DEV))  # noqa: E731
        T = some(0.8, T * (0.5 + f()), 0.0)
        k = some(0.5, (2 * k * f()).floor(), 0.0).long()
        p = some(0.7, 1 - (1 - p) * 2 * f(), 1.0)
        m = some(0.4, m * 2 * f(), 0.0)
    return logits, u, dict(temperature=T, top_k=k, top_p=p, min_p=m)


def _teach_inputs(case, seed):
    """A student's logits (B, T, V), the teacher's entries (B, T, K), the text's tokens and upstream gradients.

    The teacher's tokens are distinct, more of them among the low numbers (the frequent tokens), with logits
    falling off steeply; the student agrees with the first of them. Without `rest` they are logits, with it log
    probabilities that leave the rest of the vocabulary some mass. The first position of a batch of several may have
    no entry at all."""
    gen = _gen(seed)
    B, T, V, K, dt = case["B"], case["T"], case["V"], case["K"], DTYPES[case["dtype"]]
    rows = B * T
    f = lambda *s: torch.rand(*s, generator=gen, device=DEV)  # noqa: E731
    ids = (f(rows, K).sort(-1).values.square() * (V - K)).long() + torch.arange(K, device=DEV)
    ids = ids.gather(1, f(rows, K).argsort(-1))
    logits = 9.0 * f(rows, 1) - 6.0 * torch.log1p(torch.arange(K, device=DEV) * f(rows, 1)) + 0.3 * f(rows, K)
    student = _logits(rows, V, dt, gen, ids[:, :8].contiguous(), 4.0 + 5.0 * f(rows, min(8, K)))
    if case["rest"]:
        logits = torch.log_softmax(logits / case["tau"], -1) + torch.log1p(-0.3 * f(rows, 1) - 1e-3)
    if case["absent"]:
        first = 1 + (f(rows, 1) * 2 * (1 - case["absent"]) * K).long()   # lists of different lengths
        ids[torch.arange(K, device=DEV) >= first] = ABSENT
        if rows > 1:
            ids[0] = ABSENT
    tokens = None
    if case["labels"]:
        tokens = torch.where(f(rows) < 0.6, ids[:, 0].clamp(min=0), torch.randint(0, V, (rows,), generator=gen, device=DEV))
        if rows > 1:
            tokens[f(rows) < 0.05] = ABSENT
        tokens = tokens.view(B, T)
    up = None
    if case["kind"] == "teach":
        # the mean over the positions, softened gradients scaled back; in fp16 scaled up, as such training does
        each = (1024.0 if dt == torch.float16 else 1.0) / rows
        up = [torch.full((B, T), 0.5 * each * case["tau"] ** 2, device=DEV)]
        if case["labels"]:
            up.append(torch.full((B, T), -0.5 * each, device=DEV))
    return student.view(B, T, V), ids.view(B, T, K), logits.view(B, T, K), tokens, up


def prepare(case, seed):
    if case["kind"] == "draw":
        logits, u, how = _draw_inputs(case, seed)
        return dict(kind="draw", logits=logits, u=u, how=how)
    student, ids, logits, tokens, up = _teach_inputs(case, seed)
    return dict(kind=case["kind"], student=student.requires_grad_(up is not None), ids=ids, logits=logits, tokens=tokens,
                up=up, tau=case["tau"], rest=case["rest"])


# ---- one pass

def _column(v, rows):
    """A setting as 64-bit numbers, one a row."""
    return (v.double() if isinstance(v, torch.Tensor) else torch.full((rows,), float(v), device=DEV, dtype=torch.float64))[:, None]


def _plain_draw(x, u, temperature, top_k, top_p, min_p):
    """In 64 bits: borders of top-p and of the drawn token's share lie as near as 2^-24 of a row's mass."""
    rows, V = x.shape
    T, k, p, m = (_column(v, rows) for v in (temperature, top_k, top_p, min_p))
    k = torch.where((k <= 0) | (T == 0), torch.where(T == 0, 1.0, float(V)), k)
    sorted_x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    sorted_x = sorted_x.double()
    w = torch.exp((sorted_x - sorted_x[:, :1]) / torch.where(T == 0, 1.0, T))
    rank = torch.arange(V, device=x.device)
    w = torch.where(rank < k, w, 0.0)
    c = torch.cumsum(w, -1)
    before = torch.cat([torch.zeros_like(c[:, :1]), c[:, :-1]], -1)
    keep = (rank < k) & ((before < p * c[:, -1:]) | (p >= 1)) & (w >= m) & (sorted_x > -math.inf)
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    c = torch.cumsum(w, -1)
    Z = c[:, -1:]
    above = c > u.double()[:, None] * Z
    last = V - 1 - (w > 0).flip(-1).to(torch.uint8).argmax(-1, keepdim=True)
    token = torch.where(above.any(-1, keepdim=True), above.to(torch.uint8).argmax(-1, keepdim=True), last)
    logprob = torch.log(w.gather(-1, token) / Z).float()
    return dict(token=token[:, 0], logprob=logprob[:, 0], kept=keep.sum(-1))


def _plain_distillation(x, ids, t, tokens, up, tau, rest):
    """The loss, the tokens' log probabilities where there are tokens and, with `up`, the logits' gradient."""
    x, t = x.float(), t.float()
    there = ids != ABSENT
    at = ids.clamp(min=0)
    z = x / tau
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    logp = d.gather(-1, at) - torch.log(s)
    if rest:
        q = torch.where(there, torch.exp(t), 0.0)
        logq = t
    else:
        z = torch.where(there, t / tau, -math.inf)
        z = z - z.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
        q = torch.exp(z)
        sq = q.sum(-1, keepdim=True)
        logq = z - torch.log(sq)
        q = torch.where(sq > 0, q / sq, 0.0)
    terms = torch.where(q > 0, q * (logq - logp), 0.0)
    loss = terms.sum(-1)
    if rest:
        qr = (1 - q.sum(-1, keepdim=True)).clamp(min=0)
        listed = torch.zeros(x.shape, device=x.device, dtype=torch.int8).scatter_add_(-1, at, there.to(torch.int8)) > 0
        sr = torch.where(listed, 0.0, e).sum(-1, keepdim=True)
        loss = loss + torch.where(qr > 0, qr * (torch.log(qr) - torch.log(sr) + torch.log(s)), 0.0)[..., 0]
    out = dict(loss=loss)
    if tokens is not None:
        valid = tokens != ABSENT
        label = tokens.clamp(min=0)[..., None]
        d1 = x - x.amax(-1, keepdim=True)
        e1 = torch.exp(d1)
        s1 = e1.sum(-1, keepdim=True)
        out["logprob"] = torch.where(valid, (d1.gather(-1, label) - torch.log(s1))[..., 0], 0.0)
    if up is None:
        return out
    g = up[0][..., None] / tau
    Q = q.sum(-1, keepdim=True)
    if rest:
        dx = e * (g * (Q + qr) / s)
        dx -= torch.where(listed, 0.0, e) * torch.where(qr > 0, g * qr / sr, 0.0)
    else:
        dx = e * (g * Q / s)
    dx.scatter_add_(-1, at, torch.where(there, -g * q, 0.0))
    if tokens is not None:
        a = torch.where(valid, up[1], 0.0)[..., None]
        dx -= e1 * (a / s1)
        dx.scatter_add_(-1, label, a)
    out["dlogits"] = dx
    return out


def run(state):
    if not own:
        with torch.no_grad():
            if state["kind"] == "draw":
                return _plain_draw(state["logits"], state["u"], **state["how"])
            out = _plain_distillation(*(state[k] for k in ("student", "ids", "logits", "tokens", "up", "tau", "rest")))
            if "dlogits" in out:
                out["dlogits"] = out["dlogits"].to(state["student"].dtype)
            return out
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import kernel
    if state["kind"] == "draw":
        out = kernel.sample_tokens(state["logits"], state["u"], **state["how"])
        return dict(token=out.token, logprob=out.logprob, kept=out.kept)
    out = kernel.distillation(state["student"], state["ids"], state["logits"], state["tokens"], temperature=state["tau"],
                              rest=state["rest"])
    outs = [out.loss] if state["tokens"] is None else [out.loss, out.logprob]
    res = {k: o.detach() for k, o in zip(("loss", "logprob"), outs)}
    if state["up"] is not None:
        res["dlogits"], = torch.autograd.grad(outs, [state["student"]], state["up"])
    return res


# ---- what one pass cannot do without

def work(case):
    V, b = case["V"], 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "draw":
        rows = case["rows"]
        # the logits, the random number, the settings; the token, its log probability and how many were kept
        return {"bytes": rows * (V * b + 4 + (20 if case["each"] else 0) + 20), "flops": rows * V * 4}
    rows = case["B"] * case["T"]
    # the logits, the teacher's entries, the tokens; the loss and the log probabilities
    bytes_ = rows * (V * b + 12 * case["K"] + 4 + 12 * case["labels"])
    flops = rows * V * (4 + 3 * (case["labels"] and case["tau"] != 1))
    if case["kind"] == "teach":   # the logits' gradient and the upstream ones
        bytes_ += rows * (V * b + 4 + 4 * case["labels"])
        flops += rows * V * (3 + 3 * (case["labels"] and case["tau"] != 1))
    return {"bytes": bytes_, "flops": flops}


# ---- the same outputs in 64 bits

def _exact_draw(x, u, T, k, p, m):
    """One block of rows. The masses left over below a token, from the smallest up, say what lies above it."""
    n, V = x.shape
    x = x.double()
    greedy = (T == 0)[:, 0]
    share = torch.softmax(x / torch.where(T == 0, 1.0, T), -1)
    # from the lowest to the highest, the higher index first among equals
    flipped = x.flip(-1)
    order = V - 1 - torch.sort(flipped, dim=-1, stable=True).indices
    place = torch.arange(V - 1, -1, -1, device=x.device)   # ranks from the top
    up = share.gather(-1, order)
    take = torch.where(k > 0, place < k, True)
    up = torch.where(take, up, 0.0)
    left = torch.cumsum(up, -1)                             # this one's and all lower ones' mass
    total = left[:, -1:]
    good = take & ((total - left < p * total) | (p >= 1)) & (up >= m * up[:, -1:]) & (x.gather(-1, order) > -math.inf)
    good[:, -1] = True
    good[greedy, :-1] = False
    kept = torch.zeros_like(good).scatter_(1, order, good)
    share = share * kept
    share = share / share.sum(-1, keepdim=True)
    cdf = torch.cumsum(share, -1)
    token = torch.searchsorted(cdf, (u.double() * cdf[:, -1])[:, None], right=True)[:, 0]
    some = torch.where(share > 0, torch.arange(V, device=x.device), -1).amax(-1)
    token = torch.minimum(token, some)
    return token, torch.log(share[torch.arange(n, device=x.device), token]), kept.sum(-1)


def _exact_rows(x, ids, t, tok, up, tau, rest):
    """One block of rows: log-softmax by torch.logsumexp, the teacher's entries one by one."""
    x, t = x.double(), t.double()
    n, V = x.shape
    line = torch.arange(n, device=x.device)
    logp = x / tau - torch.logsumexp(x / tau, -1, keepdim=True)
    p = logp.exp()
    there = ids != ABSENT
    if rest:
        logq = torch.where(there, t, -math.inf)
    else:
        logq = torch.where(there, t / tau, -math.inf)
        logq = logq - torch.logsumexp(logq, -1, keepdim=True)
        logq = torch.where(there, logq, -math.inf)
    q = logq.exp()
    loss = torch.zeros(n, device=x.device, dtype=torch.float64)
    dx = p * q.sum(-1, keepdim=True)
    listed = torch.zeros(n, V, device=x.device, dtype=torch.bool)
    for k in range(ids.shape[1]):
        on = there[:, k] & (q[:, k] > 0)
        at = torch.where(there[:, k], ids[:, k], 0)
        loss[on] += (q[:, k] * (logq[:, k] - logp[line, at]))[on]
        dx[line, at] -= torch.where(there[:, k], q[:, k], 0.0)
        listed[line[there[:, k]], at[there[:, k]]] = True
    if rest:
        qr = (1 - q.sum(-1)).clamp(min=0)
        others = torch.where(listed, 0.0, p)
        pr = others.sum(-1)
        on = qr > 0
        loss[on] += (qr * (qr.log() - pr.log()))[on]
        dx += p * qr[:, None] - torch.where(on[:, None], others * (qr / pr)[:, None], 0.0)
    outs = [loss]
    if tok is not None:
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        valid, at = tok != ABSENT, torch.where(tok == ABSENT, 0, tok)
        outs.append(torch.where(valid, logp[line, at], 0.0))
    if up is not None:
        dx *= up[0][:, None].double() / tau
        if tok is not None:
            a = torch.where(valid, up[1].double(), 0.0)
            dx -= logp.exp() * a[:, None]
            dx[line, at] += a
        outs.append(dx)
    return outs


@torch.no_grad()
def exact(case, seed):
    n = max(1, (1 << 26) // case["V"])
    if case["kind"] == "draw":
        logits, u, how = _draw_inputs(case, seed)
        how = [_column(how[k], case["rows"]) for k in ("temperature", "top_k", "top_p", "min_p")]
        parts = [_exact_draw(logits[i:i + n], u[i:i + n], *(h[i:i + n] for h in how)) for i in range(0, case["rows"], n)]
        return dict(zip(("token", "logprob", "kept"), (torch.cat(t) for t in zip(*parts))))
    student, ids, logits, tokens, up = _teach_inputs(case, seed)
    B, T, V = student.shape
    flat = lambda t: None if t is None else t.reshape(B * T, *t.shape[2:])  # noqa: E731
    cut = lambda t, i: None if t is None else t[i:i + n]  # noqa: E731
    args = [flat(t) for t in (student, ids, logits, tokens)]
    ups = None if up is None else [flat(g) for g in up]
    parts = [_exact_rows(*(cut(t, i) for t in args), None if ups is None else [cut(g, i) for g in ups], case["tau"],
                         case["rest"]) for i in range(0, B * T, n)]
    names = ["loss"] + (["logprob"] if tokens is not None else []) + (["dlogits"] if up is not None else [])
    return {k: torch.cat(t).view(B, T, *t[0].shape[1:]) for k, t in zip(names, zip(*parts))}
