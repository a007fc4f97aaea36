"""The operators of a small draft model, as cases to be timed and checked: the
lookup of its tokens' embeddings, a recurrence with a gate for every step and
channel (sequences, training, single steps), its distillation from a teacher's
top logits, and the verification of the tokens that it drafts.

``run`` computes a case in plain torch operations (``own = False``) or through
``myelin_amd``'s entry points (``own = True``); ``exact`` computes it from the
operator's definition in 64 bits.

Time-major layouts as in the rest of the framework: inputs and gates ``[T, B,
N]``, states ``[B, N]``, tokens ``[T, B]``, probabilities ``[n + 1, B, V]`` of
``n`` drafted tokens and the one after them.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}


def listed():
    return [
        # a batch of prompts of different lengths (one empty) that continues earlier
        # states; odd sizes
        {"name": "recurrence_ragged", "kind": "recurrence", "train": False, "dtype": "bf16", "T": 1021, "B": 8,
         "N": 1031, "lengths": True, "initial": True},
        # one long prompt: few channels, so the time axis has to be split
        {"name": "recurrence_long", "kind": "recurrence", "train": False, "dtype": "bf16", "T": 32768, "B": 1,
         "N": 2048, "lengths": False, "initial": False},
        # a training step of the usual shape: outputs and every gradient
        {"name": "recurrence_train_bf16", "kind": "recurrence", "train": True, "dtype": "bf16", "T": 2048, "B": 8,
         "N": 2048, "lengths": False, "initial": False},
        # a training step in the framework's default type, padded samples and a
        # state that is trained through
        {"name": "recurrence_train_fp32", "kind": "recurrence", "train": True, "dtype": "fp32", "T": 501, "B": 16,
         "N": 600, "lengths": True, "initial": True},
        # drafting, one sequence: latency
        {"name": "step_one", "kind": "step", "dtype": "fp32", "B": 1, "N": 1024},
        # drafting, a full batch: the states' bandwidth
        {"name": "step_batch", "kind": "step", "dtype": "bf16", "B": 256, "N": 4096},
        # the tokens of a small model's training step: launches and host work count
        {"name": "embedding_small", "kind": "embedding", "dtype": "fp32", "T": 64, "B": 32, "V": 50, "D": 128,
         "padding": False},
        # a training step of the usual shape: frequent and rare tokens, padding
        {"name": "embedding_train", "kind": "embedding", "dtype": "bf16", "T": 2048, "B": 8, "V": 32768, "D": 2048,
         "padding": True},
        # a small vocabulary, a few of the teacher's logits
        {"name": "distillation_small", "kind": "distillation", "dtype": "fp32", "R": 2048, "V": 1000, "K": 8,
         "temperature": 1.0, "ignored": 0.0, "masked": False},
        # a training step of the usual shape, softened, padding ignored, some tokens forbidden
        {"name": "distillation_train", "kind": "distillation", "dtype": "bf16", "R": 8192, "V": 32768, "K": 64,
         "temperature": 2.0, "ignored": 0.1, "masked": True},
        # one sequence's draft: latency
        {"name": "verify_one", "kind": "verify", "dtype": "fp32", "B": 1, "n": 4, "V": 32768, "sampled": True,
         "lengths": False},
        # a batch's drafts of different lengths, a large and odd vocabulary
        {"name": "verify_batch", "kind": "verify", "dtype": "fp32", "B": 64, "n": 8, "V": 100003, "sampled": True,
         "lengths": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""

    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("recurrence", "recurrence", "train", "step", "embedding", "embedding", "distillation",
                       "distillation", "verify"))
    dtype = rng.choice(("fp32", "bf16"))
    if kind in ("recurrence", "train"):
        # elements, at most those of the largest listed case (fp32 moves twice the bytes)
        budget = (2**25 if kind == "train" else 2**26) // (2 if dtype == "fp32" else 1)
        T = _spread(rng, 1, 32768)
        N = _spread(rng, 1, max(1, min(8192, budget // T)))
        B = _spread(rng, 1, max(1, min(256, budget // (T * N))))
        return {"kind": "recurrence", "train": kind == "train", "dtype": dtype, "T": T, "B": B, "N": N,
                "lengths": rng.random() < 0.5, "initial": rng.random() < 0.5}
    if kind == "step":
        return {"kind": "step", "dtype": dtype, "B": _spread(rng, 1, 256), "N": _spread(rng, 1, 8192)}
    if kind == "embedding":
        V, T = _spread(rng, 2, 150000), _spread(rng, 1, 8192)
        B = _spread(rng, 1, max(1, 2**17 // T))
        D = _spread(rng, 1, max(1, min(4096, 2**25 // max(V, T * B))))
        return {"kind": "embedding", "dtype": dtype, "T": T, "B": B, "V": V, "D": D, "padding": rng.random() < 0.5}
    if kind == "distillation":
        V = _spread(rng, 2, 150000)
        R = _spread(rng, 1, max(1, min(16384, 2**27 // V)))
        return {"kind": "distillation", "dtype": dtype, "R": R, "V": V, "K": min(V, _spread(rng, 1, 128)),
                "temperature": rng.choice((1.0, 1.5, 4.0)), "ignored": rng.choice((0.0, 0.3)),
                "masked": rng.random() < 0.5}
    V, n = _spread(rng, 2, 150000), rng.randint(1, 12)
    B = _spread(rng, 1, max(1, min(256, 2**25 // (V * (n + 1)))))
    return {"kind": "verify", "dtype": dtype, "B": B, "n": n, "V": V, "sampled": rng.random() < 0.7,
            "lengths": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _prepare_channels(c, g, lead):
    """Unit inputs, and gates around time constants of 4 to 1024 steps over the
    channels: a membrane's ``1 - 1 / tau`` is the sigmoid of ``log(tau - 1)``."""

    dt = DTYPES[c["dtype"]]
    x = torch.randn(*lead, c["N"], generator=g, device=DEV).to(dt)
    taus = torch.logspace(2, 10, c["N"], base=2.0, device=DEV)
    gate = (torch.randn(*lead, c["N"], generator=g, device=DEV) + torch.log(taus - 1.0)).to(dt)
    return x, gate


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "recurrence":
        T, B, N = c["T"], c["B"], c["N"]
        s["x"], s["gate"] = _prepare_channels(c, g, (T, B))
        s["lengths"] = s["state"] = None
        if c["lengths"]:
            s["lengths"] = torch.randint(T // 4, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
            if B > 2:
                s["lengths"][1] = 0
        if c["initial"]:
            s["state"] = torch.randn(B, N, generator=g, device=DEV)
        if c["train"]:
            s["g_out"] = torch.randn(T, B, N, generator=g, device=DEV).to(dt)
            s["g_state"] = torch.randn(B, N, generator=g, device=DEV)
            for name in ("x", "gate", "state"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif c["kind"] == "step":
        s["x"], s["gate"] = _prepare_channels(c, g, (c["B"],))
        s["state"] = torch.randn(c["B"], c["N"], generator=g, device=DEV)
    elif c["kind"] == "embedding":
        T, B, V = c["T"], c["B"], c["V"]
        # frequencies that fall as 1 / rank, ranks spread over the vocabulary
        # (a draw's logarithm is uniform)
        first = 1 if c["padding"] else 0  # token 0 is padding
        rank = torch.exp(torch.rand(T, B, generator=g, device=DEV, dtype=torch.float64) * math.log(V + 1 - first))
        place = first + torch.randperm(V - first, generator=g, device=DEV)
        s["tokens"] = place[(rank.long() - 1).clamp(0, V - 1 - first)]
        s["padding"] = None
        if c["padding"]:
            # samples end early
            s["padding"] = 0
            ends = torch.randint(T // 2 + 1, T + 1, (B,), generator=g, device=DEV)
            s["tokens"][torch.arange(T, device=DEV)[:, None] >= ends] = 0
        s["weight"] = torch.randn(V, c["D"], generator=g, device=DEV).to(dt).requires_grad_()
        s["scale"] = c["D"] ** 0.5
        s["g"] = torch.randn(T, B, c["D"], generator=g, device=DEV).to(dt)
    elif c["kind"] == "distillation":
        R, V, K = c["R"], c["V"], c["K"]
        teacher = 3.0 * torch.randn(R, V, generator=g, device=DEV)
        if c["masked"]:
            # a tenth of the tokens forbidden to both
            m = torch.rand(V, generator=g, device=DEV) < 0.1
            m[0] = False
            teacher[:, m] = -math.inf
        top = torch.topk(teacher, K)
        s["teacher_logits"], s["teacher_tokens"] = top.values, top.indices
        # a student that has learnt something
        s["logits"] = (0.7 * teacher + torch.randn(R, V, generator=g, device=DEV)).to(dt).requires_grad_()
        none = torch.randperm(R, generator=g, device=DEV)[: int(R * c["ignored"])]
        s["teacher_logits"][none], s["teacher_tokens"][none] = -math.inf, -1
        # forbidden tokens have no place among the teacher's
        s["teacher_tokens"][s["teacher_logits"] == -math.inf] = -1
        s["g"] = torch.rand(R, generator=g, device=DEV) / R
    else:
        n, B, V = c["n"], c["B"], c["V"]
        x = 3.0 * torch.randn(n + 1, B, V, generator=g, device=DEV)
        s["target"] = torch.softmax(x, -1).to(dt)
        # a draft model that is right most of the time
        draft = torch.softmax(x[:n] + 0.7 * torch.randn(n, B, V, generator=g, device=DEV), -1).to(dt)
        if c["sampled"]:
            s["draft"] = draft
            cdf = torch.cumsum(draft.double(), -1)
            at = torch.rand(n, B, 1, generator=g, device=DEV, dtype=torch.float64) * cdf[..., -1:]
            s["tokens"] = torch.searchsorted(cdf, at, right=True)[..., 0].clamp(max=V - 1)
        else:
            s["draft"] = None
            s["tokens"] = draft.argmax(-1)
        s["uniforms"] = torch.rand(n + 1, B, generator=g, device=DEV)
        s["lengths"] = None
        if c["lengths"]:
            s["lengths"] = torch.randint(0, n + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return s


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] == "recurrence":
        n = c["T"] * c["B"] * c["N"]
        live = n * (0.625 if c["lengths"] else 1.0)
        state = 4 * c["B"] * c["N"]
        states = state * (2 if c["initial"] else 1)
        if not c["train"]:
            return {"bytes": e * (2 * live + n) + states, "flops": 8 * live}
        return {"bytes": e * (3 * live + 3 * n) + states + state * (2 if c["initial"] else 1), "flops": 24 * live}
    if c["kind"] == "step":
        n = c["B"] * c["N"]
        return {"bytes": n * (3 * e + 8), "flops": 8 * n}
    if c["kind"] == "embedding":
        m, D = c["T"] * c["B"], c["D"]
        live = m * (0.75 if c["padding"] else 1.0)
        rows = min(live, c["V"])
        return {"bytes": 16 * m + e * D * (rows + m + live + c["V"]), "flops": D * (m + live)}
    if c["kind"] == "distillation":
        n = (c["R"] - int(c["R"] * c["ignored"])) * c["V"]
        return {"bytes": e * (n + c["R"] * c["V"]) + 12 * c["R"] * c["K"], "flops": 8 * n}
    # one row of each sequence is sampled from, the drafted tokens' values aside
    n = c["B"] * c["V"] * (2 if c["sampled"] else 1)
    return {"bytes": e * n + 24 * c["n"] * c["B"], "flops": 2 * n}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return {"recurrence": _recurrence, "step": _step, "embedding": _embedding, "distillation": _distillation,
            "verify": _verify}[state["case"]["kind"]](state)


def _recurrence(s):
    wrt = [n for n in ("x", "gate", "state") if s[n] is not None]
    if own:
        import myelin_amd as myelin

        final, out = myelin.gated_recurrence(s["x"], s["gate"], s["state"], lengths=s["lengths"])
        if not s["case"]["train"]:
            return {"state": final, "out": out}
        grads = torch.autograd.grad((out, final), [s[n] for n in wrt], (s["g_out"], s["g_state"]))
        return {"state": final.detach(), "out": out.detach(), **{"g_" + n: t for n, t in zip(wrt, grads)}}
    with torch.no_grad():
        r, kept = _plain_recurrence(s["x"], s["gate"], s["state"], s["lengths"])
        if s["case"]["train"]:
            grads = _plain_recurrence_grads(s["x"], s["gate"], kept, s["g_out"], s["g_state"])
            r.update({n: t for n, t in grads.items() if n != "g_state" or s["state"] is not None})
    return r


def _step(s):
    if own:
        import myelin_amd as myelin

        state, out = myelin.gated_recurrence_step(s["x"], s["gate"], s["state"])
    else:
        a = 1.0 / (1.0 + torch.exp(-s["gate"].float()))
        b = 1.0 / (1.0 + torch.exp(s["gate"].float()))
        state = a * s["state"] + b * s["x"].float()
        out = state.to(s["x"].dtype)
    return {"state": state, "out": out}


def _embedding(s):
    if own:
        import myelin_amd as myelin

        y = myelin.token_embedding(s["tokens"], s["weight"], scale=s["scale"], padding_index=s["padding"])
        (g,) = torch.autograd.grad(y, s["weight"], s["g"])
        return {"y": y.detach(), "g_weight": g}
    with torch.no_grad():
        w = s["weight"]
        tokens = s["tokens"].view(-1)
        rows, g = w[tokens].float() * s["scale"], s["g"].view(tokens.numel(), -1).float() * s["scale"]
        if s["padding"] is not None:
            hole = (tokens == s["padding"])[:, None]
            rows, g = torch.where(hole, 0.0, rows), torch.where(hole, 0.0, g)
        total = torch.zeros(w.shape, device=w.device).index_add_(0, tokens, g)
        return {"y": rows.to(w.dtype).view(s["g"].shape), "g_weight": total.to(w.dtype)}


def _distillation(s):
    t = s["case"]["temperature"]
    if own:
        import myelin_amd as myelin

        loss = myelin.distillation_loss(s["logits"], s["teacher_logits"], s["teacher_tokens"], temperature=t)
    else:
        loss = _plain_distillation(s["logits"], s["teacher_logits"], s["teacher_tokens"], t)
    (g,) = torch.autograd.grad(loss, s["logits"], s["g"])
    return {"loss": loss.detach(), "g_logits": g}


def _verify(s):
    if own:
        import myelin_amd as myelin

        r = myelin.verify_draft(s["target"], s["tokens"], s["uniforms"], s["draft"], lengths=s["lengths"])
        return {"accepted": r.accepted, "tokens": r.tokens}
    return _plain_verify(s["target"], s["tokens"], s["uniforms"], s["draft"], s["lengths"])


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _scan(a, b):
    """``h_t = a_t h_{t-1} + b_t`` from zero, by doubling the steps that each
    element reaches back over."""

    T, d = a.shape[0], 1
    while d < T:
        b = torch.cat((b[:d], b[d:] + a[d:] * b[:-d]))
        a = torch.cat((a[:d], a[d:] * a[:-d]))
        d *= 2
    return b


def _plain_recurrence(x, gate, state, lengths):
    T, B, N = x.shape
    gate = gate.float()
    a, b = 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))
    on = None
    u = b * x.float()
    if lengths is not None:
        # steps past the end keep the state
        on = torch.arange(T, device=x.device)[:, None, None] < lengths[:, None]
        a, b, u = torch.where(on, a, 1.0), torch.where(on, b, 0.0), torch.where(on, u, 0.0)
    first = torch.zeros(B, N, device=x.device) if state is None else state
    h = _scan(a, torch.cat((u[:1] + a[:1] * first, u[1:])))
    out = h if on is None else torch.where(on, h, 0.0)
    return {"state": h[-1].clone(), "out": out.to(x.dtype)}, (a, b, on, h, first)


def _plain_recurrence_grads(x, gate, kept, g_out, g_state):
    a, b, on, h, first = kept
    x, gate, g = x.float(), gate.float(), g_out.float()
    if on is not None:
        x, g = torch.where(on, x, 0.0), torch.where(on, g, 0.0)
    g = torch.cat((g[:-1], g[-1:] + g_state))
    # the gradient of a step's state comes back through the next step's decay
    later = torch.cat((torch.zeros_like(a[:1]), a[1:].flip(0)))
    g = _scan(later, g.flip(0)).flip(0)
    before = torch.cat((first[None], h[:-1]))
    g_gate = g * (before - x) * a * b
    return {"g_x": (b * g).to(g_out.dtype), "g_gate": g_gate.to(g_out.dtype), "g_state": a[0] * g[0]}


def _plain_distillation(logits, values, tokens, temperature):
    x = logits.float() / temperature
    there = (tokens >= 0) & (values > -math.inf)
    v = torch.where(there, values / temperature, -math.inf)
    none = ~there.any(-1, keepdim=True)
    peak = torch.where(none, 0.0, v.max(-1, keepdim=True).values)
    e = torch.exp(v - peak)
    total = torch.where(none, 1.0, e.sum(-1, keepdim=True))
    p, log_p = e / total, v - peak - torch.log(total)
    with torch.no_grad():
        m = x.max(-1, keepdim=True).values
    lse = torch.log(torch.exp(x - m).sum(-1, keepdim=True)) + m
    log_q = x.gather(-1, torch.where(there, tokens, 0)) - lse
    return torch.where(there, p * (torch.where(there, log_p, 0.0) - torch.where(there, log_q, 0.0)), 0.0).sum(-1)


def _plain_verify(target, tokens, uniforms, draft, lengths):
    n, B = tokens.shape
    dev = target.device
    batch = torch.arange(B, device=dev)
    u = uniforms.double()
    p = target[:n].gather(-1, tokens[..., None])[..., 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(-1, tokens[..., None])[..., 0].double()
    steps = torch.arange(n, device=dev)[:, None]
    drafted = torch.full((B,), n, device=dev) if lengths is None else lengths.long()
    good = (u[:n] * q < p) & (steps < drafted)
    accepted = torch.cumprod(good.long(), 0).sum(0)
    refused = accepted < drafted
    last = target[accepted, batch].double()
    at = torch.where(refused, accepted, 0)
    if draft is None:
        less = torch.zeros_like(last)
        less[batch, tokens[at, batch]] = last[batch, tokens[at, batch]]
    else:
        less = draft[at, batch].double()
    rest = torch.where(refused[:, None], (last - less).clamp(min=0.0), last)
    rest = torch.where((rest > 0.0).any(-1, keepdim=True), rest, last)
    cdf = torch.cumsum(rest, -1)
    drawn = (cdf <= u[n][:, None] * cdf[:, -1:]).sum(-1)
    rows = torch.arange(n + 1, device=dev)[:, None]
    padded = torch.cat((tokens, torch.full((1, B), -1, device=dev)))
    out = torch.where(rows < accepted, padded, torch.where(rows == accepted, drawn, -1))
    return {"accepted": accepted, "tokens": out}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "step": _exact_step, "embedding": _exact_embedding,
                "distillation": _exact_distillation, "verify": _exact_verify}[case["kind"]](s)


def _exact_recurrence(s):
    """One step after the other, and the adjoint one step before the other."""

    c = s["case"]
    T, B, N = c["T"], c["B"], c["N"]
    live = torch.full((B, 1), T, device=DEV) if s["lengths"] is None else s["lengths"].long()[:, None]
    h = torch.zeros(B, N, dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].double()
    out = torch.zeros(T, B, N, dtype=torch.float64, device=DEV)
    before = torch.zeros_like(out) if c["train"] else None
    for t in range(T):
        keep = torch.sigmoid(s["gate"][t].double())
        new = h + (1.0 - keep) * (s["x"][t].double() - h)
        if c["train"]:
            before[t] = h
        h = torch.where(live > t, new, h)
        out[t] = torch.where(live > t, h, 0.0)
    r = {"state": h, "out": out}
    if not c["train"]:
        return r
    g = s["g_state"].double()
    g_x, g_gate = torch.zeros_like(out), torch.zeros_like(out)
    for t in range(T - 1, -1, -1):
        keep = torch.sigmoid(s["gate"][t].double())
        here = g + s["g_out"][t].double()
        g_x[t] = torch.where(live > t, here * (1.0 - keep), 0.0)
        g_gate[t] = torch.where(live > t, here * (before[t] - s["x"][t].double()) * keep * (1.0 - keep), 0.0)
        g = torch.where(live > t, here * keep, g)
    r |= {"g_x": g_x, "g_gate": g_gate}
    if s["state"] is not None:
        r["g_state"] = g
    return r


def _exact_step(s):
    keep = torch.sigmoid(s["gate"].double())
    h = keep * s["state"].double() + (1.0 - keep) * s["x"].double()
    return {"state": h, "out": h}


def _exact_embedding(s):
    w, tokens = s["weight"].double(), s["tokens"].flatten()
    real = torch.ones_like(tokens, dtype=torch.bool) if s["padding"] is None else tokens != s["padding"]
    g = s["g"].flatten(0, 1)
    y = torch.zeros(g.shape, dtype=torch.float64, device=DEV)
    y[real] = s["scale"] * w[tokens[real]]
    # positions by token, each token's as one difference of running sums
    g_w = torch.zeros_like(w)
    order = torch.argsort(tokens)
    order = order[real[order]]
    if order.numel():
        ids, counts = torch.unique_consecutive(tokens[order], return_counts=True)
        ends = torch.cumsum(counts, 0)
        for cols in torch.arange(w.shape[1], device=DEV).split(256):
            sums = torch.cumsum(g[order][:, cols].double(), 0)[ends - 1]
            g_w[ids[:, None], cols] = s["scale"] * torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1]))
    return {"y": y.view(s["g"].shape), "g_weight": g_w}


def _exact_distillation(s):
    c = s["case"]
    R, V, tau = c["R"], c["V"], c["temperature"]
    loss = torch.zeros(R, dtype=torch.float64, device=DEV)
    g_logits = torch.zeros(R, V, dtype=torch.float64, device=DEV)
    rows = (s["teacher_tokens"] >= 0).any(-1).nonzero()[:, 0]
    for some in rows.split(max(1, 2**25 // V)):
        log_q = torch.log_softmax(s["logits"][some].double() / tau, -1)
        tokens = s["teacher_tokens"][some]
        v = torch.where(tokens >= 0, s["teacher_logits"][some].double() / tau, -math.inf)
        p = torch.softmax(v, -1)
        full = torch.zeros_like(log_q).scatter_add_(-1, tokens.clamp(min=0), p)
        loss[some] = (torch.xlogy(p, p) - torch.where(p > 0, p * log_q.gather(-1, tokens.clamp(min=0)), 0.0)).sum(-1)
        g_logits[some] = s["g"][some].double()[:, None] / tau * (torch.exp(log_q) - full)
    return {"loss": loss, "g_logits": g_logits}


def _exact_verify(s):
    """One sequence after the other, as it is told: tokens are taken while the
    target agrees, then one is drawn from what the draft left over."""

    n, B = s["tokens"].shape
    tokens, u = s["tokens"].tolist(), s["uniforms"].tolist()
    lengths = [n] * B if s["lengths"] is None else s["lengths"].tolist()
    accepted, out = [], [[-1] * B for _ in range(n + 1)]
    for b in range(B):
        i = 0
        while i < lengths[b]:
            x = tokens[i][b]
            q = 1.0 if s["draft"] is None else float(s["draft"][i, b, x])
            if not u[i][b] * q < float(s["target"][i, b, x]):
                break
            out[i][b] = x
            i += 1
        accepted.append(i)
        p = s["target"][i, b].double()
        left = p
        if i < lengths[b]:
            left = p.clone()
            if s["draft"] is None:
                left[tokens[i][b]] = 0.0
            else:
                left = torch.relu(p - s["draft"][i, b].double())
            if float(left.max()) <= 0.0:
                left = p
        cdf = left.cumsum(0)
        out[i][b] = int(torch.searchsorted(cdf, u[n][b] * cdf[-1], right=True))
    return {"accepted": torch.tensor(accepted, device=DEV), "tokens": torch.tensor(out, device=DEV)}
