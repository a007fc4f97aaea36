"""The sequence-model operators beside the spiking layers, as cases to be timed
and checked: linear attention with a decay for each head (prompt, training
step, single token), counter-based dropout, and the log probabilities of given
tokens with entropy and top alternatives.

``run`` computes a case in plain torch operations (``own = False``) or through
``myelin_amd``'s entry points (``own = True``); ``exact`` computes it from the
operator's definition in 64 bits.

Time-major layouts as in the rest of the framework: queries ``[T, B, H, Dk]``,
keys ``[T, B, Hk, Dk]``, values ``[T, B, Hk, Dv]``, states ``[B, H, Dk, Dv]``.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "bf16": 2}
IGNORE = -100
LOWEST = -3.0e38  # a mask value near the lowest of both types


def listed():
    return [
        # a short fp32 sequence through a small layer: launches and host work count
        {"name": "attention_small", "kind": "attention", "train": False, "dtype": "fp32", "T": 100, "B": 4, "H": 4,
         "Hk": 4, "Dk": 32, "Dv": 32, "lengths": False, "initial": False},
        # a batch of prompts of different lengths (one empty) that continues earlier
        # states; keys and values shared by groups of query heads, ragged sizes
        {"name": "attention_ragged", "kind": "attention", "train": False, "dtype": "bf16", "T": 1021, "B": 8, "H": 16,
         "Hk": 4, "Dk": 64, "Dv": 96, "lengths": True, "initial": True},
        # one long prompt: few heads, so the time axis has to be split
        {"name": "attention_long", "kind": "attention", "train": False, "dtype": "bf16", "T": 32768, "B": 1, "H": 16,
         "Hk": 16, "Dk": 128, "Dv": 128, "lengths": False, "initial": False},
        # a training step of the usual shape: outputs and every gradient
        {"name": "attention_train_bf16", "kind": "attention", "train": True, "dtype": "bf16", "T": 2048, "B": 8,
         "H": 16, "Hk": 16, "Dk": 128, "Dv": 128, "lengths": False, "initial": False},
        # a training step in the framework's default type with odd sizes, shared
        # heads, padded samples and a state that is trained through
        {"name": "attention_train_fp32", "kind": "attention", "train": True, "dtype": "fp32", "T": 501, "B": 16,
         "H": 8, "Hk": 4, "Dk": 50, "Dv": 75, "lengths": True, "initial": True},
        # generation, one sequence: latency
        {"name": "step_one", "kind": "step", "dtype": "fp32", "B": 1, "H": 8, "Hk": 8, "Dk": 64, "Dv": 64},
        # generation, a full batch: the states' bandwidth
        {"name": "step_batch", "kind": "step", "dtype": "bf16", "B": 256, "H": 16, "Hk": 16, "Dk": 128, "Dv": 128},
        # spikes of a hidden layer, one mask for all steps, training
        {"name": "dropout_spikes", "kind": "dropout", "dtype": "fp32", "T": 50, "B": 256, "N": 2048, "p": 0.2,
         "shared": True, "residual": False},
        # a residual branch of a long sequence, odd sizes, training
        {"name": "dropout_residual", "kind": "dropout", "dtype": "bf16", "T": 1000, "B": 37, "N": 1031, "p": 0.1,
         "shared": False, "residual": True},
        # the loss of a small classifier at every step of its readout
        {"name": "log_probs_classes", "kind": "log_probs", "train": True, "dtype": "fp32", "R": 12800, "V": 10,
         "top": 0, "ignored": 0.0, "masked": False},
        # generation: few rows of a large vocabulary, some tokens forbidden, with the alternatives
        {"name": "log_probs_serving", "kind": "log_probs", "train": False, "dtype": "bf16", "R": 8, "V": 100003,
         "top": 20, "ignored": 0.0, "masked": True},
        # the loss of a sequence model, padding ignored, with an entropy term
        {"name": "log_probs_train", "kind": "log_probs", "train": True, "dtype": "bf16", "R": 8192, "V": 32768,
         "top": 0, "ignored": 0.1, "masked": False},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""

    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "train", "step", "dropout", "log_probs", "log_probs"))
    dtype = rng.choice(("fp32", "bf16"))
    if kind in ("attention", "train", "step"):
        group = rng.choice((1, 1, 2, 4))
        Hk = rng.randint(1, max(1, 16 // group))
        H = Hk * group
        Dk, Dv = (rng.choice((16, 32, 64, 128, rng.randint(16, 128))) for _ in range(2))
        if kind == "step":
            return {"kind": "step", "dtype": dtype, "B": _spread(rng, 1, 256), "H": H, "Hk": Hk, "Dk": Dk, "Dv": Dv}
        train = kind == "train"
        # token-heads times width, below that of the largest listed case (fp32 moves twice the bytes)
        budget = (2**25 if train else 2**26) // (4 if dtype == "fp32" else 1)
        T = _spread(rng, 1, 4096 if train else 32768)
        B = _spread(rng, 1, max(1, min(64, budget // (T * H * max(Dk, Dv)))))
        T = max(1, min(T, budget // (B * H * max(Dk, Dv))))
        return {"kind": "attention", "train": train, "dtype": dtype, "T": T, "B": B, "H": H, "Hk": Hk, "Dk": Dk,
                "Dv": Dv, "lengths": rng.random() < 0.5, "initial": rng.random() < 0.5}
    if kind == "dropout":
        T, B = _spread(rng, 1, 1000), _spread(rng, 1, 256)
        N = _spread(rng, 1, max(1, min(4096, 2**25 // (T * B))))
        return {"kind": "dropout", "dtype": dtype, "T": T, "B": B, "N": N, "p": rng.choice((0.1, 0.2, 0.5)),
                "shared": rng.random() < 0.5, "residual": rng.random() < 0.5}
    train = rng.random() < 0.6
    V = _spread(rng, 2, 150000)
    R = _spread(rng, 1, max(1, min(16384, (2**27 if train else 2**24) // V)))
    return {"kind": "log_probs", "train": train, "dtype": dtype, "R": R, "V": V,
            "top": 0 if train else min(V, rng.choice((1, 5, 20, 50))), "ignored": rng.choice((0.0, 0.3)),
            "masked": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _prepare_heads(c, g, dt, lead):
    """Normalised queries and keys, as such layers feed them, and unit values."""

    def unit(*shape):
        x = torch.randn(*shape, generator=g, device=DEV)
        return torch.nn.functional.normalize(x, dim=-1).to(dt)

    q = unit(*lead, c["H"], c["Dk"])
    k = unit(*lead, c["Hk"], c["Dk"])
    v = torch.randn(*lead, c["Hk"], c["Dv"], generator=g, device=DEV).to(dt)
    # time constants of 4 to 1024 steps over the heads, as 1 - 1 / tau
    taus = torch.logspace(2, 10, c["H"], base=2.0, dtype=torch.float64)
    return q, k, v, (1.0 - 1.0 / taus).to(torch.float32).to(DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "attention":
        T, B, H = c["T"], c["B"], c["H"]
        s["q"], s["k"], s["v"], s["decay"] = _prepare_heads(c, g, dt, (T, B))
        s["lengths"] = s["state"] = None
        if c["lengths"]:
            s["lengths"] = torch.randint(T // 4, T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
            if B > 2:
                s["lengths"][1] = 0
        if c["initial"]:
            s["state"] = torch.randn(B, H, c["Dk"], c["Dv"], generator=g, device=DEV)
        if c["train"]:
            s["g_out"] = torch.randn(T, B, H, c["Dv"], generator=g, device=DEV).to(dt)
            s["g_state"] = torch.randn(B, H, c["Dk"], c["Dv"], generator=g, device=DEV)
            for name in ("q", "k", "v", "state"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif c["kind"] == "step":
        s["q"], s["k"], s["v"], s["decay"] = _prepare_heads(c, g, dt, (c["B"],))
        s["state"] = torch.randn(c["B"], c["H"], c["Dk"], c["Dv"], generator=g, device=DEV)
    elif c["kind"] == "dropout":
        shape = (c["T"], c["B"], c["N"])
        x = torch.rand(shape, generator=g, device=DEV) < 0.1 if c["shared"] else torch.randn(shape, generator=g, device=DEV)
        s["x"] = x.to(dt).requires_grad_()
        s["residual"] = torch.randn(shape, generator=g, device=DEV).to(dt).requires_grad_() if c["residual"] else None
        s["g"] = torch.randn(shape, generator=g, device=DEV).to(dt)
        s["seed"], s["offset"] = 0x1234567 * (seed + 1) % 2**62, seed
    else:
        R, V = c["R"], c["V"]
        x = 3.0 * torch.randn(R, V, generator=g, device=DEV)
        if c["masked"]:
            # a tenth of the tokens forbidden, half of them by the lowest value;
            # in a batch of rows one has nothing allowed
            m = torch.rand(V, generator=g, device=DEV)
            m[0] = 1.0
            x[:, m < 0.05] = -math.inf
            x[:, (m >= 0.05) & (m < 0.1)] = LOWEST
            if R > 2:
                x[1] = -math.inf
        s["logits"] = x.to(dt)
        s["targets"] = torch.randint(0, V, (R,), generator=g, device=DEV)
        if c["masked"]:
            allowed = (m >= 0.1).nonzero()[:, 0]
            s["targets"] = allowed[s["targets"] % allowed.numel()]
        n = int(R * c["ignored"])
        s["targets"][torch.randperm(R, generator=g, device=DEV)[:n]] = IGNORE
        if c["train"]:
            s["logits"].requires_grad_()
            s["g_log_probs"] = -torch.rand(R, generator=g, device=DEV) / R
            s["g_entropy"] = -0.01 * torch.rand(R, generator=g, device=DEV) / R
    return s


def work(case):
    c = case
    e = SIZE[c["dtype"]]
    if c["kind"] in ("attention", "step"):
        T = c.get("T", 1)
        live = (0.625 if c.get("lengths") else 1.0) * T
        B, H, Hk, Dk, Dv = (c[n] for n in ("B", "H", "Hk", "Dk", "Dv"))
        ins = live * B * e * (H * Dk + Hk * (Dk + Dv))
        out = T * B * H * Dv * e
        state = 4 * B * H * Dk * Dv
        states = state * (2 if c["kind"] == "step" or c["initial"] else 1)
        if not c.get("train"):
            return {"bytes": ins + out + states, "flops": live * B * H * 4 * Dk * Dv}
        grads = T * B * e * (H * Dk + Hk * (Dk + Dv))
        return {"bytes": ins + 2 * out + grads + states + state * (2 if c["initial"] else 1),
                "flops": live * B * H * 16 * Dk * Dv}
    if c["kind"] == "dropout":
        n = c["T"] * c["B"] * c["N"]
        return {"bytes": n * e * (5 if c["residual"] else 4), "flops": 4 * n}
    n = (c["R"] - int(c["R"] * c["ignored"])) * c["V"]
    if c["train"]:
        return {"bytes": e * (n + c["R"] * c["V"]), "flops": 12 * n}
    return {"bytes": e * n + c["R"] * (8 + 12 * c["top"]), "flops": 6 * n}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    return {"attention": _attention, "step": _step, "dropout": _dropout, "log_probs": _log_probs}[
        state["case"]["kind"]](state)


def _attention(s):
    if own:
        import myelin_amd as myelin

        final, out = myelin.decay_attention(s["q"], s["k"], s["v"], s["decay"], s["state"], lengths=s["lengths"])
    else:
        final, out = _plain_attention(s["q"], s["k"], s["v"], s["decay"], s["state"], s["lengths"])
    if not s["case"]["train"]:
        return {"state": final, "out": out}
    wrt = [n for n in ("q", "k", "v", "state") if s[n] is not None]
    grads = torch.autograd.grad((out, final), [s[n] for n in wrt], (s["g_out"], s["g_state"]))
    return {"state": final.detach(), "out": out.detach(), **{"g_" + n: t for n, t in zip(wrt, grads)}}


def _step(s):
    if own:
        import myelin_amd as myelin

        state, out = myelin.decay_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"])
    else:
        group = s["case"]["H"] // s["case"]["Hk"]
        q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        state = s["state"] * s["decay"][:, None, None] + k[..., None] * v[..., None, :]
        out = (q[..., None, :] @ state)[..., 0, :] * s["case"]["Dk"] ** -0.5
        out = out.to(s["q"].dtype)
    return {"state": state, "out": out}


def _dropout(s):
    c = s["case"]
    if own:
        import myelin_amd as myelin

        y = myelin.counter_dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"],
                                   time_shared=c["shared"])
    else:
        y = _plain_dropout(s["x"], c["p"], s["seed"], s["offset"], s["residual"], c["shared"])
    wrt = [t for t in (s["x"], s["residual"]) if t is not None]
    return {"y": y.detach(), "grads": torch.autograd.grad(y, wrt, s["g"])}


def _log_probs(s):
    c = s["case"]
    if own:
        import myelin_amd as myelin

        r = myelin.token_log_probs(s["logits"], s["targets"], top=c["top"], ignore_index=IGNORE)
        lp, entropy, top_lp, top_tokens = r.log_probs, r.entropy, r.top_log_probs, r.top_tokens
    else:
        lp, entropy, top_lp, top_tokens = _plain_log_probs(s["logits"], s["targets"], c["top"])
    if not c["train"]:
        return {"log_probs": lp, "entropy": entropy, "top_log_probs": top_lp, "top_tokens": top_tokens}
    (g,) = torch.autograd.grad((lp, entropy), s["logits"], (s["g_log_probs"], s["g_entropy"]))
    return {"log_probs": lp.detach(), "entropy": entropy.detach(), "g_logits": g}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _plain_attention(q, k, v, decay, state, lengths):
    """Chunks of 64 steps as masked products, and the chunks' states joined by
    one product with the decays between them."""

    T, B, H, Dk = q.shape
    Dv, C, dt = v.shape[-1], 64, q.dtype
    group = H // k.shape[2]
    n = -(-T // C)
    pad = n * C - T
    live = torch.full((B,), T, device=q.device) if lengths is None else lengths.long()
    steps = torch.arange(n * C, device=q.device)
    on = (steps < live[:, None]).float().view(B, 1, n, C, 1)

    def chunks(x, heads):
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, 0, 0, pad)).permute(1, 2, 0, 3)
        x = x.repeat_interleave(H // heads, 1).reshape(B, H, n, C, x.shape[-1])
        return torch.where(on > 0, x, 0.0)

    q, k, v = chunks(q, H), chunks(k, H // group), chunks(v, H // group)
    d = decay.float().view(1, H, 1, 1, 1)
    # steps that have decayed the state up to and with each one; padding decays nothing
    count = torch.minimum(steps + 1, live[:, None]).view(B, 1, n, C)
    last = count[..., -1]
    first = torch.nn.functional.pad(last, (1, 0))[..., :-1]
    i, j = count[..., :, None], count[..., None, :]
    causal = torch.ones(C, C, device=q.device).tril()
    inside = causal * torch.pow(d, (i - j).clamp(min=0).float())
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    # each chunk's own contribution, then the state that each chunk starts from
    own_state = (k * torch.pow(d, (last[..., None] - count).float()[..., None])).transpose(-1, -2) @ v
    before = torch.ones(n, n, device=q.device).tril(-1)
    between = before * torch.pow(d[..., 0], (first[..., :, None] - last[..., None, :]).clamp(min=0).float())
    start = (between @ own_state.reshape(B, H, n, Dk * Dv)).view(B, H, n, Dk, Dv)
    if state is not None:
        start = start + torch.pow(d, first[..., None, None].float()) * state[:, :, None]
    out = out + torch.pow(d, (count - first[..., None]).float()[..., None]) * (q @ start)
    tail = torch.pow(d[..., 0, 0], (last[..., -1:] - first[..., -1:]).float())[..., None]
    final = start[:, :, -1] * tail + own_state[:, :, -1]
    out = (out * on * Dk**-0.5).reshape(B, H, n * C, Dv)[:, :, :T].permute(2, 0, 1, 3)
    return final, out.to(dt)


def _philox(group, offset, seed):
    """Four 32-bit words for each counter (group, offset) and key seed: Philox
    4x32 of 10 rounds (Salmon, Moraes, Dror and Shaw, 2011), in 64-bit integers."""

    low = 0xFFFFFFFF

    def product(a, m):
        # a * m mod 2^64 in two's complement: both halves are its bits
        t = a * m
        return (t >> 32) & low, t & low

    c0, c1 = group & low, group >> 32
    c2 = torch.full_like(c0, offset & low)
    c3 = torch.full_like(c0, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), -1)


def _plain_dropout(x, p, seed, offset, residual, shared):
    shape = x.shape[1:] if shared else x.shape
    n = math.prod(shape)
    words = _philox(torch.arange(-(-n // 4), device=x.device), offset, seed).view(-1)[:n]
    keep = (words >= int(p * 2**32)).view(shape)
    y = torch.where(keep, x.float() * (1.0 / (1.0 - p)), 0.0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def _plain_log_probs(logits, targets, top):
    x = logits.float()
    R, V = x.shape
    ignored = targets == IGNORE
    with torch.no_grad():
        peak = x.max(-1, keepdim=True).values
        empty = peak == -math.inf
        peak = torch.where(empty, 0.0, peak)
    x = torch.where(empty, x.detach(), x)
    total = torch.exp(x - peak).sum(-1, keepdim=True)
    lse = torch.log(torch.where(empty, 1.0, total)) + peak
    log_p = x - lse
    lp = log_p.gather(-1, torch.where(ignored, 0, targets)[:, None])[:, 0]
    p = torch.exp(log_p)
    entropy = -(p * torch.where(p > 0, log_p, 0.0)).sum(-1)
    lp, entropy = torch.where(ignored, 0.0, lp), torch.where(ignored, 0.0, entropy)
    if not top:
        return lp, entropy, None, None
    # equal values go to the lowest index
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    top_lp = torch.where(ignored[:, None], -math.inf, log_p.gather(-1, order))
    return lp, entropy, top_lp, torch.where(ignored[:, None], -1, order)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "step": _exact_step, "dropout": _exact_dropout,
                "log_probs": _exact_log_probs}[case["kind"]](s)


def _exact_attention(s):
    """The recurrence and its adjoint, one step after the other."""

    c = s["case"]
    T, B, H, Hk, Dk, Dv = (c[n] for n in ("T", "B", "H", "Hk", "Dk", "Dv"))
    heads = torch.arange(H, device=DEV) // (H // Hk)
    d = s["decay"].double().view(1, H, 1, 1)
    scale = Dk**-0.5
    live = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    live = torch.tensor(live, device=DEV).view(B, 1, 1, 1)

    def at(name, t, side):
        x = s[name][t].double()
        x = x if x.shape[1] == H else x[:, heads]
        x = x[..., None] if side == "column" else x[..., None, :]
        return torch.where(live > t, x, 0.0)

    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=DEV) if s["state"] is None else s["state"].double()
    out = torch.zeros(T, B, H, Dv, dtype=torch.float64, device=DEV)
    g_q = torch.zeros(T, B, H, Dk, dtype=torch.float64, device=DEV) if c["train"] else None
    one = torch.ones((), dtype=torch.float64, device=DEV)
    for t in range(T):
        S = S * torch.where(live > t, d, one) + at("k", t, "column") * at("v", t, "row")
        out[t] = scale * (at("q", t, "row") @ S)[..., 0, :]
        if c["train"]:
            g_q[t] = scale * (S @ at("g_out", t, "column"))[..., 0]
    r = {"state": S, "out": out}
    if not c["train"]:
        return r
    G = s["g_state"].double()
    g_k = torch.zeros(T, B, Hk, Dk, dtype=torch.float64, device=DEV)
    g_v = torch.zeros(T, B, Hk, Dv, dtype=torch.float64, device=DEV)
    for t in range(T - 1, -1, -1):
        G = G + scale * at("q", t, "column") * at("g_out", t, "row")
        g_k[t] = (G @ at("v", t, "column"))[..., 0].view(B, Hk, H // Hk, Dk).sum(2)
        g_v[t] = (at("k", t, "row") @ G)[..., 0, :].view(B, Hk, H // Hk, Dv).sum(2)
        G = G * torch.where(live > t, d, one)
    r |= {"g_q": g_q, "g_k": g_k, "g_v": g_v}
    if s["state"] is not None:
        r["g_state"] = G
    return r


def _exact_step(s):
    c = s["case"]
    heads = torch.arange(c["H"], device=DEV) // (c["H"] // c["Hk"])
    k, v = s["k"].double()[:, heads], s["v"].double()[:, heads]
    S = s["decay"].double().view(1, -1, 1, 1) * s["state"].double() + k.unsqueeze(-1) * v.unsqueeze(-2)
    return {"state": S, "out": (S * s["q"].double().unsqueeze(-1)).sum(-2) * c["Dk"] ** -0.5}


def _exact_dropout(s):
    c = s["case"]
    shape = (c["B"], c["N"]) if c["shared"] else (c["T"], c["B"], c["N"])
    n = math.prod(shape)
    u32 = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    counter = [np.arange(-(-n // 4), dtype=np.uint64), None, None, None]
    counter[1] = counter[0] >> half
    counter[0] = counter[0] & u32
    counter[2] = np.full_like(counter[0], s["offset"] & 0xFFFFFFFF)
    counter[3] = np.full_like(counter[0], s["offset"] >> 32)
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for r in range(10):
        k0, k1 = (np.uint64((key[i] + r * w) & 0xFFFFFFFF) for i, w in enumerate((0x9E3779B9, 0xBB67AE85)))
        a = np.uint64(0xD2511F53) * counter[0]
        b = np.uint64(0xCD9E8D57) * counter[2]
        counter = [(b >> half) ^ counter[1] ^ k0, b & u32, (a >> half) ^ counter[3] ^ k1, a & u32]
    keep = torch.from_numpy((np.stack(counter, 1).reshape(-1)[:n] >= np.uint64(int(c["p"] * 2**32))).reshape(shape))
    factor = keep.to(DEV).double() / (1.0 - c["p"])
    y = s["x"].double() * factor
    grads = [s["g"].double() * factor]
    if s["residual"] is not None:
        y = y + s["residual"].double()
        grads.append(s["g"].double())
    return {"y": y, "grads": grads}


def _exact_log_probs(s):
    c = s["case"]
    R, V = c["R"], c["V"]
    t = s["targets"]
    r = {"log_probs": torch.zeros(R, dtype=torch.float64, device=DEV)}
    r["entropy"] = torch.zeros_like(r["log_probs"])
    if c["train"]:
        r["g_logits"] = torch.zeros(R, V, dtype=torch.float64, device=DEV)
    else:
        r["top_log_probs"] = torch.full((R, c["top"]), -math.inf, dtype=torch.float64, device=DEV)
        r["top_tokens"] = torch.full((R, c["top"]), -1, device=DEV)
    rows = (t != IGNORE).nonzero()[:, 0]
    for some in rows.split(max(1, 2**25 // V)):
        x = s["logits"][some].double()
        nothing = (x == -math.inf).all(-1, keepdim=True)
        lse = torch.where(nothing, 0.0, torch.logsumexp(x, -1, keepdim=True))
        log_p = x - lse
        p = log_p.exp()
        each = torch.where(p > 0, p * log_p, 0.0)
        hit = torch.arange(V, device=DEV) == t[some, None]
        r["log_probs"][some] = log_p.gather(-1, t[some, None])[:, 0]
        r["entropy"][some] = -each.sum(-1)
        if c["train"]:
            g_lp, g_h = s["g_log_probs"].double()[some, None], s["g_entropy"].double()[some, None]
            g = g_lp * (hit.double() - p) - g_h * (each - p * each.sum(-1, keepdim=True))
            r["g_logits"][some] = torch.where(nothing, 0.0, g)
        else:
            # equal values keep the order of their indices
            order = torch.argsort(-x, dim=-1, stable=True)[:, : c["top"]]
            r["top_tokens"][some] = order
            r["top_log_probs"][some] = log_p.gather(-1, order)
    return r
