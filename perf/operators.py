"""The losses over vocabulary logits, as cases to measure: what each stands for, its inputs,
one pass in plain torch operations or through ``lema_b200.ops``, and its definition in 64 bits.

``op`` is one of

* ``logprobs``    log-probability of each target token, alone (``train`` false: the frozen
                  reference model, an old policy) or with the gradient of the logits;
* ``preference``  the loss of chosen / rejected pairs over summed log ratios, with gradient;
* ``policy``      the clipped policy loss with a KL term, with gradient;
* ``distill``     distillation from a teacher's top logits, with gradient.

Logits are [B, S, V]; a target of -100 (a prompt, padding) leaves its row out.
"""
import math

import torch

own = False

IGNORE = -100
BF16, FP32 = "bf16", "fp32"


def listed():
    return [
        # the reference model's pass over a training batch (B 8, S 512, vocabulary 32000)
        {"name": "logprobs batch", "op": "logprobs", "train": False, "B": 8, "S": 512, "V": 32000,
         "dtype": BF16, "tau": 1.0},
        # one short answer of a small model: latency
        {"name": "logprobs short", "op": "logprobs", "train": False, "B": 1, "S": 7, "V": 512,
         "dtype": FP32, "tau": 1.0},
        # a loss of the user's own over log-probabilities, rows that start at any even byte
        {"name": "logprobs odd train", "op": "logprobs", "train": True, "B": 4, "S": 333,
         "V": 50257, "dtype": BF16, "tau": 0.7},
        # four pairs of the training batch's length
        {"name": "preference batch", "op": "preference", "B": 8, "S": 512, "V": 32000,
         "dtype": BF16, "beta": 0.1, "smooth": 0.0},
        # two long pairs over a large vocabulary: the largest call
        {"name": "preference wide", "op": "preference", "B": 4, "S": 1031, "V": 128256,
         "dtype": BF16, "beta": 0.1, "smooth": 0.1},
        # one short pair, logits kept in fp32
        {"name": "preference short", "op": "preference", "B": 2, "S": 37, "V": 8192,
         "dtype": FP32, "beta": 0.3, "smooth": 0.0},
        # a group of sixteen rollouts
        {"name": "policy batch", "op": "policy", "B": 16, "S": 512, "V": 32000, "dtype": BF16,
         "tau": 1.0, "kl": 0.04, "per": "token", "per_token_adv": False},
        # a large odd vocabulary, sampled at a temperature
        {"name": "policy wide", "op": "policy", "B": 3, "S": 611, "V": 100277, "dtype": BF16,
         "tau": 0.8, "kl": 0.1, "per": "sequence", "per_token_adv": True},
        # fewer tokens than SMs
        {"name": "policy few tokens", "op": "policy", "B": 2, "S": 9, "V": 32000, "dtype": BF16,
         "tau": 1.0, "kl": 0.0, "per": "sequence", "per_token_adv": False},
        {"name": "policy fp32", "op": "policy", "B": 4, "S": 256, "V": 32000, "dtype": FP32,
         "tau": 1.0, "kl": 0.02, "per": "token", "per_token_adv": True},
        # a batch against a teacher's 64 best tokens of each position
        {"name": "distill batch", "op": "distill", "B": 8, "S": 512, "V": 32000, "dtype": BF16,
         "tau": 2.0, "K": 64},
        # a few short sequences, odd everywhere
        {"name": "distill odd", "op": "distill", "B": 3, "S": 41, "V": 50257, "dtype": FP32,
         "tau": 1.0, "K": 17},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "preference", "policy", "distill"])
    dtype = rng.choice([BF16, BF16, BF16, FP32])
    V = _log_uniform(rng, 500, 160000)
    if rng.random() < 0.5:
        V = max(8, V // 64 * 64)
    rows = _log_uniform(rng, 4, max(5, min(16384, 400_000_000 // (V * (1 if dtype == BF16 else 2)))))
    B = rng.choice([1, 2, 3, 4, 8]) if op != "preference" else rng.choice([2, 4, 8])
    B = min(B, rows) if op != "preference" else B
    case = {"op": op, "B": B, "S": max(1, rows // B), "V": V, "dtype": dtype}
    if op == "logprobs":
        case |= {"train": rng.random() < 0.5, "tau": rng.choice([1.0, 0.7, 1.3])}
    elif op == "preference":
        case |= {"beta": rng.choice([0.05, 0.1, 0.5]), "smooth": rng.choice([0.0, 0.1])}
    elif op == "policy":
        case |= {"tau": rng.choice([1.0, 0.8]), "kl": rng.choice([0.0, 0.04]),
                 "per": rng.choice(["token", "sequence"]), "per_token_adv": rng.random() < 0.5}
    else:
        case |= {"tau": rng.choice([1.0, 2.0, 4.0]), "K": min(V, _log_uniform(rng, 1, 256))}
    return case


def _spans(case):
    """First and one past the last counted position of each sequence: prompts of up to half a
    sequence, padding of up to a quarter."""
    S = case["S"]
    return [(int((S - 1) * 0.5 * (0.618 * b % 1)), S - int((S - 1) * 0.25 * ((0.3 + 0.414 * b) % 1)))
            for b in range(case["B"])]


def _chunks(rows, V):
    step = max(1, (1 << 27) // V)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def prepare(case, seed):
    B, S, V = case["B"], case["S"], case["V"]
    dt = torch.bfloat16 if case["dtype"] == BF16 else torch.float32
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows = B * S
    # logits of a model that knows something: a wide bulk, the target raised above it
    logits = torch.empty(rows, V, dtype=dt, device=dev)
    for r0, r1 in _chunks(rows, V):
        logits[r0:r1] = (torch.randn(r1 - r0, V, device=dev, generator=gen) * 2.0).to(dt)
    tok = torch.randint(0, V, (rows,), device=dev, generator=gen)
    at = torch.arange(rows, device=dev)
    up = 2.0 + 10.0 * torch.rand(rows, device=dev, generator=gen)
    logits[at, tok] = (logits[at, tok].float() + up).to(dt)
    span = torch.tensor(_spans(case))
    pos = torch.arange(S)[None]
    counts = ((pos >= span[:, :1]) & (pos < span[:, 1:])).to(dev)
    targets = torch.where(counts, tok.view(B, S), torch.full((), IGNORE, device=dev))
    state = {"case": case, "logits": logits.view(B, S, V), "targets": targets, "counts": counts}
    if case["op"] == "logprobs":
        state["upstream"] = torch.randn(B, S, device=dev, generator=gen) / rows
        return state
    if case["op"] == "distill":
        # the teacher agrees with the student in part: its best tokens are the best of a
        # disturbed copy of the student's logits
        K = case["K"]
        ids = torch.empty(rows, K, dtype=torch.int64, device=dev)
        val = torch.empty(rows, K, device=dev)
        for r0, r1 in _chunks(rows, V):
            t = logits[r0:r1].float()
            t = t + torch.randn(t.shape, device=dev, generator=gen)
            val[r0:r1], ids[r0:r1] = torch.topk(t, K, dim=-1)
        state |= {"teacher_ids": ids.view(B, S, K), "teacher_logits": val.view(B, S, K)}
        return state
    lp = torch.empty(rows, device=dev)
    for r0, r1 in _chunks(rows, V):
        z = logits[r0:r1].float() / case.get("tau", 1.0)
        lp[r0:r1] = torch.log_softmax(z, -1)[torch.arange(r1 - r0, device=dev), tok[r0:r1]]
    lp = lp.view(B, S)
    noise = torch.randn(B, S, device=dev, generator=gen) * 0.1
    state["ref_logps"] = torch.where(counts, lp + noise, torch.zeros((), device=dev))
    if case["op"] == "policy":
        # ratios around 1, some of them past the clip range; none within 1e-3 of its ends, where
        # the gradient jumps
        d = torch.randn(B, S, device=dev, generator=gen) * 0.15
        for edge in (math.log1p(-CLIP[0]), math.log1p(CLIP[1])):
            near = (d - edge).abs() < 1e-3
            d = torch.where(near, torch.full((), edge + 2e-3, device=dev), d)
        state["old_logps"] = torch.where(counts, lp - d, torch.zeros((), device=dev))
        shape = (B, S) if case["per_token_adv"] else (B,)
        state["advantages"] = torch.randn(shape, device=dev, generator=gen)
        if not case["kl"]:
            state["ref_logps"] = None
    return state


CLIP = (0.2, 0.28)


# ---- the plain form -----------------------------------------------------------

def _softmax_rows(logits, tau):
    """exp(z - max) / sum in 32 bits, and (z - max, log sum) for log-probabilities in 64."""
    z = logits.float() / tau
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    s = e.sum(-1, keepdim=True)
    return z, e / s, torch.log(s.double())


def _token_logps(z, log_s, targets, counts):
    at = targets.clamp(min=0)[..., None]
    lp = (z.gather(-1, at).double() - log_s)[..., 0]
    return torch.where(counts, lp, torch.zeros_like(lp))


def _dlogits(q, coef, targets, counts, like):
    """coef * (onehot - q) of the rows that count, rounded once."""
    coef = torch.where(counts, coef, torch.zeros_like(coef))[..., None].float()
    g = -coef * q
    g.scatter_add_(-1, targets.clamp(min=0)[..., None], coef)
    return torch.where(counts[..., None], g, torch.zeros_like(g)).to(like.dtype)


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain(state):
    case, x, targets, counts = (state[k] for k in ("case", "logits", "targets", "counts"))
    tau = case.get("tau", 1.0)
    z, q, log_s = _softmax_rows(x, tau)
    if case["op"] == "distill":
        p = torch.exp((state["teacher_logits"] - state["teacher_logits"].amax(-1, keepdim=True))
                      .double() / tau)
        p = p / p.sum(-1, keepdim=True)
        lq = z.gather(-1, state["teacher_ids"]).double() - log_s
        kl = (p * (torch.log(p) - lq)).sum(-1)
        n = counts.sum()
        loss = tau * tau * torch.where(counts, kl, torch.zeros_like(kl)).sum() / n
        w = torch.where(counts, tau / n.double(), torch.zeros((), device=x.device))[..., None]
        g = q * w.float()
        g.scatter_add_(-1, state["teacher_ids"], (-w * p).float())
        return {"loss": loss.float(), "dlogits": g.to(x.dtype)}
    lp = _token_logps(z, log_s, targets, counts)
    if case["op"] == "logprobs":
        if not case["train"]:
            return {"logps": lp.float()}
        return {"logps": lp.float(),
                "dlogits": _dlogits(q, state["upstream"] / tau, targets, counts, x)}
    if case["op"] == "preference":
        P = case["B"] // 2
        rewards = case["beta"] * (lp - state["ref_logps"].double()).sum(-1)
        h = rewards[:P] - rewards[P:]
        e = case["smooth"]
        loss = ((1 - e) * _softplus(-h) + e * _softplus(h)).mean()
        dh = (e / (1 + torch.exp(-h)) - (1 - e) / (1 + torch.exp(h))) * (case["beta"] / P)
        coef = torch.cat([dh, -dh])[:, None].expand(lp.shape)
        return {"loss": loss.float(), "rewards": rewards.float(),
                "dlogits": _dlogits(q, coef, targets, counts, x)}
    A = state["advantages"].double()
    A = A if A.dim() == 2 else A[:, None].expand(lp.shape)
    n = counts.sum() if case["per"] == "token" else case["B"] * counts.sum(-1, keepdim=True)
    w = torch.where(counts, 1.0 / n.double(), torch.zeros((), device=x.device, dtype=torch.float64))
    r = torch.exp(lp - state["old_logps"].double())
    bent = torch.clamp(r, 1 - CLIP[0], 1 + CLIP[1])
    surr = -torch.minimum(r * A, bent * A)
    coef = torch.where(r * A <= bent * A, -r * A, torch.zeros_like(r))
    kl = torch.zeros_like(lp)
    if state["ref_logps"] is not None:
        d = state["ref_logps"].double() - lp
        kl = torch.expm1(d) - d
        coef = coef - case["kl"] * torch.expm1(d)
    loss = (w * (surr + case["kl"] * kl)).sum()
    return {"loss": loss.float(), "logps": lp.float(), "kl": (w * kl).sum().float(),
            "dlogits": _dlogits(q, w * coef / tau, targets, counts, x)}


# ---- the framework's calls ------------------------------------------------------

def _own(state):
    from lema_b200 import ops
    case, x, targets = (state[k] for k in ("case", "logits", "targets"))
    if case["op"] == "logprobs":
        if not case["train"]:
            return {"logps": ops.token_logprobs(x, targets, temperature=case["tau"])}
        x = x.detach().requires_grad_(True)
        lp = ops.token_logprobs(x, targets, temperature=case["tau"])
        return {"logps": lp.detach(), "dlogits": torch.autograd.grad(lp, x, state["upstream"])[0]}
    if case["op"] == "preference":
        loss, rewards, dx = ops.preference_loss_grad(x, targets, state["ref_logps"],
                                                     beta=case["beta"],
                                                     label_smoothing=case["smooth"])
        return {"loss": loss, "rewards": rewards, "dlogits": dx}
    if case["op"] == "policy":
        loss, logps, kl, dx = ops.policy_loss_grad(
            x, targets, state["old_logps"], state["advantages"], state["ref_logps"], clip=CLIP,
            kl_coef=case["kl"], temperature=case["tau"], reduction=case["per"])
        return {"loss": loss, "logps": logps, "kl": kl, "dlogits": dx}
    loss, dx = ops.distill_loss_grad(x, state["teacher_ids"], state["teacher_logits"],
                                     state["counts"], temperature=case["tau"])
    return {"loss": loss, "dlogits": dx}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    B, S, V = case["B"], case["S"], case["V"]
    size = 2 if case["dtype"] == BF16 else 4
    rows = B * S
    # rows that do not count are not read, their gradient is written
    read = sum(end - first for first, end in _spans(case))
    train = case["op"] != "logprobs" or case["train"]
    total = read * V * size + (rows * V * size if train else 0)
    small = {"logprobs": 12, "preference": 16, "policy": 28, "distill": 5}[case["op"]]
    total += rows * (small + (12 * case["K"] if case["op"] == "distill" else 0))
    # a difference, a product, an exponential and a sum; two more for a gradient
    return {"bytes": total, "flops": read * V * (6 if train else 4)}


# ---- the definitions in 64 bits ------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    x64 = st["logits"].double()
    train = case["op"] != "logprobs" or case["train"]
    x64.requires_grad_(train)
    keep = st["counts"].double()
    tau = case.get("tau", 1.0)
    lsm = torch.log_softmax(x64 / tau, dim=-1)
    if case["op"] == "distill":
        lt = torch.log_softmax(st["teacher_logits"].double() / tau, dim=-1)
        lq = torch.take_along_dim(lsm, st["teacher_ids"], -1)
        per_row = (lt.exp() * (lt - lq)).sum(-1)
        loss = tau ** 2 * (per_row * keep).sum() / keep.sum()
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, x64)[0]}
    safe = torch.where(st["counts"], st["targets"], 0)
    lp = torch.take_along_dim(lsm, safe[..., None], -1)[..., 0] * keep
    if case["op"] == "logprobs":
        if not case["train"]:
            return {"logps": lp}
        g = torch.autograd.grad((lp * st["upstream"].double()).sum(), x64)[0]
        return {"logps": lp.detach(), "dlogits": g}
    if case["op"] == "preference":
        won, was = lp.sum(1).chunk(2), st["ref_logps"].double().sum(1).chunk(2)
        h = case["beta"] * ((won[0] - won[1]) - (was[0] - was[1]))
        loss = -((1 - case["smooth"]) * torch.nn.functional.logsigmoid(h)
                 + case["smooth"] * torch.nn.functional.logsigmoid(-h)).mean()
        rewards = case["beta"] * (lp.sum(1) - st["ref_logps"].double().sum(1))
        return {"loss": loss.detach(), "rewards": rewards.detach(),
                "dlogits": torch.autograd.grad(loss, x64)[0]}
    adv = st["advantages"].double().reshape(case["B"], -1)
    ratio = (lp - st["old_logps"].double()).exp()
    gain = torch.min(ratio * adv, ratio.clip(1 - CLIP[0], 1 + CLIP[1]) * adv)
    kl = torch.zeros_like(lp)
    if st["ref_logps"] is not None:
        diff = st["ref_logps"].double() - lp
        kl = diff.exp() - 1 - diff
    each = case["kl"] * kl - gain
    if case["per"] == "token":
        loss, mean_kl = (each * keep).sum() / keep.sum(), (kl * keep).sum() / keep.sum()
    else:
        n = keep.sum(1)
        loss = ((each * keep).sum(1) / n).mean()
        mean_kl = ((kl * keep).sum(1) / n).mean()
    return {"loss": loss.detach(), "logps": lp.detach(), "kl": mean_kl.detach(),
            "dlogits": torch.autograd.grad(loss, x64)[0]}
