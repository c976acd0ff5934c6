"""Operators of preference and policy tuning, and of the optimizer step behind it, with their plain forms.

``run`` makes one pass through an operator: the plain torch form, or (``own``) the call a user makes of this package.
``exact`` says in 64 bits what the outputs are.  The operators:

* ``logprobs``: log-probabilities of given tokens from logits, alone or with the gradient of the logits;
* ``logprobs_with_grad``: the same in one pass, the gradient of every row scaled by the row's weight;
* ``policy``: the clipped policy loss with a KL term over token log-probabilities, and its gradient;
* ``preference``: the loss over pairs of sequences (paired log ratios), and its gradient;
* ``clip``: the global norm of a list of gradients, and the clipped gradients.
"""
import itertools
import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one sampled token for each of four sequences, scored at the sampler's temperature: a call whose latency counts
        {"name": "logprobs-4x151936", "op": "logprobs", "rows": 4, "vocab": 151936, "dtype": "bf16", "temperature": 0.7,
         "ignored": 0.0, "masked_vocab": 0, "backward": False},
        # a micro-batch of 8 x 1024 tokens scored by the old or the reference policy: forward only
        {"name": "logprobs-8192x151936", "op": "logprobs", "rows": 8192, "vocab": 151936, "dtype": "bf16", "temperature": 1.0,
         "ignored": 0.0, "masked_vocab": 0, "backward": False},
        # training through the logits of a trainable head, the prompts' tokens left out
        {"name": "logprobs-train-2048x128256", "op": "logprobs", "rows": 2048, "vocab": 128256, "dtype": "bf16",
         "temperature": 1.0, "ignored": 0.2, "masked_vocab": 0, "backward": True},
        # fp32 logits, an odd vocabulary whose padding columns are switched off with -inf
        {"name": "logprobs-train-511x50257-fp32", "op": "logprobs", "rows": 511, "vocab": 50257, "dtype": "fp32",
         "temperature": 0.9, "ignored": 0.1, "masked_vocab": 157, "backward": True},
        # the frozen head of a training micro-batch: log-probabilities and the unit gradient of every token in one pass
        {"name": "with-grad-8192x151936", "op": "logprobs_with_grad", "rows": 8192, "vocab": 151936, "dtype": "bf16",
         "temperature": 1.0, "ignored": 0.0, "masked_vocab": 0},
        # a short batch with an odd vocabulary in fp32, weights per token
        {"name": "with-grad-301x32003-fp32", "op": "logprobs_with_grad", "rows": 301, "vocab": 32003, "dtype": "fp32",
         "temperature": 1.3, "ignored": 0.3, "masked_vocab": 0},
        # a handful of short completions: latency
        {"name": "policy-4x64", "op": "policy", "batch": 4, "seq": 64, "ref": False, "reduction": "token",
         "per_token_advantage": True},
        # a large rollout batch of ragged completions against a reference policy, averaged over sequences
        {"name": "policy-512x4096", "op": "policy", "batch": 512, "seq": 4096, "ref": True, "reduction": "sequence",
         "per_token_advantage": False},
        # two pairs of one-paragraph answers: latency
        {"name": "preference-2x129", "op": "preference", "pairs": 2, "seq": 129, "kind": "sigmoid", "smoothing": 0.0,
         "average": False},
        # a large batch of long pairs with an odd length
        {"name": "preference-256x8191", "op": "preference", "pairs": 256, "seq": 8191, "kind": "sigmoid", "smoothing": 0.1,
         "average": False},
        # the adapters of a 28-layer model, rank 16 (fourteen fp32 tensors per layer), in one gradient arena
        {"name": "clip-arena-28-layers", "op": "clip", "layers": 28, "hidden": 1536, "inner": 8960, "kv": 256, "rank": 16,
         "half": False, "norm": "2", "odd": 0, "arena": True},
        # a list of 84 gradients of wide trainable layers, bf16 ones beside fp32 ones, odd sizes
        {"name": "clip-list-84-mixed", "op": "clip", "layers": 6, "hidden": 4096, "inner": 14336, "kv": 1024, "rank": 512,
         "half": True, "norm": "2", "odd": 3, "arena": False},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_with_grad", "policy", "preference", "clip"])
    if op in ("logprobs", "logprobs_with_grad"):
        dtype = rng.choice(["bf16", "fp32"])
        vocab = _log_uniform(rng, 500, 152000)
        limit = 8192 * 151936 // (1 if dtype == "bf16" else 4) // vocab
        case = {"op": op, "rows": _log_uniform(rng, 1, max(2, min(16384, limit // 2))), "vocab": vocab, "dtype": dtype,
                "temperature": round(rng.uniform(0.5, 1.5), 2), "ignored": rng.choice([0.0, 0.0, 0.3]),
                "masked_vocab": rng.choice([0, 0, vocab // 50])}
        if op == "logprobs":
            case["backward"] = rng.random() < 0.6
        return case
    if op == "policy":
        return {"op": op, "batch": _log_uniform(rng, 1, 512), "seq": _log_uniform(rng, 1, 4096), "ref": rng.random() < 0.6,
                "reduction": rng.choice(["token", "sequence"]), "per_token_advantage": rng.random() < 0.5}
    if op == "preference":
        return {"op": op, "pairs": _log_uniform(rng, 1, 256), "seq": _log_uniform(rng, 1, 8191),
                "kind": rng.choice(["sigmoid", "hinge", "ipo"]), "smoothing": rng.choice([0.0, 0.1]), "average": rng.random() < 0.3}
    return {"op": op, "layers": rng.randint(1, 28), "hidden": rng.randint(64, 2048), "inner": rng.randint(64, 8960),
            "kv": rng.randint(16, 512), "rank": _log_uniform(rng, 1, 64), "half": rng.random() < 0.5, "norm": rng.choice(["2", "2", "inf"]),
            "odd": rng.randint(0, 3), "arena": rng.random() < 0.3}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _clip_sizes(case):
    """Element counts of the adapter pairs (A, B) of seven projections per layer; ``odd`` elements more in each."""
    h, i, kv, r = case["hidden"], case["inner"], case["kv"], case["rank"]
    per_layer = [(h, h), (kv, h), (kv, h), (h, h), (i, h), (i, h), (h, i)]
    return [r * width + case["odd"] for _ in range(case["layers"]) for n, k in per_layer for width in (k, n)]


def _arena(sizes, dtype):
    """Tensors of the given sizes in one zero-padded buffer, each on a 256-byte boundary: (buffer, tensors)."""
    step = 256 // dtype.itemsize
    begins = [0, *itertools.accumulate(-(-size // step) * step for size in sizes)]
    flat = torch.zeros(begins[-1], dtype=dtype, device="cuda")
    return flat, [flat[b:b + s] for b, s in zip(begins, sizes)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    if op in ("logprobs", "logprobs_with_grad"):
        rows, vocab = case["rows"], case["vocab"]
        # a trained model's logits: a broad bulk, and a few tokens (the target often among them) far above it
        logits = torch.empty(rows, vocab, dtype=DTYPES[case["dtype"]], device="cuda").normal_(0.0, 2.0, generator=gen)
        live = vocab - case["masked_vocab"]
        ids = torch.randint(0, live, (rows,), device="cuda", generator=gen)
        every = torch.arange(rows, device="cuda")
        logits[every, ids] += (16.0 * uniform(rows) - 2.0).to(logits.dtype)
        other = torch.randint(0, live, (rows,), device="cuda", generator=gen)
        logits[every, other] += (10.0 * uniform(rows)).to(logits.dtype)
        logits[:, live:] = float("-inf")
        ids[uniform(rows) < case["ignored"]] = IGNORE
        return {"case": case, "logits": logits, "leaf": logits.detach().requires_grad_(), "ids": ids, "row_grad": normal(rows),
                "out": torch.empty_like(logits) if op == "logprobs_with_grad" else None}
    if op in ("policy", "preference"):
        batch = case["batch"] if op == "policy" else 2 * case["pairs"]
        seq = case["seq"]
        # completions of all lengths behind prompts of all lengths; what is masked holds whatever was there
        first = (uniform(batch, 1) * 0.3 * seq).long()
        last = first + 1 + (uniform(batch, 1) * (seq - first)).long()
        at = torch.arange(seq, device="cuda")
        mask = (at >= first) & (at < last)
        logprobs = -4.0 * uniform(batch, seq).square() - 1e-3
        noise = float("nan")
        state = {"case": case, "mask": mask, "leaf": logprobs.masked_fill(~mask, noise).requires_grad_()}
        if op == "policy":
            mask &= uniform(batch, 1) >= 0.05          # sequences that were filtered out of the batch
            state["leaf"].data.masked_fill_(~mask, noise)
            # a few optimizer steps away from the policy that sampled, further from the reference
            state["old"] = (logprobs + 0.15 * normal(batch, seq)).masked_fill(~mask, noise)
            state["ref"] = (logprobs + 0.3 * normal(batch, seq)).masked_fill(~mask, noise) if case["ref"] else None
            state["advantages"] = normal(batch, seq) if case["per_token_advantage"] else normal(batch)
        else:
            state["ref"] = (logprobs + 0.2 * normal(batch, seq) / math.sqrt(max(1, seq) / 64)).masked_fill(~mask, noise)
        return state
    sizes = _clip_sizes(case)
    half = [s for k, s in enumerate(sizes) if case["half"] and k % 2]
    full = [s for k, s in enumerate(sizes) if not (case["half"] and k % 2)]
    state = {"case": case, "flats": [], "outs": [], "grads": [], "targets": []}
    for group, dtype in ((full, torch.float32), (half, torch.bfloat16)):
        if group:
            flat, views = _arena(group, dtype)
            for k, view in enumerate(views):   # gradients of one model differ in size from layer to layer
                view.normal_(0.0, 10.0 ** (k % 5 - 5), generator=gen)
            out, targets = _arena(group, dtype)
            state["flats"].append(flat)
            state["outs"].append(out)
            state["grads"] += [flat] if case["arena"] else views
            state["targets"] += [out] if case["arena"] else targets
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------

CLIP_LOW, CLIP_HIGH, KL, BETA, MAX_NORM = 0.2, 0.28, 0.04, 0.1, 1.0


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from molt_b200 import kernels

    case = state["case"]
    op = case["op"]
    if op == "logprobs":
        if not case["backward"]:
            return kernels.token_logprobs(state["logits"], state["ids"], temperature=case["temperature"])
        logprobs = kernels.token_logprobs(state["leaf"], state["ids"], temperature=case["temperature"])
        return logprobs.detach(), torch.autograd.grad(logprobs, state["leaf"], state["row_grad"])[0]
    if op == "logprobs_with_grad":
        return kernels.token_logprobs_with_grad(state["logits"], state["ids"], weight=state["row_grad"],
                                                temperature=case["temperature"], out=state["out"])
    if op == "policy":
        got = kernels.clipped_policy_loss(state["leaf"], state["old"], state["advantages"], mask=state["mask"],
                                          ref_logprobs=state["ref"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                                          kl_coef=KL if case["ref"] else 0.0, reduction=case["reduction"])
        (grad,) = torch.autograd.grad(got.loss, state["leaf"])
        return got.loss.detach(), got.kl, got.clip_fraction, grad
    if op == "preference":
        got = kernels.preference_loss(state["leaf"], state["ref"], mask=state["mask"], beta=BETA,
                                      label_smoothing=case["smoothing"] if case["kind"] == "sigmoid" else 0.0,
                                      kind=case["kind"], average=case["average"])
        (grad,) = torch.autograd.grad(got.loss, state["leaf"])
        return got.loss.detach(), got.chosen_rewards, got.rejected_rewards, grad
    norm = kernels.clip_grad_norm(state["grads"], MAX_NORM, norm_type=float(case["norm"]), out=state["targets"])
    return norm, state["outs"]


@torch.no_grad()
def _run_plain(state):
    return {"logprobs": _plain_logprobs, "logprobs_with_grad": _plain_logprobs, "policy": _plain_policy,
            "preference": _plain_preference, "clip": _plain_clip}[state["case"]["op"]](state)


def _plain_logprobs(state):
    case, ids = state["case"], state["ids"]
    x = state["logits"].float()
    vocab = x.shape[1]
    kept = (ids >= 0) & (ids < vocab)
    x = x - x.amax(dim=1, keepdim=True)
    x = x / case["temperature"]
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    at = ids.clamp(0, vocab - 1)[:, None]
    logprobs = torch.where(kept, (x.gather(1, at) - torch.log(total))[:, 0], 0.0)
    if case["op"] == "logprobs" and not case["backward"]:
        return logprobs
    grad = e / -total
    grad.scatter_add_(1, at, torch.ones_like(total))
    grad = grad * (torch.where(kept, state["row_grad"], 0.0) / case["temperature"])[:, None]
    return logprobs, grad.to(state["logits"].dtype)


def _weights(mask, reduction):
    """Weight of every token in the mean, in 64 bits."""
    kept = mask.double()
    lengths = kept.sum(dim=1, keepdim=True)
    if reduction == "token":
        return kept / lengths.sum().clamp(min=1)
    return kept / lengths.clamp(min=1) / (lengths > 0).sum().clamp(min=1)


def _plain_policy(state):
    # in 64 bits: ratios next to a clipping border, a KL term that is a small difference, long sums
    case, mask = state["case"], state["mask"]

    def of(t):
        return torch.where(mask, t.double(), 0.0)

    lp, advantages = of(state["leaf"]), state["advantages"].double()
    advantages = of(advantages if case["per_token_advantage"] else advantages[:, None].expand_as(lp))
    ratio = torch.exp(lp - of(state["old"]))
    cut = ((advantages > 0) & (ratio > 1 + CLIP_HIGH)) | ((advantages < 0) & (ratio < 1 - CLIP_LOW))
    loss = -torch.where(cut, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH), ratio) * advantages
    grad = -torch.where(cut, 0.0, ratio) * advantages
    kl = torch.zeros_like(lp)
    if case["ref"]:
        d = of(state["ref"]) - lp
        kl = torch.exp(d) - d - 1
        loss = loss + KL * kl
        grad = grad + KL * (1 - torch.exp(d))
    w = _weights(mask, case["reduction"])
    return (w * loss).sum().float(), (w * kl).sum().float(), (w * cut).sum().float(), (w * grad).float()


def _plain_preference(state):
    # in 64 bits: sums over whole sequences, and their differences
    case, mask = state["case"], state["mask"]
    ratio = torch.where(mask, state["leaf"].double() - state["ref"].double(), 0.0).sum(dim=1)
    share = mask.double()
    if case["average"]:
        length = share.sum(dim=1).clamp(min=1)
        ratio, share = ratio / length, share / length[:, None]
    chosen, rejected = ratio[:case["pairs"]], ratio[case["pairs"]:]
    h = chosen - rejected
    if case["kind"] == "sigmoid":
        smoothing = case["smoothing"]
        z = BETA * h
        loss = (1 - smoothing) * torch.log1p(torch.exp(-z.abs())) + smoothing * torch.log1p(torch.exp(-z.abs()))
        loss = loss + (1 - smoothing) * torch.relu(-z) + smoothing * torch.relu(z)
        slope = -BETA * ((1 - smoothing) / (1 + torch.exp(z)) - smoothing / (1 + torch.exp(-z)))
    elif case["kind"] == "hinge":
        loss, slope = torch.relu(1 - BETA * h), torch.where(BETA * h < 1, -BETA, 0.0)
    else:
        loss, slope = (h - 0.5 / BETA).square(), 2 * (h - 0.5 / BETA)
    slope = slope / case["pairs"]
    grad = torch.cat([slope, -slope])[:, None] * share
    return loss.mean().float(), (BETA * chosen).float(), (BETA * rejected).float(), grad.float()


def _plain_clip(state):
    if state["case"]["norm"] == "inf":
        norm = torch.stack([f.float().abs().max() for f in state["flats"]]).max()
    else:
        norm = torch.stack([f.float().square().sum(dtype=torch.float64) for f in state["flats"]]).sum().sqrt().float()
    scale = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    return norm, [(f.float() * scale).to(f.dtype) for f in state["flats"]]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------


def work(case):
    op = case["op"]
    if op in ("logprobs", "logprobs_with_grad"):
        rows = case["rows"] * (1.0 - case["ignored"])
        size = DTYPES[case["dtype"]].itemsize
        values = rows * case["vocab"]
        trained = op == "logprobs_with_grad" or case["backward"]
        total = values * size + case["rows"] * 12.0
        if trained:
            total += case["rows"] * (case["vocab"] * float(size) + 4.0)
        return {"bytes": total, "flops": values * (8.0 if trained else 4.0)}
    if op == "policy":
        tokens = case["batch"] * case["seq"]
        read = 9.0 + 4.0 * case["ref"] + 4.0 * case["per_token_advantage"]
        return {"bytes": tokens * (read + 4.0) + 4.0 * case["batch"], "flops": tokens * 20.0}
    if op == "preference":
        tokens = 2 * case["pairs"] * case["seq"]
        return {"bytes": tokens * 13.0 + 8.0 * case["pairs"], "flops": tokens * 4.0}
    sizes = _clip_sizes(case)
    values = [s * (2 if case["half"] and k % 2 else 4) for k, s in enumerate(sizes)]
    return {"bytes": 2.0 * sum(values), "flops": 3.0 * sum(sizes)}


# ---- the definition, in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "policy":
        return _exact_policy(case, state)
    if op == "preference":
        return _exact_preference(case, state)
    if op == "clip":
        total = torch.cat([f.double() for f in state["flats"]])
        norm = torch.linalg.vector_norm(total, ord=float(case["norm"]))
        return norm, [f.double() * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0) for f in state["flats"]]
    trained = op == "logprobs_with_grad" or case["backward"]
    parts, grads = [], []
    for begin in range(0, case["rows"], 1024):
        x = state["logits"][begin:begin + 1024].double().requires_grad_()
        target = state["ids"][begin:begin + 1024]
        scaled = x / case["temperature"]
        row = torch.arange(len(target), device="cuda")
        lp = scaled[row, target.clamp(min=0)] - torch.logsumexp(scaled, dim=1)
        lp = torch.where(target != IGNORE, lp, torch.zeros_like(lp))
        parts.append(lp.detach())
        if trained:
            (g,) = torch.autograd.grad(lp, x, state["row_grad"][begin:begin + 1024].double())
            grads.append(g)
    return (torch.cat(parts), torch.cat(grads)) if trained else torch.cat(parts)


def _exact_policy(case, state):
    mask, low, high = state["mask"], 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH
    where = mask.nonzero(as_tuple=True)
    leaf = state["leaf"].detach().double().requires_grad_()
    lp = leaf[where]
    adv = (state["advantages"] if case["per_token_advantage"] else state["advantages"][:, None].expand_as(mask))[where].double()
    lengths = mask.sum(dim=1)
    if case["reduction"] == "token":
        w = torch.full_like(adv, 1.0 / max(1, int(lengths.sum())))
    else:
        w = 1.0 / (lengths[where[0]].double() * max(1, int((lengths > 0).sum())))
    ratio = torch.exp(lp - state["old"][where].double())
    surrogate = torch.minimum(ratio * adv, torch.clamp(ratio, low, high) * adv)
    kl = torch.zeros_like(adv)
    if case["ref"]:
        d = state["ref"][where].double() - lp
        kl = torch.expm1(d) - d
    loss = (w * (KL * kl - surrogate)).sum()
    (grad,) = torch.autograd.grad(loss, leaf)
    cut = surrogate.detach() < (ratio * adv).detach()
    return loss.detach(), (w * kl).sum().detach(), (w * cut).sum(), grad


def _exact_preference(case, state):
    mask, pairs = state["mask"], case["pairs"]
    leaf = state["leaf"].detach().double().requires_grad_()
    gap = leaf - state["ref"].double()
    sums = torch.stack([gap[r][mask[r]].sum() for r in range(2 * pairs)])
    if case["average"]:
        sums = sums / mask.sum(dim=1)
    margin = sums[:pairs] - sums[pairs:]
    if case["kind"] == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1.0 - case["smoothing"]) * ls(BETA * margin) - case["smoothing"] * ls(-BETA * margin)
    elif case["kind"] == "hinge":
        loss = torch.clamp(1.0 - BETA * margin, min=0.0)
    else:
        loss = (margin - 1.0 / (2.0 * BETA)) ** 2
    loss = loss.mean()
    (grad,) = torch.autograd.grad(loss, leaf)
    return loss.detach(), BETA * sums[:pairs].detach(), BETA * sums[pairs:].detach(), grad
