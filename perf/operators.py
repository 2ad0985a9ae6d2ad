"""Operators for fine-tuning a language model on rewards and preferences, as a list of cases that a timing program can run.

* ``token``       `fused.ops.token_logprobs`: log-probabilities of given tokens from logits, and their gradient
* ``linear``      `fused.ops.linear_logprobs`: the same from hidden states and the head's weight, without the logits in memory
* ``policy``      `fused.ops.policy_loss`: clipped policy loss with KL and entropy terms, forward and backward
* ``preference``  `fused.ops.preference_loss`: paired log-ratio loss, forward and backward
* ``clip``        `fused.ops.clip_grad_norm_`: global norm of the gradients of many tensors, and the clipped gradients

The plain form (`own` false) states each operator in elementary operations on FP32 values; `exact` states it in 64 bits through
the derivative that autograd finds.  Weights, logits and log-probabilities are random: there are no checkpoints to load."""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a judge or a guard scores a five-token answer: latency; rows of the unpadded GPT-2 vocabulary start at odd addresses
        dict(name="token_answer_5", kind="token", batch=1, length=5, vocab=50257, pitch=50257, dtype="bf16", grad=False),
        # sequence-level objective on FP32 logits of a small model, ragged sequences
        dict(name="token_fp32_609", kind="token", batch=3, length=203, vocab=32000, pitch=32000, dtype="fp32", grad=True),
        # log-probabilities of sampled tokens beside decoding: eight rows of GPT-2 XL, weights read once
        dict(name="linear_decode_8", kind="linear", batch=8, length=1, width=1600, vocab=50257, dtype="bf16", grad=False),
        # fine-tuning at the llama2-7b preset's head: 8192 tokens
        dict(name="linear_7b_8192", kind="linear", batch=4, length=2048, width=4096, vocab=32000, dtype="bf16", grad=True),
        # the qwen2-0.5b preset's head (narrow, large vocabulary) on an odd number of rows
        dict(name="linear_qwen_609", kind="linear", batch=3, length=203, width=896, vocab=151936, dtype="fp16", grad=True),
        # a small policy on short answers: latency
        dict(name="policy_small", kind="policy", batch=2, length=37, vocab=8192, pitch=8192, dtype="fp32", reduction="token",
             advantages="token", kl="k2", kl_coef=0.1, entropy_coef=0.0),
        # the headline benchmark's batch as a policy step: GPT-2 124M, padded vocabulary, group-relative advantages
        dict(name="policy_gpt2_16384", kind="policy", batch=16, length=1024, vocab=50257, pitch=50304, dtype="bf16",
             reduction="token", advantages="sequence", kl="k3", kl_coef=0.04, entropy_coef=0.0),
        # the llama3-8b preset's vocabulary, long answers, entropy bonus
        dict(name="policy_8b_8192", kind="policy", batch=4, length=2048, vocab=128256, pitch=128256, dtype="bf16",
             reduction="sequence", advantages="sequence", kl="k3", kl_coef=0.001, entropy_coef=0.01),
        # two short preference pairs
        dict(name="preference_2x203", kind="preference", pairs=2, length=203, vocab=32000, pitch=32000, dtype="fp16",
             loss="sigmoid", average=False),
        # eight pairs at the GPT-2 context
        dict(name="preference_8x1024", kind="preference", pairs=8, length=1024, vocab=50257, pitch=50304, dtype="bf16",
             loss="sigmoid", average=False),
        # gradients of a small model in BF16, odd sizes
        dict(name="clip_small", kind="clip", layers=3, width=257, vocab=8191, dtype="bf16", biases=True),
        # FP32 gradients of six GPT-2 XL layers and the embedding
        dict(name="clip_xl_6", kind="clip", layers=6, width=1600, vocab=50257, dtype="fp32", biases=True),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["token", "linear", "policy", "preference", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "clip":
        return dict(kind=kind, layers=rng.randint(1, 6), width=rng.choice([256, 513, 896, 1280, 1601]), vocab=_log(rng, 500, 50257),
                    dtype=dtype, biases=rng.random() < 0.5)
    if kind == "linear":
        width, vocab, batch = 8 * _log(rng, 16, 512), _log(rng, 1000, 152000), _log(rng, 1, 8)
        most = max(8, min(8192, 500_000_000_000 // (width * vocab)))
        return dict(kind=kind, batch=batch, length=_log(rng, 1, most // batch), width=width, vocab=vocab,
                    dtype=rng.choice(["bf16", "fp16"]), grad=rng.random() < 0.5)
    vocab = _log(rng, 500, 152000)
    pitch = rng.choice([vocab, vocab, (vocab + 63) // 64 * 64])
    most = max(4, min(8192, 400_000_000 // vocab))
    batch = _log(rng, 1, min(16, most // 2))
    length = _log(rng, 1, max(1, most // batch))
    if kind == "token":
        return dict(kind=kind, batch=batch, length=length, vocab=vocab, pitch=pitch, dtype=dtype, grad=rng.random() < 0.7)
    if kind == "preference":
        return dict(kind=kind, pairs=max(1, batch // 2), length=length, vocab=vocab, pitch=pitch, dtype=dtype,
                    loss=rng.choice(["sigmoid", "sigmoid", "ipo"]), average=rng.random() < 0.3)
    return dict(kind=kind, batch=batch, length=length, vocab=vocab, pitch=pitch, dtype=dtype, reduction=rng.choice(["token", "sequence"]),
                advantages=rng.choice(["token", "sequence"]), kl=rng.choice(["k1", "k2", "k3"]), kl_coef=rng.choice([0.001, 0.04, 0.1]),
                entropy_coef=rng.choice([0.0, 0.01]))


# ------------------------------------------------------------------------------------------------ inputs
CLIP_LOW, CLIP_HIGH, BETA, MAX_NORM = 0.2, 0.28, 0.1, 1.0


def _spans(batch, length):
    """(first, end) of the tokens that count in each sequence: a prompt of a quarter goes before them, ragged padding behind."""
    return [(length // 4, length - (b * length) // (4 * batch)) for b in range(batch)]


def _kept(batch, length):
    return sum(end - first for first, end in _spans(batch, length))


def _targets(batch, length, vocab, gen):
    t = torch.randint(0, vocab, (batch, length), device=DEV, generator=gen)
    first, end = torch.tensor(_spans(batch, length), device=DEV).t()[:, :, None]
    at = torch.arange(length, device=DEV)
    return torch.where((at >= first) & (at < end), t, IGNORE)


def _logits(batch, length, pitch, dtype, targets, gen):
    """Logits with a spread of 2.5 in which the given token mostly stands out; columns behind the vocabulary are padding."""
    x = (2.5 * torch.randn((batch, length, pitch), device=DEV, generator=gen)).to(TYPES[dtype])
    at = targets.clamp(min=0)[..., None]
    lift = 4.0 + 4.0 * torch.rand(at.shape, device=DEV, generator=gen)
    return x.scatter_(2, at, (x.gather(2, at).float() + lift).to(x.dtype))


def _scored(logits, targets, vocab):
    """Log-probabilities of the targets: what the sampler of an earlier model wrote down."""
    x = logits[..., :vocab].float()
    return x.gather(2, targets.clamp(min=0)[..., None])[..., 0] - torch.logsumexp(x, -1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, s = case["kind"], dict(case)
    rand = lambda *shape: torch.randn(shape, device=DEV, generator=gen)  # noqa: E731
    if kind == "clip":
        w, dt = case["width"], TYPES[case["dtype"]]
        shapes = [(case["vocab"], w)]
        for _ in range(case["layers"]):
            shapes += [(w,), (3 * w, w), (w, w), (w,), (4 * w, w), (w, 4 * w)]
            shapes += [(3 * w,), (w,), (4 * w,), (w,)] if case["biases"] else []
        shapes += [(w,)]
        s["grads"] = [(rand(*sh) * 10.0 ** (-2.0 - (i % 3))).to(dt) for i, sh in enumerate(shapes)]
        s["clipped"] = [torch.empty_like(g) for g in s["grads"]]
        return s
    if kind == "linear":
        b, t, d, v = case["batch"], case["length"], case["width"], case["vocab"]
        s["hidden"] = rand(b, t, d).to(TYPES[case["dtype"]])
        s["weight"] = (rand(v, d) * (2.0 / math.sqrt(d))).to(TYPES[case["dtype"]])
        s["targets"] = _targets(b, t, v, gen)
        s["dlogp"] = rand(b, t) / (b * t)
        if case["grad"]:
            s["hidden"].requires_grad_(True)
            s["weight"].requires_grad_(True)
        return s
    rows = 2 * case["pairs"] if kind == "preference" else case["batch"]
    t, v = case["length"], case["vocab"]
    s["targets"] = _targets(rows, t, v, gen)
    s["logits"] = _logits(rows, t, case["pitch"], case["dtype"], s["targets"], gen)
    keep = s["targets"] != IGNORE
    if kind == "token":
        s["dlogp"] = rand(rows, t) / (rows * t)
        s["logits"].requires_grad_(case["grad"])
        return s
    logp = _scored(s["logits"], s["targets"], v)
    if kind == "policy":
        # the policy has moved by steps of 1/64 from the model that sampled: no ratio stands within rounding of a clip border
        s["old_logp"] = logp - torch.round(rand(rows, t) * 8.0) / 64.0
        s["ref_logp"] = logp + 0.2 * rand(rows, t)
        s["advantages"] = rand(rows, t) if case["advantages"] == "token" else rand(rows)
    else:
        total = (logp * keep).sum(-1)
        if case["average"]:
            total = total / keep.sum(-1).clamp(min=1)
        s["ref_logp"] = total + (0.1 if case["average"] else 5.0) * rand(rows)
    s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    return {"token": _plain_token, "linear": _plain_linear, "policy": _plain_policy, "preference": _plain_preference,
            "clip": _plain_clip}[s["kind"]](s)


def _run_own(s):
    from nexus_b200.fused import ops
    kind = s["kind"]
    if kind == "clip":
        norm = ops.clip_grad_norm_(s["grads"], MAX_NORM, out=s["clipped"])
        return {"norm": norm, "grads": s["clipped"]}
    if kind == "linear":
        s["hidden"].grad = s["weight"].grad = None
        logp = ops.linear_logprobs(s["hidden"], s["weight"], s["targets"])
        if not s["grad"]:
            return {"logp": logp}
        logp.backward(s["dlogp"])
        return {"logp": logp.detach(), "d_hidden": s["hidden"].grad, "d_weight": s["weight"].grad}
    s["logits"].grad = None
    if kind == "token":
        logp = ops.token_logprobs(s["logits"], s["targets"], vocab=s["vocab"])
        if not s["grad"]:
            return {"logp": logp}
        logp.backward(s["dlogp"])
        return {"logp": logp.detach(), "grad": s["logits"].grad}
    if kind == "policy":
        r = ops.policy_loss(s["logits"], s["targets"], s["old_logp"], s["advantages"], s["ref_logp"], clip_low=CLIP_LOW,
                            clip_high=CLIP_HIGH, kl_coef=s["kl_coef"], kl=s["kl"], entropy_coef=s["entropy_coef"],
                            reduction=s["reduction"], vocab=s["vocab"])
        r.loss.backward()
        return {"loss": r.loss.detach(), "logp": r.logp, "kl": r.kl, "entropy": r.entropy, "grad": s["logits"].grad}
    r = ops.preference_loss(s["logits"], s["targets"], s["ref_logp"], beta=BETA, kind=s["loss"], average=s["average"], vocab=s["vocab"])
    r.loss.backward()
    return {"loss": r.loss.detach(), "logp": r.logp, "margin": r.margin, "grad": s["logits"].grad}


def _softmax_parts(x, targets):
    """FP32 rows x [N, V]: exponentials, their sums, the maximum, and the target's log-probability (zero where none counts)."""
    keep = targets != IGNORE
    at = targets.clamp(min=0)[:, None]
    top = x.max(-1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    logp = torch.where(keep, ((x.gather(1, at) - top) - torch.log(total))[:, 0], 0.0)
    return keep, at, e, total, top, logp


def _padded(g, like):
    """A gradient [N, vocab] in FP32, rounded once, with zeros behind the vocabulary."""
    out = torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    out.view(-1, like.shape[-1])[:, : g.shape[1]] = g.to(like.dtype)
    return out


def _rows(s):
    logits = s["logits"].detach()
    return logits.view(-1, logits.shape[-1])[:, : s["vocab"]].float(), s["targets"].reshape(-1)


def _row_gradient(e, total, at, c):
    """c (delta - p) of every row."""
    g = e * (-c / total[:, 0])[:, None]
    return g.scatter_add_(1, at, c[:, None])


def _plain_token(s):
    x, t = _rows(s)
    keep, at, e, total, _, logp = _softmax_parts(x, t)
    shape = s["targets"].shape
    if not s["grad"]:
        return {"logp": logp.view(shape)}
    c = torch.where(keep, s["dlogp"].reshape(-1), 0.0)
    return {"logp": logp.view(shape), "grad": _padded(_row_gradient(e, total, at, c), s["logits"])}


def _plain_linear(s):
    h = s["hidden"].detach().reshape(-1, s["width"]).float()
    w = s["weight"].detach().float()
    keep, at, e, total, _, logp = _softmax_parts(h @ w.t(), s["targets"].reshape(-1))
    shape = s["targets"].shape
    if not s["grad"]:
        return {"logp": logp.view(shape)}
    g = _row_gradient(e, total, at, torch.where(keep, s["dlogp"].reshape(-1), 0.0))
    return {"logp": logp.view(shape), "d_hidden": (g @ w).to(s["hidden"].dtype).view(s["hidden"].shape),
            "d_weight": (g.t() @ h).to(s["weight"].dtype)}


def _plain_policy(s):
    x, t = _rows(s)
    keep, at, e, total, top, logp = _softmax_parts(x, t)
    shape = s["targets"].shape
    p = e / total
    lp = (x - top) - torch.log(total)
    entropy = torch.where(keep, -(p * lp).sum(-1), 0.0)
    a = s["advantages"] if s["advantages"].dim() == 2 else s["advantages"][:, None].expand(shape)
    a = a.reshape(-1)
    ratio = torch.exp(logp - s["old_logp"].reshape(-1))
    bounded = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
    gain = torch.minimum(ratio * a, bounded * a)
    c = torch.where(ratio * a <= bounded * a, -ratio * a, 0.0)
    d = s["ref_logp"].reshape(-1) - logp
    if s["kl"] == "k3":
        kl, dkl = torch.exp(d) - d - 1.0, 1.0 - torch.exp(d)
    elif s["kl"] == "k2":
        kl, dkl = 0.5 * d * d, -d
    else:
        kl, dkl = -d, torch.ones_like(d)
    kl = torch.where(keep, kl, 0.0)
    counts = keep.view(shape).sum(-1)
    if s["reduction"] == "token":
        weight = torch.full_like(logp, 1.0) / counts.sum().clamp(min=1)
    else:
        weight = (1.0 / (counts.clamp(min=1) * (counts > 0).sum().clamp(min=1)))[:, None].expand(shape).reshape(-1)
    weight = torch.where(keep, weight, 0.0)
    loss = (weight * (-gain + s["kl_coef"] * kl - s["entropy_coef"] * entropy)).sum()
    g = _row_gradient(e, total, at, weight * (c + s["kl_coef"] * dkl))
    if s["entropy_coef"]:
        g = g + (weight * s["entropy_coef"])[:, None] * p * (lp + entropy[:, None])
    return {"loss": loss, "logp": logp.view(shape), "kl": kl.view(shape), "entropy": entropy.view(shape),
            "grad": _padded(g, s["logits"])}


def _plain_preference(s):
    x, t = _rows(s)
    keep, at, e, total, _, logp = _softmax_parts(x, t)
    shape, pairs = s["targets"].shape, s["pairs"]
    score = logp.double().view(shape).sum(-1)
    count = keep.view(shape).sum(-1).clamp(min=1).double()
    if s["average"]:
        score = score / count
    ratio = score - s["ref_logp"].double()
    margin = ratio[:pairs] - ratio[pairs:]
    if s["loss"] == "sigmoid":
        z = BETA * margin
        each = torch.log(1.0 + torch.exp(-z.abs())) + (-z).clamp(min=0.0)
        slope = -BETA / (1.0 + torch.exp(z))
    else:
        each = (margin - 0.5 / BETA) ** 2
        slope = 2.0 * (margin - 0.5 / BETA)
    slope = torch.cat([slope, -slope]) / pairs
    if s["average"]:
        slope = slope / count
    c = torch.where(keep, slope.float()[:, None].expand(shape).reshape(-1), 0.0)
    return {"loss": each.mean().float(), "logp": score.float(), "margin": margin.float(),
            "grad": _padded(_row_gradient(e, total, at, c), s["logits"])}


def _plain_clip(s):
    total = torch.stack([g.double().pow(2).sum() for g in s["grads"]]).sum()
    norm = total.sqrt()
    factor = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    return {"norm": norm.float(), "grads": [(g.float() * factor).to(g.dtype) for g in s["grads"]]}


# ------------------------------------------------------------------------------------------------ work of a pass
def work(case):
    kind, es = case["kind"], SIZE[case["dtype"]]
    if kind == "clip":
        w = case["width"]
        n = case["vocab"] * w + case["layers"] * (12 * w * w + 2 * w + (9 * w if case["biases"] else 0)) + w
        return {"bytes": 2 * n * es, "flops": 3 * n}
    v = case["vocab"]
    if kind == "linear":
        rows, d = case["batch"] * case["length"], case["width"]
        kept = _kept(case["batch"], case["length"])
        passes = 3 if case["grad"] else 1
        return {"bytes": (2 if case["grad"] else 1) * (rows + v) * d * es + rows * 16, "flops": passes * 2 * kept * v * d}
    batch = 2 * case["pairs"] if kind == "preference" else case["batch"]
    rows, kept = batch * case["length"], _kept(batch, case["length"])
    read = kept * v * es + rows * 12
    if kind == "token" and not case["grad"]:
        return {"bytes": read + rows * 4, "flops": 4 * kept * v}
    return {"bytes": read + rows * case["pitch"] * es + rows * 16, "flops": 8 * kept * v}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions on FP64 values, a piece of the rows at a time, with the derivatives that autograd finds."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        wide = [g.double() for g in s["grads"]]
        norm = math.sqrt(sum(float((g * g).sum()) for g in wide))
        return {"norm": torch.tensor(norm, dtype=torch.float64, device=DEV), "grads": [g * min(1.0, MAX_NORM / (norm + 1e-6)) for g in wide]}
    targets = s["targets"]
    flat, n = targets.reshape(-1), targets.numel()
    keep = flat != IGNORE
    if kind == "linear":
        h, w = s["hidden"].detach().reshape(n, -1).double(), s["weight"].detach().double()
        piece = max(1, 400_000_000 // case["vocab"])
    else:
        rows = s["logits"].detach().view(n, -1)
        piece = max(1, 100_000_000 // case["vocab"])

    def scores(lo, hi):
        """Log-probabilities of all tokens for the rows lo to hi, as a function of a leaf."""
        leaf = (h[lo:hi] @ w.t()) if kind == "linear" else rows[lo:hi, : case["vocab"]].double()
        leaf.requires_grad_(True)
        with torch.enable_grad():
            return leaf, torch.log_softmax(leaf, -1)

    def chosen(lp, lo, hi):
        return lp[torch.arange(hi - lo, device=DEV), flat[lo:hi].clamp(min=0)] * keep[lo:hi]

    spans = [(lo, min(n, lo + piece)) for lo in range(0, n, piece)]
    if kind in ("token", "linear"):
        logp = torch.zeros(n, dtype=torch.float64, device=DEV)
        if kind == "token":
            grad = torch.zeros((n, case["pitch"]), dtype=torch.float64, device=DEV) if case["grad"] else None
        elif case["grad"]:
            dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        for lo, hi in spans:
            leaf, lp = scores(lo, hi)
            with torch.enable_grad():
                one = chosen(lp, lo, hi)
            logp[lo:hi] = one.detach()
            if case["grad"]:
                (g,) = torch.autograd.grad(one, leaf, s["dlogp"].reshape(-1)[lo:hi].double())
                if kind == "token":
                    grad[lo:hi, : case["vocab"]] = g
                else:
                    dh[lo:hi] = g @ w
                    dw += g.t() @ h[lo:hi]
        out = {"logp": logp.view(targets.shape)}
        if case["grad"] and kind == "token":
            out["grad"] = grad.view(s["logits"].shape)
        elif case["grad"]:
            out |= {"d_hidden": dh.view(s["hidden"].shape), "d_weight": dw}
        return out

    grad = torch.zeros((n, case["pitch"]), dtype=torch.float64, device=DEV)
    if kind == "policy":
        old, ref = s["old_logp"].reshape(-1).double(), s["ref_logp"].reshape(-1).double()
        adv = s["advantages"].double()
        adv = (adv if adv.dim() == 2 else adv[:, None].expand(targets.shape)).reshape(-1)
        per = keep.view(targets.shape).sum(-1).double()
        if case["reduction"] == "token":
            weight = keep.double() / per.sum().clamp(min=1)
        else:
            weight = (keep.view(targets.shape) / per.clamp(min=1)[:, None] / (per > 0).sum().clamp(min=1)).reshape(-1)
        loss = 0.0
        logp, kls, ents = (torch.zeros(n, dtype=torch.float64, device=DEV) for _ in range(3))
        for lo, hi in spans:
            leaf, lp = scores(lo, hi)
            with torch.enable_grad():
                one = chosen(lp, lo, hi)
                ent = -(lp.exp() * lp).sum(-1) * keep[lo:hi]
                r = torch.exp(one - old[lo:hi])
                gain = torch.minimum(r * adv[lo:hi], r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv[lo:hi])
                d = ref[lo:hi] - one
                kl = {"k1": -d, "k2": d * d / 2, "k3": torch.expm1(d) - d}[case["kl"]] * keep[lo:hi]
                part = (weight[lo:hi] * (case["kl_coef"] * kl - gain - case["entropy_coef"] * ent)).sum()
            (g,) = torch.autograd.grad(part, leaf)
            grad[lo:hi, : case["vocab"]] = g
            loss = loss + part.detach()
            logp[lo:hi], kls[lo:hi], ents[lo:hi] = one.detach(), kl.detach(), ent.detach()
        shaped = [v.view(targets.shape) for v in (logp, kls, ents)]
        return {"loss": loss, "logp": shaped[0], "kl": shaped[1], "entropy": shaped[2], "grad": grad.view(s["logits"].shape)}

    logp = torch.cat([chosen(scores(lo, hi)[1].detach(), lo, hi) for lo, hi in spans])
    pairs = case["pairs"]
    per = keep.view(targets.shape).sum(-1).clamp(min=1).double()
    lp = logp.view(targets.shape).clone().requires_grad_(True)
    with torch.enable_grad():
        score = lp.sum(-1) / per if case["average"] else lp.sum(-1)
        ratio = score - s["ref_logp"].double()
        margin = ratio[:pairs] - ratio[pairs:]
        if case["loss"] == "sigmoid":
            loss = -torch.nn.functional.logsigmoid(BETA * margin).mean()
        else:
            loss = (margin - 1.0 / (2.0 * BETA)).square().mean()
    (slope,) = torch.autograd.grad(loss, lp)
    slope = slope.reshape(-1)
    for lo, hi in spans:
        leaf, all_lp = scores(lo, hi)
        with torch.enable_grad():
            one = chosen(all_lp, lo, hi)
        (g,) = torch.autograd.grad(one, leaf, slope[lo:hi])
        grad[lo:hi, : case["vocab"]] = g
    return {"loss": loss.detach(), "logp": score.detach(), "margin": margin.detach(), "grad": grad.view(s["logits"].shape)}
