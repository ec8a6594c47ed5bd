"""The loss operators of a policy / preference training step as measured cases: their inputs, their plain forms in
elementary torch operations, the calls that a program makes of the library's own operators, and their definitions in
64 bits.

Operators (the "op" of a case):
  score      log-probability, log-sum-exp and entropy of one target per row of logits
  score_grad gradient of the logits from the gradients of those log-probabilities and entropies
  policy     clipped policy loss with a KL term over per-token log-probabilities, with its gradient
  fused      the same from the logits themselves: loss, log-probabilities and the gradient of the logits
  pairs      preference loss over pairs of sequences, with its gradient
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
QWEN3_VOCAB = 151936
LIMIT = 4096 * QWEN3_VOCAB * 2            # bytes of logits of the largest case
LOSS = {"clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.04}


def listed():
    return [
        # one drafted or sampled token scored while serving: latency
        {"name": "score one token", "op": "score", "rows": 1, "vocab": QWEN3_VOCAB, "dtype": "fp16", "temperature": 1.0,
         "entropy": False, "banned": 0, "ignored": 0.0},
        # the answer tokens of a few short sequences, an odd vocabulary (rows start at any element), entropies logged
        {"name": "score odd vocabulary", "op": "score", "rows": 129, "vocab": 50257, "dtype": "bf16", "temperature": 0.7,
         "entropy": True, "banned": 17, "ignored": 0.1},
        # old or reference log-probabilities of a whole micro-batch of rollouts
        {"name": "score micro-batch", "op": "score", "rows": 4096, "vocab": QWEN3_VOCAB, "dtype": "fp16",
         "temperature": 1.0, "entropy": False, "banned": 0, "ignored": 0.0},
        # backward of a small batch kept in 32 bits, with an entropy bonus
        {"name": "score_grad fp32", "op": "score_grad", "rows": 333, "vocab": 32003, "dtype": "fp32", "temperature": 0.9,
         "entropy": True, "banned": 0, "ignored": 0.2},
        # backward of a whole micro-batch; a quarter of its rows are prompt tokens
        {"name": "score_grad micro-batch", "op": "score_grad", "rows": 4096, "vocab": QWEN3_VOCAB, "dtype": "bf16",
         "temperature": 1.0, "entropy": False, "banned": 0, "ignored": 0.25},
        # one short group of rollouts: log-probabilities to their gradient, latency
        {"name": "policy short group", "op": "policy", "seqs": 8, "longest": 128, "per_token": False,
         "reduction": "sequence", "entropy_coef": 0.0},
        # a whole rollout batch, per-token advantages, mean over tokens, entropy bonus
        {"name": "policy rollout batch", "op": "policy", "seqs": 512, "longest": 4095, "per_token": True,
         "reduction": "token", "entropy_coef": 0.01},
        # a few answer tokens (the last micro-batch of an uneven split)
        {"name": "fused few tokens", "op": "fused", "seqs": 3, "longest": 11, "vocab": QWEN3_VOCAB, "dtype": "fp16",
         "temperature": 1.0, "per_token": False, "reduction": "sequence", "entropy_coef": 0.0},
        # a middling micro-batch over an odd vocabulary, entropy bonus
        {"name": "fused odd vocabulary", "op": "fused", "seqs": 12, "longest": 251, "vocab": 50257, "dtype": "bf16",
         "temperature": 0.7, "per_token": True, "reduction": "token", "entropy_coef": 0.01},
        # the group-relative policy step's micro-batch at full vocabulary
        {"name": "fused micro-batch", "op": "fused", "seqs": 16, "longest": 510, "vocab": QWEN3_VOCAB, "dtype": "fp16",
         "temperature": 1.0, "per_token": False, "reduction": "sequence", "entropy_coef": 0.0},
        # a preference step on two short pairs: latency
        {"name": "pairs short", "op": "pairs", "seqs": 4, "longest": 100, "smoothing": 0.0, "margin": 0.0,
         "average": False},
        # a whole preference batch of long answers, smoothed labels, mean log ratios
        {"name": "pairs batch", "op": "pairs", "seqs": 1024, "longest": 4001, "smoothing": 0.1, "margin": 0.5,
         "average": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score_grad", "policy", "fused", "pairs"])
    case = {"op": op}
    if op in ("score", "score_grad", "fused"):
        case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
        case["vocab"] = rng.choice([QWEN3_VOCAB, _log_int(rng, 1000, QWEN3_VOCAB), _log_int(rng, 1000, QWEN3_VOCAB)])
        case["temperature"] = rng.choice([1.0, round(rng.uniform(0.5, 1.5), 2)])
        size = 4 if case["dtype"] == "fp32" else 2
        rows = _log_int(rng, 1, max(1, min(16384, LIMIT // (case["vocab"] * size))))
    if op in ("score", "score_grad"):
        case.update(rows=rows, entropy=rng.random() < 0.5, banned=rng.choice([0, 0, 50]),
                    ignored=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]))
    if op in ("policy", "fused"):
        if op == "policy":
            case.update(seqs=_log_int(rng, 1, 512), longest=_log_int(rng, 2, 4095))
        else:
            case["seqs"] = _log_int(rng, 1, max(1, min(64, rows)))
            case["longest"] = max(1, rows // case["seqs"])
        case.update(per_token=rng.random() < 0.5, reduction=rng.choice(["sequence", "token"]),
                    entropy_coef=rng.choice([0.0, 0.01]))
    if op == "pairs":
        case.update(seqs=2 * _log_int(rng, 1, 512), longest=_log_int(rng, 2, 4001),
                    smoothing=rng.choice([0.0, 0.1]), margin=rng.choice([0.0, 0.5]), average=rng.random() < 0.5)
    return case


# --- inputs ---------------------------------------------------------------------------------------------------------

def _lengths(seqs, longest):
    """Lengths of the sequences, a fixed ragged pattern from `longest` down to half of it: cases stay the same size
    from seed to seed."""
    return [longest - (i * 7919) % (longest // 2 + 1) for i in range(seqs)]


def _tokens(case):
    return sum(_lengths(case["seqs"], case["longest"]))


def _logits(case, rows, gen):
    v = case["vocab"]
    x = torch.empty(rows, v, dtype=DTYPES[case["dtype"]], device=DEVICE).normal_(0.0, 2.0, generator=gen)
    targets = torch.randint(0, v - case.get("banned", 0), (rows,), generator=gen, device=DEVICE)
    # the token that was sampled is one that the model finds likely
    lift = torch.rand(rows, generator=gen, device=DEVICE) * 14.0
    at = torch.arange(rows, device=DEVICE)
    x[at, targets] += lift.to(x.dtype)
    if case.get("banned", 0):
        x[:, v - case["banned"]:] = -math.inf
    return x, targets


def _sequences(case, gen):
    """Offsets, mask and per-token log-probability differences of a ragged batch; the first part of every sequence is
    its prompt (masked out)."""
    lens = _lengths(case["seqs"], case["longest"])
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    total = cu[-1]
    lens_t = torch.tensor(lens, device=DEVICE)
    cu_t = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
    prompt = (lens_t * (0.4 * torch.rand(len(lens), generator=gen, device=DEVICE))).long()
    at = torch.arange(total, device=DEVICE)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), lens_t, output_size=total)
    mask = (at - cu_t[:-1].long()[seq]) >= prompt[seq]
    return cu_t, mask, total


def _log_ratio(n, gen):
    """Differences of two policies' log-probabilities: small, with a tail that the clip cuts.  Those within 1e-3 of a
    border of the clip are moved away from it: which side a rounded log-probability falls on says nothing."""
    d = torch.randn(n, generator=gen, device=DEVICE) * 0.12
    for border in (math.log(1.0 - LOSS["clip_low"]), math.log(1.0 + LOSS["clip_high"])):
        d = torch.where((d - border).abs() < 1e-3, torch.full_like(d, border + 2e-3), d)
    return d


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    op, s = case["op"], {"case": case}
    if op in ("score", "score_grad"):
        rows = case["rows"]
        s["logits"], targets = _logits(case, rows, gen)
        if case["ignored"]:
            targets = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < case["ignored"],
                                  torch.full_like(targets, -1), targets)
        s["targets"] = targets
        if op == "score_grad":
            z = s["logits"].float() * (1.0 / case["temperature"])
            top = z.amax(1, keepdim=True)
            e = (z - top).exp()
            total = e.sum(1)
            lse = top[:, 0] + total.log()
            e *= torch.where(z > -math.inf, z, torch.zeros((), device=DEVICE))
            s["lse"] = lse
            s["dlogp"] = torch.randn(rows, generator=gen, device=DEVICE)
            if case["entropy"]:
                s["entropy"] = lse - e.sum(1) / total
                s["dentropy"] = torch.full((rows,), -0.01, device=DEVICE)
        return s
    cu, mask, total = _sequences(case, gen)
    s.update(cu=cu, mask=mask)
    if op == "fused":
        s["logits"], s["targets"] = _logits(case, total, gen)
        z = s["logits"].float() * (1.0 / case["temperature"])
        top = z.amax(1, keepdim=True)
        base = z[torch.arange(total, device=DEVICE), s["targets"]] - top[:, 0] - (z - top).exp().sum(1).log()
        del z
    else:
        base = -torch.empty(total, device=DEVICE).exponential_(1.0, generator=gen)
        s["logp"] = base
    if op in ("policy", "fused"):
        s["old"] = base - _log_ratio(total, gen)
        s["ref"] = base + torch.randn(total, generator=gen, device=DEVICE) * 0.2
        n_adv = total if case["per_token"] else case["seqs"]
        s["adv"] = torch.randn(n_adv, generator=gen, device=DEVICE)
        if op == "policy" and case["entropy_coef"]:
            s["entropy"] = torch.rand(total, generator=gen, device=DEVICE) * 3.0
        # what a program multiplies the gradients with so that they keep their place in 16 bits
        s["grad_scale"] = 1024.0 if op == "fused" and case["dtype"] == "fp16" else 1.0
    else:
        s["ref"] = base + torch.randn(total, generator=gen, device=DEVICE) * 0.2
        # the prompt's values are never used
        s["ref"] = torch.where(mask, s["ref"], torch.full_like(base, math.nan))
    return s


# --- plain forms ----------------------------------------------------------------------------------------------------

def _segment(cu, total):
    """Sequence number of every token."""
    marks = torch.zeros(total + 1, dtype=torch.int64, device=DEVICE)
    marks.index_add_(0, cu[1:-1].long(), torch.ones(cu.numel() - 2, dtype=torch.int64, device=DEVICE))
    return marks.cumsum(0)[:total]


def _segment_sum(x, cu):
    c = torch.cat([torch.zeros(1, dtype=torch.float64, device=DEVICE), x.double().cumsum(0)])
    at = cu.long()
    return c[at[1:]] - c[at[:-1]]


def _plain_rows(logits, targets, temperature, want_entropy):
    z = logits.float() * (1.0 / temperature)
    top = z.amax(1, keepdim=True)
    z -= top
    e = z.exp()
    total = e.sum(1)
    log_total = total.log()
    at = torch.arange(z.shape[0], device=DEVICE)
    keep = targets >= 0
    zero = torch.zeros((), device=DEVICE)
    logp = torch.where(keep, z[at, targets.clamp(min=0)] - log_total, zero)
    lse = torch.where(keep, top[:, 0] + log_total, zero)
    ent = None
    if want_entropy:
        ent = torch.where(keep, log_total - (e * torch.where(z > -math.inf, z, zero)).sum(1) / total, zero)
    return logp, lse, ent


def _plain_grad(logits, targets, temperature, lse, dlogp, ent, dent, scale=1.0):
    """Gradient of the logits; rows whose target is negative get zero."""
    it = 1.0 / temperature
    lp = logits.float() * it
    lp -= lse[:, None]
    p = lp.exp()
    keep = targets >= 0
    zero = torch.zeros((), device=DEVICE)
    g = torch.where(keep, dlogp * (it * scale), zero)
    d = p * -g[:, None]
    if dent is not None:
        c = torch.where(keep, dent * (it * scale), zero)
        d -= c[:, None] * (p * (torch.where(p > 0, lp, zero) + ent[:, None]))
    at = torch.arange(lp.shape[0], device=DEVICE)
    d[at, targets.clamp(min=0)] += g
    d = torch.where(keep[:, None], d, zero)
    return d.to(logits.dtype)


def _plain_policy(case, logp, old, ref, adv, entropy, mask, cu):
    total = logp.numel()
    seq = _segment(cu, total)
    m = mask.double()
    counts = _segment_sum(m, cu)
    if case["reduction"] == "sequence":
        w = (1.0 / (case["seqs"] * counts.clamp(min=1.0)))[seq]
    else:
        w = (1.0 / counts.sum().clamp(min=1.0)).expand(total)
    zero = torch.zeros((), device=DEVICE)
    zero64 = zero.double()
    w = torch.where(mask, w, zero64)
    a = adv if case["per_token"] else adv[seq]
    # the border is decided in 64 bits
    lr = logp.double() - old.double()
    inside = torch.where(a >= 0, lr <= math.log1p(LOSS["clip_high"]), lr >= math.log1p(-LOSS["clip_low"])) & mask
    ratio = torch.where(mask, lr, zero64).float().exp()
    bound = torch.where(a >= 0, torch.full_like(ratio, 1.0 + LOSS["clip_high"]),
                        torch.full_like(ratio, 1.0 - LOSS["clip_low"]))
    pol = -(a * torch.where(inside, ratio, bound))
    d = torch.where(mask, ref.double() - logp.double(), zero64)
    em1 = d.expm1()
    kl = em1 - d
    ent = torch.where(mask, entropy, zero) if entropy is not None else torch.zeros_like(logp)
    pol_sum, kl_sum, ent_sum = ((w * torch.where(mask, v.double(), zero64)).sum() for v in (pol, kl, ent))
    n = m.sum()
    clipped = torch.where(mask & ~inside, m, zero64).sum() / n.clamp(min=1.0)
    mean_ratio = torch.where(mask, ratio.double(), zero64).sum() / n.clamp(min=1.0)
    loss = pol_sum + LOSS["kl_coef"] * kl_sum - case["entropy_coef"] * ent_sum
    stats = torch.stack([loss, pol_sum, kl_sum, ent_sum, clipped, mean_ratio]).float()
    g = torch.where(inside, -(a * ratio), zero).double() - LOSS["kl_coef"] * em1
    dlogp = torch.where(mask, w * g, zero64).float()
    dent = (w * -case["entropy_coef"]).float() if case["entropy_coef"] else None
    return stats, mask.sum(), dlogp, dent


def _plain_pairs(case, logp, ref, mask, cu, beta):
    total, pairs = logp.numel(), case["seqs"] // 2
    seq = _segment(cu, total)
    zero = torch.zeros((), dtype=torch.float64, device=DEVICE)
    sums = _segment_sum(torch.where(mask, logp.double() - ref.double(), zero), cu)
    counts = _segment_sum(mask.double(), cu).clamp(min=1.0)
    per = 1.0 / counts if case["average"] else torch.ones_like(counts)
    rewards = beta * sums * per
    diff = rewards[:pairs] - rewards[pairs:]
    x = diff - case["margin"]
    log_sig = torch.minimum(x, zero) - (-x.abs()).exp().log1p()
    log_sig_neg = torch.minimum(-x, zero) - (-x.abs()).exp().log1p()
    ls = case["smoothing"]
    loss = (-(1.0 - ls) * log_sig - ls * log_sig_neg).mean()
    dx = (-(1.0 - ls) * log_sig_neg.exp() + ls * log_sig.exp()) / pairs
    stats = torch.stack([loss, (diff > 0).double().mean(), diff.mean(), rewards[:pairs].mean(),
                         rewards[pairs:].mean()]).float()
    coef = torch.cat([dx, -dx]) * beta * per
    dlogp = torch.where(mask, coef[seq], zero).float()
    return stats, rewards.float(), dlogp


# --- one pass -------------------------------------------------------------------------------------------------------

def _library():
    import importlib

    import __graft_entry__ as entry
    return importlib.import_module(entry.load_package().__name__ + ".losses")


BETA = 0.1


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        lib = _library()
        if op == "score":
            r = lib.token_logprobs(state["logits"], state["targets"], temperature=case["temperature"],
                                   with_entropy=case["entropy"])
            return {"logp": r.logp, "lse": r.lse, "entropy": r.entropy}
        if op == "score_grad":
            return {"dlogits": lib.token_logprobs_backward(
                state["logits"], state["targets"], state["lse"], state["dlogp"], temperature=case["temperature"],
                entropy=state.get("entropy"), dentropy=state.get("dentropy"))}
        if op == "policy":
            r = lib.policy_loss(state["logp"], state["adv"], old_logp=state["old"], ref_logp=state["ref"],
                                entropy=state.get("entropy"), mask=state["mask"], cu_seqlens=state["cu"],
                                reduction=case["reduction"], entropy_coef=case["entropy_coef"], **LOSS)
            return {"stats": r.stats, "tokens": r.tokens, "dlogp": r.dlogp, "dentropy": r.dentropy}
        if op == "fused":
            r = lib.policy_loss_logits(state["logits"], state["targets"], state["adv"], old_logp=state["old"],
                                       ref_logp=state["ref"], mask=state["mask"], cu_seqlens=state["cu"],
                                       temperature=case["temperature"], reduction=case["reduction"],
                                       entropy_coef=case["entropy_coef"], grad_scale=state["grad_scale"], **LOSS)
            return {"stats": r.stats, "tokens": r.tokens, "logp": r.logp, "dlogits": r.dlogits}
        r = lib.preference_loss(state["logp"], ref_logp=state["ref"], mask=state["mask"], cu_seqlens=state["cu"],
                                beta=BETA, label_smoothing=case["smoothing"], margin=case["margin"],
                                average=case["average"])
        return {"stats": r.stats, "rewards": r.rewards, "dlogp": r.dlogp}
    if op == "score":
        logp, lse, ent = _plain_rows(state["logits"], state["targets"], case["temperature"], case["entropy"])
        return {"logp": logp, "lse": lse, "entropy": ent}
    if op == "score_grad":
        return {"dlogits": _plain_grad(state["logits"], state["targets"], case["temperature"], state["lse"],
                                       state["dlogp"], state.get("entropy"), state.get("dentropy"))}
    if op == "policy":
        stats, tokens, dlogp, dent = _plain_policy(case, state["logp"], state["old"], state["ref"], state["adv"],
                                                   state.get("entropy"), state["mask"], state["cu"])
        return {"stats": stats, "tokens": tokens, "dlogp": dlogp, "dentropy": dent}
    if op == "fused":
        targets = torch.where(state["mask"], state["targets"], torch.full_like(state["targets"], -1))
        logp, lse, ent = _plain_rows(state["logits"], targets, case["temperature"], True)
        stats, tokens, dlogp, dent = _plain_policy(case, logp, state["old"], state["ref"], state["adv"], ent,
                                                   state["mask"], state["cu"])
        dlogits = _plain_grad(state["logits"], targets, case["temperature"], lse, dlogp, ent, dent,
                              state["grad_scale"])
        return {"stats": stats, "tokens": tokens, "logp": logp, "dlogits": dlogits}
    stats, rewards, dlogp = _plain_pairs(case, state["logp"], state["ref"], state["mask"], state["cu"], BETA)
    return {"stats": stats, "rewards": rewards, "dlogp": dlogp}


def work(case):
    op = case["op"]
    if op in ("policy", "pairs"):
        t = _tokens(case)
        floats = (4 if not case["per_token"] else 5) + (2 if case["entropy_coef"] else 0) if op == "policy" else 3
        return {"bytes": t * (4 * floats + 1), "flops": t * 20}
    rows = case["rows"] if op != "fused" else _tokens(case)
    n = rows * case["vocab"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "score":
        read = n * size * (1.0 - case["ignored"])
        return {"bytes": read + rows * 16, "flops": 4 * read / size}
    if op == "score_grad":
        read = n * size * (1.0 - case["ignored"])
        return {"bytes": read + n * size + rows * 16, "flops": 5 * read / size}
    # about a fifth of the tokens are prompt: their rows are written only
    return {"bytes": 1.8 * n * size + rows * 30, "flops": 9 * 0.8 * n}


# --- definitions in 64 bits -----------------------------------------------------------------------------------------

BLOCK = 256                   # rows at a time


def _exact_rows(logits, targets, temperature):
    """Per row: lse, log-probability of the target and entropy, rows without a target 0."""
    lse, logp, ent = [], [], []
    for lo in range(0, logits.shape[0], BLOCK):
        z = logits[lo:lo + BLOCK].double() / temperature
        t = targets[lo:lo + BLOCK]
        lq = torch.log_softmax(z, 1)
        on = (t >= 0).double()
        lse.append(torch.logsumexp(z, 1) * on)
        logp.append(torch.gather(lq, 1, t.clamp(min=0)[:, None])[:, 0] * on)
        ent.append(torch.special.entr(lq.exp()).sum(1) * on)
    return torch.cat(lse), torch.cat(logp), torch.cat(ent)


def _exact_policy(case, logp, s, entropy):
    cu, mask = s["cu"].tolist(), s["mask"]
    old, ref, adv = s["old"].double(), s["ref"].double(), s["adv"].double()
    lens = [b - a for a, b in zip(cu[:-1], cu[1:])]
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(logp.device)
    if not case["per_token"]:
        adv = adv[seq]
    n_all = int(mask.sum())
    if case["reduction"] == "token":
        w = torch.full_like(logp, 1.0 / max(n_all, 1))
    else:
        n = torch.zeros(len(lens), dtype=torch.float64, device=logp.device).index_add_(0, seq, mask.double())
        w = 1.0 / (len(lens) * n.clamp(min=1.0)[seq])
    at = mask.nonzero()[:, 0]
    w, a, lp = w[at], adv[at], logp[at]
    ratio = (lp - old[at]).exp()
    low, high = 1.0 - LOSS["clip_low"], 1.0 + LOSS["clip_high"]
    cut = ((a >= 0) & (ratio > high)) | ((a < 0) & (ratio < low))
    pol = -torch.minimum(ratio * a, ratio.clamp(low, high) * a)
    d = ref[at] - lp
    kl = torch.expm1(d) - d
    ent = entropy[at] if entropy is not None else torch.zeros_like(lp)
    parts = [(w * pol).sum(), (w * kl).sum(), (w * ent).sum()]
    loss = parts[0] + LOSS["kl_coef"] * parts[1] - case["entropy_coef"] * parts[2]
    stats = torch.stack([loss] + parts + [cut.double().sum() / max(n_all, 1), ratio.sum() / max(n_all, 1)])
    dlogp, dent = torch.zeros_like(logp), torch.zeros_like(logp)
    dlogp[at] = w * (torch.where(cut, torch.zeros_like(a), -a * ratio) - LOSS["kl_coef"] * torch.expm1(d))
    dent[at] = -case["entropy_coef"] * w
    return stats, dlogp, dent


def _exact_grad(logits, targets, temperature, lse, dlogp, ent, dent, scale):
    out = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    for lo in range(0, logits.shape[0], BLOCK):
        on = (targets[lo:lo + BLOCK] >= 0).nonzero()[:, 0] + lo
        if not on.numel():
            continue
        lq = logits[on].double() / temperature - lse[on].double()[:, None]
        g = dlogp[on].double()[:, None]
        hot = torch.zeros_like(lq).scatter_(1, targets[on][:, None], 1.0)
        d = g * (hot - lq.exp())
        if dent is not None:
            # p (log p + H), with p log p -> 0 where p is 0
            d += dent[on].double()[:, None] * (torch.special.entr(lq.exp()) - lq.exp() * ent[on].double()[:, None])
        out[on] = d * (scale / temperature)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "score":
        lse, logp, ent = _exact_rows(s["logits"], s["targets"], case["temperature"])
        return {"logp": logp, "lse": lse, "entropy": ent if case["entropy"] else None}
    if op == "score_grad":
        return {"dlogits": _exact_grad(s["logits"], s["targets"], case["temperature"], s["lse"], s["dlogp"],
                                       s.get("entropy"), s.get("dentropy"), 1.0)}
    if op == "policy":
        ent = s["entropy"].double() if "entropy" in s else None
        stats, dlogp, dent = _exact_policy(case, s["logp"].double(), s, ent)
        return {"stats": stats, "tokens": None, "dlogp": dlogp, "dentropy": dent if case["entropy_coef"] else None}
    if op == "fused":
        targets = s["targets"].masked_fill(~s["mask"], -1)
        lse, logp, ent = _exact_rows(s["logits"], targets, case["temperature"])
        stats, dlogp, dent = _exact_policy(case, logp, s, ent)
        dlogits = _exact_grad(s["logits"], targets, case["temperature"], lse, dlogp, ent,
                              dent if case["entropy_coef"] else None, s["grad_scale"])
        return {"stats": stats, "tokens": None, "logp": logp, "dlogits": dlogits}
    cu, pairs = s["cu"].tolist(), case["seqs"] // 2
    lens = torch.tensor([b - a for a, b in zip(cu[:-1], cu[1:])])
    seq = torch.repeat_interleave(torch.arange(len(lens)), lens).to(DEVICE)
    at = s["mask"].nonzero()[:, 0]
    zero = torch.zeros(len(lens), dtype=torch.float64, device=DEVICE)
    sums = zero.index_add(0, seq[at], (s["logp"].double() - s["ref"].double())[at])
    n = zero.index_add(0, seq[at], torch.ones(len(at), dtype=torch.float64, device=DEVICE)).clamp(min=1.0)
    per = 1.0 / n if case["average"] else torch.ones_like(n)
    r = BETA * sums * per
    diff = r[:pairs] - r[pairs:]
    x = diff - case["margin"]
    ls = case["smoothing"]
    loss = -(1 - ls) * torch.nn.functional.logsigmoid(x) - ls * torch.nn.functional.logsigmoid(-x)
    stats = torch.stack([loss.mean(), (diff > 0).double().mean(), diff.mean(), r[:pairs].mean(), r[pairs:].mean()])
    dx = (ls * torch.sigmoid(x) - (1 - ls) * torch.sigmoid(-x)) / pairs
    dlogp = torch.zeros_like(s["logp"], dtype=torch.float64)
    dlogp[at] = (torch.cat([dx, -dx]) * BETA * per)[seq[at]]
    return {"stats": stats, "rewards": r, "dlogp": dlogp}
