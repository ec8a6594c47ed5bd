"""The loss operators restated in 64 bits (numpy on the host), and how far a correct FP32 computation may be from them.

Error bounds (u = 2^-24, half a step of FP32 relative to the value).  z = logits / temperature, lp = log p:
  * the factor k = log2(e) / temperature carries at most 2 roundings, so every z k is off by 2u|z k|; seen from the row's
    maximum this moves a log-probability by at most 2u times the spread of z around its mean: 4u max|z| covers it;
  * z k - ref is rounded once, relative to log p: u|lp|; the exponential adds 2u (1 ulp), the product or sum that follows u;
  * a lane of a workgroup of 256 or more adds at most V/256 + 16 terms one after the other, all positive: (V/256 + 16) u,
    then 10 joins: 10u;
  * the logarithm, the last difference and the conversion to nats: 4u (1 + |lp|).
So log-probabilities and log-sum-exps are off by at most slack(V, Z, lp) = u (4 Z + 6|lp| + V/256 + 40), and a probability by that
relative to itself.
"""
import numpy as np

U = 2.0 ** -24
EPS = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}       # half a step
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -126, "float32": 2.0 ** -126}   # half a subnormal step / flushed


def slack(vocab, zmax, lp):
    return U * (4.0 * zmax + 6.0 * np.abs(lp) + vocab / 256.0 + 40.0)


def finite_max(z):
    f = np.where(np.isfinite(z), np.abs(z), 0.0)
    # masked values (a type's lowest) take no part in the sums
    f = np.where(f > 1e30, 0.0, f)
    return f.max(axis=-1)


def log_softmax(z):
    top = z.max(axis=-1, keepdims=True)
    with np.errstate(all="ignore"):
        d = z - top
        return d - np.log(np.exp(d).sum(axis=-1, keepdims=True))


def rows(logits, targets, temperature):
    """logp, lse, entropy per row; rows with a negative target 0, with a target beyond the vocabulary NaN."""
    z = logits.astype(np.float64) / temperature
    v = z.shape[-1]
    with np.errstate(all="ignore"):
        lq = log_softmax(z)
        top = z.max(axis=-1)
        lse = top + np.log(np.exp(z - top[..., None]).sum(axis=-1))
        p = np.exp(lq)
        ent = -(p * np.where(p > 0, lq, np.where(np.isnan(lq), np.nan, 0.0))).sum(axis=-1)
    logp = np.take_along_axis(lq, np.clip(targets, 0, v - 1)[..., None], -1)[..., 0]
    out = []
    for a in (logp, lse, ent):
        a = np.where(targets >= v, np.nan, a)
        out.append(np.where(targets < 0, 0.0, a))
    return out


def rows_grad(logits, targets, temperature, lse, dlogp, ent=None, dent=None):
    """Gradient of the logits from given lse / entropy, and the bound of an FP32 computation rounded to `name`."""
    z = logits.astype(np.float64) / temperature
    with np.errstate(all="ignore"):
        lq = z - lse[..., None]
        p = np.exp(lq)
        hot = np.zeros_like(z)
        np.put_along_axis(hot, np.clip(targets, 0, z.shape[-1] - 1)[..., None], 1.0, -1)
        g = dlogp[..., None].astype(np.float64)
        d = g * (hot - p)
        size = np.abs(g) * (p + hot)
        if dent is not None:
            c = dent[..., None].astype(np.float64)
            plq = np.where(p > 0, p * lq, 0.0)
            d = d - c * (plq + p * ent[..., None])
            size = size + np.abs(c) * (np.abs(plq) + p * (np.abs(ent[..., None]) + 1.0))
    d = np.where((targets < 0)[..., None], 0.0, d / temperature)
    size = np.where((targets < 0)[..., None], 0.0, size / temperature)
    return d, size


def grad_bound(name, d, size, rel):
    """|error| of a gradient whose terms of size `size` are each off by `rel`, rounded to the type."""
    return np.abs(d) * EPS[name] * 1.01 + size * (rel + 8 * U) + TINY[name]


def sequences(tokens, cu=None, n_seqs=None):
    """Sequence number per token, -1 outside."""
    seq = np.full(tokens, -1, np.int64)
    if cu is None:
        n = tokens // n_seqs if n_seqs else 0
        return np.arange(tokens) // n if n else seq
    for s in range(len(cu) - 1):
        seq[cu[s]:cu[s + 1]] = s
    return seq


def policy(logp, adv, seq, n_seqs, counts, old=None, ref=None, entropy=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
           entropy_coef=0.0, reduction="sequence", norm=1.0, grad_scale=1.0):
    """Statistics and gradients; `counts` says which tokens count.  All inputs flat; adv per sequence or per token."""
    t = len(logp)
    lo, hi = float(np.float32(clip_low)), float(np.float32(clip_high))
    kl_coef, entropy_coef = float(np.float32(kl_coef)), float(np.float32(entropy_coef))
    norm, grad_scale = float(np.float32(norm)), float(np.float32(grad_scale))
    at = np.nonzero(counts & (seq >= 0))[0]
    lp = logp.astype(np.float64)[at]
    a = (adv[at] if len(adv) == t and len(adv) != n_seqs else adv[seq[at]]).astype(np.float64)
    with np.errstate(all="ignore"):
        lr = lp - old.astype(np.float64)[at] if old is not None else np.zeros_like(lp)
        ratio = np.exp(lr)
        cut = np.where(a >= 0, lr > np.log1p(hi), lr < np.log1p(-lo))
        pol = -a * np.where(cut, np.where(a >= 0, 1 + hi, 1 - lo), ratio)
        d = ref.astype(np.float64)[at] - lp if ref is not None else np.zeros_like(lp)
        em1 = np.expm1(d)
        kl = em1 - d
    h = entropy.astype(np.float64)[at] if entropy is not None else np.zeros_like(lp)
    if reduction == "token":
        w = np.full(len(at), norm / max(len(at), 1))
    elif reduction == "sum":
        w = np.full(len(at), norm)
    else:
        n = np.bincount(seq[at], minlength=max(n_seqs, 1))
        w = norm / (n_seqs * n[seq[at]].astype(np.float64))
    parts = [(w * pol).sum(), (w * kl).sum(), (w * h).sum()]
    loss = parts[0] + (kl_coef * parts[1] if kl_coef else 0.0) - (entropy_coef * parts[2] if entropy_coef else 0.0)
    m = max(len(at), 1)
    stats = np.array([loss] + parts + [cut.sum() / m, ratio.sum() / m])
    dlogp, dent = np.zeros(t), np.zeros(t)
    dlogp[at] = grad_scale * w * (np.where(cut, 0.0, -a * ratio) - (kl_coef * em1 if kl_coef else 0.0))
    dent[at] = -grad_scale * w * entropy_coef
    # sizes of what is added up, for the bounds
    size = np.zeros(t)
    size[at] = np.abs(grad_scale) * w * (np.where(cut, 0.0, np.abs(a) * ratio) + np.abs(kl_coef * em1))
    terms = np.array([(w * (np.abs(pol) + abs(kl_coef) * np.abs(kl) + abs(entropy_coef) * np.abs(h))).sum(),
                      (w * np.abs(pol)).sum(), (w * np.abs(kl)).sum(), (w * np.abs(h)).sum(), 1.0, ratio.sum() / m])
    # how fast the terms move with the log-probability (for those that are computed, not given)
    moves = np.array([(w * (np.abs(a) * ratio + abs(kl_coef) * np.abs(em1))).sum(), (w * np.abs(a) * ratio).sum(),
                      (w * np.abs(em1)).sum(), 0.0, 0.0, ratio.sum() / m])
    return stats, len(at), dlogp, dent, size, terms, moves


def preference(logp, seq, n_pairs, counts, ref=None, beta=0.1, smoothing=0.0, margin=0.0, average=False, grad_scale=1.0):
    beta, smoothing, margin = (float(np.float32(x)) for x in (beta, smoothing, margin))
    at = np.nonzero(counts & (seq >= 0))[0]
    d = logp.astype(np.float64)[at] - (ref.astype(np.float64)[at] if ref is not None else 0.0)
    sums = np.bincount(seq[at], weights=d, minlength=2 * n_pairs)
    n = np.maximum(np.bincount(seq[at], minlength=2 * n_pairs), 1)
    per = beta / n if average else np.full(2 * n_pairs, beta)
    r = sums * per
    diff = r[:n_pairs] - r[n_pairs:]
    x = diff - margin
    ls, lsn = -np.logaddexp(0.0, -x), -np.logaddexp(0.0, x)
    loss = -(1 - smoothing) * ls - smoothing * lsn
    dx = (smoothing * np.exp(ls) - (1 - smoothing) * np.exp(lsn)) / max(n_pairs, 1)
    m = max(n_pairs, 1)
    stats = np.array([loss.sum(), (diff > 0).sum(), diff.sum(), r[:n_pairs].sum(), r[n_pairs:].sum()]) / m
    dlogp = np.zeros(len(logp))
    dlogp[at] = (np.concatenate([dx, -dx]) * per)[seq[at]] * grad_scale
    return stats, r, dlogp
