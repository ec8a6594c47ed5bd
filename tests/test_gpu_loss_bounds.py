"""What the loss operators promise beyond ordinary rows and sizes, on the GPU: one rounding of what is computed in 64 bits,
gradients of near-certain targets and of rows whose log-sum-exp tells nothing, results that hold no scratch memory, and
gradients over the logits that autograd and the allocator know of."""
import importlib
import math
import weakref

import numpy as np
import pytest

import loss_oracle as LO

pytestmark = pytest.mark.gpu

U = LO.U
TYPES = ["float16", "bfloat16", "float32"]


@pytest.fixture(scope="module")
def T(torch_gpu):
    return torch_gpu


@pytest.fixture(scope="module")
def losses(pkg, torch_gpu):
    return importlib.import_module(pkg.__name__ + ".losses")


def host64(t):
    return t.detach().cpu().double().numpy()


def within(got, want, bound, what):
    got, want = host64(got), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    bound = np.broadcast_to(bound, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(off - bound, nan=np.inf), -np.inf)), bad.shape) if bad.size else ()
    assert not bad.any(), "%s: %d of %d off, worst at %s by %.3g of %.3g where %.3g is allowed" % (
        what, bad.sum(), bad.size, at, off[at], want[at], bound[at])


# --- one rounding of what is computed in 64 bits ---------------------------------------------------------------------------

# Errors of one token's terms in FP64: 2^-53 for each difference, product and quotient, and for the exponential, e^d - 1 and
# e^d - d - 1 below 2^-40, 2^-38 and 2^-36 of themselves (a series up to r^10 with |r| <= ln 2 / 2).  Sums add at most a few
# thousand times 2^-53.  2^-34 of the terms' sizes covers it, a thousandth of an FP32 rounding.
REL64 = 2.0 ** -34
FLUSHED = 2.0 ** -126


def once(want, size):
    """Bound of a value that is computed in 64 bits and rounded to FP32 at the end."""
    return np.abs(want) * U * (1.0 + 1e-6) + size * REL64 + FLUSHED


def cancelling(rng, tokens, n_seqs, per_token):
    """Log-probabilities, old and reference ones, and advantages of either sign whose loss is far below its terms."""
    lp = -rng.exponential(1.0, tokens)
    old, ref = lp - rng.normal(0, 0.15, tokens), lp + rng.normal(0, 0.4, tokens)
    n = tokens if per_token else n_seqs
    adv = rng.normal(0, 1, n) + np.where(np.arange(n) % 2, 3.0, -3.0)
    return [a.astype(np.float32) for a in (lp, old, ref, rng.random(tokens) * 3, adv)]


@pytest.mark.parametrize("reduction", ["sequence", "token", "sum"])
@pytest.mark.parametrize("cu", [[0, 5], [1, 8, 10, 13], [0, 300, 307, 900, 2000], [0, 7, 1200, 4001, 4003, 30000],
                                list(range(0, 700 * 13 + 1, 13))], ids=lambda c: "%d-%d" % (len(c) - 1, c[-1]))
def test_policy_loss_is_rounded_once(losses, T, cu, reduction):
    tokens, n_seqs = cu[-1] + 2, len(cu) - 1
    seq = LO.sequences(tokens, cu)
    cu_t = T.tensor(np.array(cu, np.int32)).cuda()
    for variant in range(3):
        rng = np.random.default_rng(tokens + variant)
        per_token = variant != 1 or n_seqs == 1
        lp, old, ref, ent, adv = cancelling(rng, tokens, n_seqs, per_token)
        mask = rng.random(tokens) < 0.8
        kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.07 if variant else 0.0, entropy_coef=0.013 if variant == 2 else 0.0,
                  reduction=reduction, norm=0.3, grad_scale=3.0)
        put = lambda a: T.tensor(a).cuda()  # noqa: E731
        r = losses.policy_loss(put(lp), put(adv), old_logp=put(old), ref_logp=put(ref), entropy=put(ent),
                               mask=put(mask), cu_seqlens=cu_t, **kw)
        stats, n, dlogp, dent, size, terms, _ = LO.policy(lp, adv, seq, n_seqs, mask, old=old, ref=ref, entropy=ent, **kw)
        assert int(r.tokens) == n
        within(r.dlogp, dlogp, once(dlogp, size), "dlogp, variant %d" % variant)
        if kw["entropy_coef"]:
            within(r.dentropy, dent, once(dent, np.abs(dent)), "dentropy")
        within(r.stats, stats, once(stats, terms), "statistics, variant %d" % variant)


@pytest.mark.parametrize("rows", [14, 130])
def test_statistics_of_the_loss_from_logits_are_rounded_once(losses, T, rows):
    """Given the log-probabilities and entropies that the call returns (FP32), its statistics are sums in 64 bits."""
    vocab = 20001
    gen = T.Generator().manual_seed(rows)
    x = (T.randn(rows, vocab, generator=gen) * 2).cuda()
    t = T.randint(0, vocab, (rows,), generator=gen).cuda()
    cu = [0, 3, rows - 4, rows]
    rng = np.random.default_rng(rows)
    for reduction in ("sequence", "token", "sum"):
        lp = losses.token_logprobs(x, t).logp
        _, noise, shift, _, adv = cancelling(rng, rows, 3, True)
        old, ref = lp + T.tensor(noise).cuda() * 0.1, lp + T.tensor(shift).cuda() * 0.1
        kw = dict(kl_coef=0.07, entropy_coef=0.013, reduction=reduction, norm=0.3)
        r = losses.policy_loss_logits(x, t, T.tensor(adv).cuda(), old_logp=old, ref_logp=ref, with_entropy=True,
                                      cu_seqlens=T.tensor(cu, dtype=T.int32).cuda(), **kw)
        stats, n, _, _, _, terms, _ = LO.policy(r.logp.cpu().numpy(), adv, LO.sequences(rows, cu), 3, np.ones(rows, bool),
                                                old=old.cpu().numpy(), ref=ref.cpu().numpy(), entropy=r.entropy.cpu().numpy(), **kw)
        within(r.stats, stats, once(stats, terms), reduction)


def test_policy_gradients_of_values_out_of_range(losses, T):
    """Infinities, NaN and differences whose exponential overflows or vanishes, each token by the formula and none by its neighbours."""
    inf, nan = math.inf, math.nan
    rows = [(0, -inf, 0, 1), (0, -inf, 0, -1), (-inf, 0, 0, 1), (0, 0, -inf, 1), (nan, 0, 0, 1), (0, nan, 0, 1), (0, 0, nan, 1),
            (0, 3e38, 0, 1), (3e38, 0, 3e38, -1), (0, 0, 3e38, 1), (0, -800, 0, -1), (0, -300, 0, -1), (0, -85, 0, -1),
            (-1, -1, -1, 1), (0, 0, 0, 0), (0, 0, -3e38, 1), (-2000.5, 0, -2000, 1)]
    for copies in (1, 200):                                   # one workgroup, and more
        logp, old, ref, adv = (np.tile(np.array(c, np.float32), copies) for c in zip(*rows))
        n = len(logp)
        put = lambda a: T.tensor(a).cuda()  # noqa: E731
        r = losses.policy_loss(put(logp), put(adv), old_logp=put(old), ref_logp=put(ref), kl_coef=0.25, reduction="sum",
                               cu_seqlens=T.tensor([0, n - 1, n], dtype=T.int32).cuda())
        seq = LO.sequences(n, [0, n - 1, n])
        with np.errstate(all="ignore"):
            _, _, dlogp, _, size, _, _ = LO.policy(logp, adv, seq, 2, np.ones(n, bool), old=old, ref=ref, kl_coef=0.25, reduction="sum")
            want = np.where(np.abs(dlogp) > 3.4e38, np.sign(dlogp) * np.inf, dlogp)
        got = host64(r.dlogp)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).sum() == 3 * copies
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        assert (np.abs(got[fine] - want[fine]) <= once(want[fine], size[fine])).all()
        # the KL estimate itself: infinite where either exponential or difference is
        for i, kl in ((3, inf), (9, inf), (13, 0.0), (15, inf)):
            one = losses.policy_loss(put(logp[i:i + 1]), T.ones(1).cuda(), old_logp=put(old[i:i + 1]), ref_logp=put(ref[i:i + 1]))
            assert float(one.stats[2]) == (kl if i != 15 else float(np.float32(3e38)))


# --- gradients of near-certain targets ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (6, 513), (300, 1003), (120, 50257), (2, 151936)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("name", TYPES)
def test_certain_targets_in_the_backward(losses, T, name, temperature, rows, vocab):
    """Given the forward's log p, a target's own gradient g (1 - p) - c p (log p + H) holds relative to 1 - p.

    With R = sum over the others of exp(z_i - z_t): log p = -log1p(R) with an error of rel R / (1 + R) + 6u|log p| (rel: that of
    R, a sum like the one that slack() counts, with exponents of log(V) + |log R| on the mean), so 1 - p = -expm1(log p) moves by
    rel + 6u of itself, and expm1 (2 ulp), the temperature and two products add 8u.  The entropy is given with an error of
    2 rel (H + 1 - p), which the formula takes over, and each sum and product of that term rounds by u.
    """
    rng = np.random.default_rng(rows)
    gen = T.Generator().manual_seed(rows * 7 + vocab)
    x = (T.randn(rows, vocab, generator=gen) * 2.5).to(getattr(T, name)).cuda()
    th = np.resize([0, vocab - 1, vocab // 2, vocab - vocab % 8 - 1, vocab * 5 // 7], rows).clip(0, vocab - 1)
    t, pick = T.tensor(th).cuda(), T.arange(rows).cuda()
    lift = T.tensor(rng.uniform(1.0, 20.0, rows)).cuda()
    x[pick, t] = (((x.double() / temperature).logsumexp(1) + lift) * temperature).to(x.dtype)
    xh = host64(x) / float(np.float32(temperature))
    z = xh - xh[np.arange(rows), th][:, None]
    z[np.arange(rows), th] = -np.inf
    with np.errstate(all="ignore"):
        e = np.exp(z)
        R = e.sum(1)
        logp, miss = -np.log1p(R), R / (1 + R)
        ent = ((e * np.where(e > 0, -z, 0.0)).sum(1) + R * np.log1p(R) + np.log1p(R)) / (1 + R)
        far = np.where(R > 0, np.abs(np.log(R)), 0.0)
    assert (miss < 0.4).all()
    rel = LO.slack(vocab, LO.finite_max(xh), np.log(vocab) + far)
    g, c = (rng.normal(size=rows).astype(np.float32) for _ in range(2))
    f = losses.token_logprobs(x, t, temperature=temperature, with_entropy=True)
    put = lambda a: T.tensor(a).cuda()  # noqa: E731
    bound = np.abs(g) * miss * (rel + 14 * U)
    got = losses.token_logprobs_backward(x, t, f.lse, put(g), temperature=temperature, logp=f.logp)
    want = g * miss / temperature
    within(got[pick, t], want, np.abs(want) * LO.EPS[name] * 1.01 + bound / temperature + LO.TINY[name], "gradient")
    both = losses.token_logprobs_backward(x, t, f.lse, put(g), temperature=temperature, entropy=f.entropy, dentropy=put(c),
                                          logp=f.logp)
    want = (g * miss - c * (1 - miss) * (logp + ent)) / temperature
    bound = bound + np.abs(c) * (2 * rel * (ent + miss) + rel * miss + 16 * U * (np.abs(logp) + ent))
    within(both[pick, t], want, np.abs(want) * LO.EPS[name] * 1.01 + bound / temperature + LO.TINY[name], "with the entropy's")
    # the other logits' gradients do not ask for log p
    for a, kw in ((got, {}), (both, dict(entropy=f.entropy, dentropy=put(c)))):
        b = losses.token_logprobs_backward(x, t, f.lse, put(g), temperature=temperature, **kw)
        a[pick, t], b[pick, t] = 0.0, 0.0
        assert T.equal(a, b)
    with pytest.raises(ValueError):
        losses.token_logprobs_backward(x, t, f.lse, put(g), temperature=temperature, logp=f.logp.double())


def test_targets_without_probability_in_the_backward(losses, T):
    """log p given: targets at -inf and at a type's lowest value (p = 0), ignored and bad ones."""
    for name in TYPES:
        x = (T.randn(5, 2003, generator=T.Generator().manual_seed(4)) * 2).to(getattr(T, name)).cuda()
        x[0, 5], x[1, 6] = -math.inf, T.finfo(x.dtype).min
        t = T.tensor([5, 6, -1, 2003, 0]).cuda()
        f = losses.token_logprobs(x, t, with_entropy=True)
        g, c = T.full((5,), 0.5).cuda(), T.full((5,), 0.25).cuda()
        for kw in ({}, dict(entropy=f.entropy, dentropy=c)):
            d = losses.token_logprobs_backward(x, t, f.lse, g, logp=f.logp, **kw).float()
            assert d[0, 5] == 0.5 and d[1, 6] == 0.5 and (d[2] == 0).all() and d[3].isnan().all() and d[4].isfinite().all()
            assert T.equal(d[:2], losses.token_logprobs_backward(x, t, f.lse, g, **kw).float()[:2])


# --- rows whose log-sum-exp tells nothing ------------------------------------------------------------------------------------

@pytest.mark.parametrize("over", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("vocab", [5, 3001, 50001])
@pytest.mark.parametrize("name", TYPES)
def test_backward_of_rows_of_huge_logits(losses, T, name, vocab, temperature, over):
    """Rows whose log-sum-exp is so large that its rounding hides log V (or that overflow once divided by the temperature): the
    gradient is that of the logits less their maximum.  p is off by the rounding of (z - max) k (2u|lp|, and 2u of the
    factor), the sum and the quotient: slack() of the logits that have a share, which lie within 200 of the maximum."""
    lowest = T.finfo(getattr(T, name)).min
    rng = np.random.default_rng(vocab)
    x = T.randn(9, vocab, generator=T.Generator().manual_seed(vocab)) * 2
    t = T.tensor([0, 1, 2, vocab - 1, 3, 4, 2, 1, 0])
    x[0] = lowest
    x[1] = lowest
    x[1, 1] = -math.inf                                 # the target among those that have no share
    x[2] = 60000.0 + 32.0 * T.tensor(rng.integers(-2, 3, vocab)).float()
    x[3] = -60000.0 - 32.0 * T.tensor(rng.integers(0, 3, vocab)).float()
    x[4] = lowest
    x[4, vocab // 2:] = -math.inf
    x[5, 0] = 50000.0                                   # one logit far above the others
    x[6] = lowest                                       # ignored
    x[7] = lowest                                       # gradients of 0
    t[6] = -1
    x = x.to(getattr(T, name))
    xh, th = host64(x) / float(np.float32(temperature)), t.numpy()
    x, t = x.cuda(), t.cuda()
    g, c = rng.normal(size=9).astype(np.float32), rng.normal(size=9).astype(np.float32)
    g[7] = c[7] = 0.0
    f = losses.token_logprobs(x, t, temperature=temperature, with_entropy=True)
    top = xh.max(1, keepdims=True)
    off = xh - top
    own = np.log(np.exp(off).sum(1))
    lq = off - own[:, None]
    ent = -(np.exp(lq) * np.where(np.exp(lq) > 0, lq, 0.0)).sum(1)
    zeros = np.array([6, 7])
    for kw, with_c in (({}, False), (dict(entropy=f.entropy, dentropy=T.tensor(c).cuda()), True)):
        into = x.clone() if over else None
        for more in (dict(logp=f.logp), {}):
            got = losses.token_logprobs_backward(into if over else x, t, f.lse, T.tensor(g).cuda(), temperature=temperature,
                                                 out=into, **more, **kw)
            # of logits already divided: the temperature is 1 for the oracle, and divides its result
            d, size = LO.rows_grad(off, th, 1.0, own, g, ent, c if with_c else None)
            d, size = d / temperature, size / temperature
            rel = LO.slack(vocab, 200.0, np.abs(np.nan_to_num(lq, neginf=0.0)).clip(0, 200))
            # a p below 2^-126 comes out as 0: off by that p, times g and times c (log p + H)
            flushed = np.abs(g)[:, None] + np.abs(c)[:, None] * (np.abs(np.nan_to_num(lq, neginf=0.0)) + ent[:, None] + 1)
            bound = LO.grad_bound(name, d, size, rel) + 2.0 ** -126 * flushed / temperature
            d[zeros], bound[zeros] = 0.0, 0.0
            want_rows = [0, 1, 2, 3, 4, 5, 6, 7]
            within(got[want_rows], d[want_rows], bound[want_rows], "%s %r" % (name, sorted(kw)))
            if over:
                into = x.clone()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 3001), (40, 3001), (43, 50001)])
def test_backward_of_rows_without_an_answer(losses, T, name, rows, vocab):
    """Rows of -inf only, with a NaN, with +inf, with a bad target: NaN all over; their neighbours keep theirs."""
    import test_gpu_losses as other
    _, kind, x, t = other.broken_rows(T, name, rows, vocab)
    x, t = x.cuda(), t.cuda()
    f = losses.token_logprobs(x, t, with_entropy=True)
    one = T.ones(rows).cuda()
    for kw in ({}, dict(logp=f.logp), dict(entropy=f.entropy, dentropy=one)):
        got = losses.token_logprobs_backward(x, t, f.lse, one, **kw)
        for i, k in enumerate(kind):
            if k in (3, 4, 5, 7):
                assert got[i].isnan().all(), (i, k)
            elif k in (6, 11):
                assert (got[i] == 0).all(), (i, k)
            else:
                assert got[i].isfinite().all(), (i, k)


# --- gradients over the logits, and autograd ---------------------------------------------------------------------------------

def gradients_over(losses, T, z, t):
    """Every call that can write over the logits, as (name, call(out))."""
    f = losses.token_logprobs(z, t)
    adv, g = T.ones(1, device="cuda"), T.ones(t.shape, device="cuda")
    return [("token_logprobs_backward", lambda out: losses.token_logprobs_backward(z, t, f.lse, g, out=out)),
            ("policy_loss_logits", lambda out: losses.policy_loss_logits(
                z, t, adv, cu_seqlens=T.tensor([0, t.numel()], dtype=T.int32, device="cuda"), out=out).dlogits)]


def test_autograd_learns_that_logits_were_overwritten(losses, T):
    """A forward pass that keeps its logits for its own backward pass (a tanh) gets torch's error, not wrong gradients; one
    that does not, or whose gradient goes elsewhere, gets the right ones."""
    rows, vocab = 6, 301
    gen = T.Generator().manual_seed(0)
    h = (T.randn(rows, vocab, generator=gen) * 0.5).cuda()
    t = T.randint(0, vocab, (rows,), generator=gen).cuda()
    for which in range(2):
        w = h.clone().requires_grad_()
        z = T.tanh(w)
        what, call = gradients_over(losses, T, z, t)[which]
        before = z._version
        call(None)
        other = T.empty_like(z)
        v = other._version
        d = call(other)
        assert d is other and z._version == before and other._version > v, what
        z.backward(d)
        want = (1.0 - T.tanh(h) ** 2) * d
        assert T.allclose(w.grad, want, rtol=1e-5, atol=1e-7), what
        w = h.clone().requires_grad_()
        z = T.tanh(w)
        what, call = gradients_over(losses, T, z, t)[which]
        before = z._version
        d = call(z)
        assert d is z and z._version > before, what
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward(d)
        w = h.clone().requires_grad_()
        z = w * 2.0                                           # does not need its result
        d = gradients_over(losses, T, z, t)[which][1](z)
        z.backward(d.detach().clone())
        assert T.allclose(w.grad, 2.0 * d.detach(), rtol=1e-6)


def step_parts(host, L, T, rows=24, vocab=257, hidden=16, n_micro=3):
    st = host.ParamStore([L.TensorSpec("lm_head", vocab * hidden, L.DTYPE_F32, L.NO_DECAY, hidden)], "cuda:0")
    gen = T.Generator().manual_seed(0)
    st.param(0).copy_((T.randn(vocab, hidden, generator=gen) * 0.3).reshape(-1))
    acts = [T.randn(rows, hidden, generator=gen).cuda() for _ in range(n_micro)]
    targets = [T.randint(0, vocab, (rows,), generator=gen).cuda() for _ in range(n_micro)]
    adv = [T.randn(3, generator=gen).cuda() for _ in range(n_micro)]
    return st, host.AdamWOptimizer(st, lr=1e-2), acts, targets, adv, T.tensor([0, 7, 15, 24], dtype=T.int32).cuda()


@pytest.mark.parametrize("own_buffer", [False, True])
def test_policy_step_of_logits_that_autograd_keeps(losses, host, L, T, own_buffer):
    """A model that ends in a tanh: policy_step over its logits raises, with `out` (None, or a buffer) it is right."""
    vocab, hidden, n_micro = 257, 16, 3
    st, opt, acts, targets, adv, cu = step_parts(host, L, T)
    ref_st, ref_opt, *_ = step_parts(host, L, T)
    buffer = T.empty(24, vocab, device="cuda") if own_buffer else None

    live = {}

    def forward(k, **more):
        w = st.param(0).view(vocab, hidden).detach().clone().requires_grad_()
        z = T.tanh(acts[k] @ w.t())
        live["w"], live["z"] = w, z
        return dict(logits=z, targets=targets[k], advantages=adv[k], **more)

    def backward(k, dlogits):
        live["z"].backward(dlogits)
        st.grad(0).view(vocab, hidden).add_(live["w"].grad)

    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        host.policy_step(opt, forward, backward, n_micro, 0.01, cu_seqlens=cu)
    loss, norm, results = host.policy_step(opt, lambda k: forward(k, out=buffer), backward, n_micro, 0.01, cu_seqlens=cu)

    def plain_forward(k):
        with T.no_grad():
            z = T.tanh(acts[k] @ ref_st.param(0).view(vocab, hidden).t())
        live["y"] = z.clone()
        return dict(logits=z, targets=targets[k], advantages=adv[k])

    def plain_backward(k, d):
        ref_st.grad(0).view(vocab, hidden).add_(((1.0 - live["y"] ** 2) * d).t() @ acts[k])

    loss2, norm2, _ = host.policy_step(ref_opt, plain_forward, plain_backward, n_micro, 0.01, cu_seqlens=cu)
    assert loss == loss2 and abs(norm - norm2) <= 1e-5 * norm2 and norm > 0
    assert len(results) == n_micro and T.allclose(st.param(0), ref_st.param(0), atol=1e-5)


# --- memory ------------------------------------------------------------------------------------------------------------------

def test_policy_step_holds_one_buffer_of_logits(losses, host, L, T):
    """When forward(k + 1) runs, and when the clip does, the logits of every earlier micro-batch are gone."""
    vocab, hidden, n_micro = 257, 16, 3
    st, opt, acts, targets, adv, cu = step_parts(host, L, T)
    made = []

    def gone():
        return [r() is None for r in made]

    def forward(k):
        assert gone() == [True] * k
        z = acts[k] @ st.param(0).view(vocab, hidden).t()
        made.append(weakref.ref(z))
        return dict(logits=z, targets=targets[k], advantages=adv[k])

    def backward(k, dlogits):
        st.grad(0).view(vocab, hidden).add_(dlogits.t() @ acts[k])

    clip = opt.clip_grad_norm_

    def watched(*args, **kw):
        assert gone() == [True] * n_micro
        return clip(*args, **kw)

    opt.clip_grad_norm_ = watched
    host.policy_step(opt, forward, backward, n_micro, 1.0, cu_seqlens=cu)
    assert gone() == [True] * n_micro


@pytest.mark.parametrize("rows,vocab", [(9, 50257), (2000, 700)])
def test_results_hold_no_scratch_memory(losses, T, rows, vocab):
    """Kept statistics keep 32 bytes, not what the call worked with."""
    x, t = T.randn(rows, vocab, device="cuda"), T.zeros(rows, dtype=T.int64, device="cuda")
    adv, cu = T.ones(2, device="cuda"), T.tensor([0, 3, rows], dtype=T.int32, device="cuda")
    many = T.zeros(30000, device="cuda")
    far = T.tensor([0, 3, 30000], dtype=T.int32, device="cuda")
    for r in (losses.policy_loss_logits(x, t, adv, cu_seqlens=cu), losses.policy_loss(many, adv, cu_seqlens=far)):
        assert r.stats.untyped_storage().nbytes() == 32 and r.tokens.untyped_storage().nbytes() == 32
        assert int(r.tokens) in (rows, 30000)
