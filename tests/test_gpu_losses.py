"""The loss operators on the GPU against their restatement in 64 bits (loss_oracle, whose docstring derives the bounds)."""
import importlib
import math

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


def make_logits(torch, rows, vocab, name, seed, lift=True):
    """Rows of a type's own values on the GPU, their FP64 values on the host, and targets that are often likely."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2.5
    t = torch.randint(0, vocab, (rows,), generator=g)
    if lift:
        x[torch.arange(rows), t] += torch.rand(rows, generator=g) * 12
    x = x.to(getattr(torch, name))
    return x.cuda(), x.double().numpy(), t.cuda(), t.numpy()


def host(t):
    return t.detach().cpu().double().numpy()


def check(got, want, bound, what):
    got, want = host(got), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what + ": infinities"
    bound = np.broadcast_to(bound, want.shape)[fine]
    off = np.abs(got[fine] - want[fine])
    assert (off <= bound).all(), "%s: off by %.3g where %.3g is allowed" % (
        what, off[np.argmax(off - bound)], bound[np.argmax(off - bound)])


def check_forward(losses, torch, x, xh, t, th, temperature, what, entropy=True):
    r = losses.token_logprobs(x, t, temperature=temperature, with_entropy=entropy)
    logp, lse, ent = LO.rows(xh, th, temperature)
    v, z = xh.shape[-1], LO.finite_max(xh / temperature)
    check(r.logp, logp, LO.slack(v, z, np.nan_to_num(logp, neginf=0.0)), what + " logp")
    check(r.lse, lse, LO.slack(v, z, np.nan_to_num(lse, neginf=0.0)), what + " lse")
    if entropy:
        # the entropy is a mean of -log p: the same bound with the size of the log p that weigh (at most log V + H)
        check(r.entropy, ent, LO.slack(v, z, np.log(v) + np.nan_to_num(ent)) * 2, what + " entropy")
    else:
        assert r.entropy is None
    return r


SHAPES = [(1, 1), (1, 2), (3, 7), (2, 8), (4, 9), (70, 33), (3, 513), (2, 4095), (5, 4099), (300, 1000), (2, 32003),
          (9, 50257), (1, 151936), (17, 151936), (2, 200001)]
# statistics of whole rows by one large workgroup
WIDE = [(11, 20003), (3, 32768), (97, 32777), (129, 50257), (99, 70001)]


@pytest.mark.parametrize("rows,vocab", SHAPES + WIDE)
@pytest.mark.parametrize("name", TYPES)
def test_forward(losses, T, name, rows, vocab):
    x, xh, t, th = make_logits(T, rows, vocab, name, rows * 31 + vocab)
    for temperature, entropy in ((1.0, True), (0.7, False)):
        check_forward(losses, T, x, xh, t, th, temperature, "%s %dx%d" % (name, rows, vocab), entropy)
    r32 = losses.token_logprobs(x, t.int(), with_entropy=True)
    r64 = losses.token_logprobs(x, t, with_entropy=True)
    for a, b in zip(r32, r64):
        assert T.equal(a, b)                        # both index types, and the same bits on every run


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (6, 513), (300, 1003), (4, 50257), (120, 50257), (2, 151936), (99, 200001)])
@pytest.mark.parametrize("name", TYPES)
def test_certain_targets(losses, T, name, rows, vocab):
    """A target with nearly all of the probability: log p, 1 - p and the entropy hold relative to themselves.

    With R = sum over the others of exp(z_i - z_t): log p = -log1p(R), and 1 - p = R / (1 + R) moves by R's relative error
    times 1 - p at most.  R is a sum of positive terms like the one that slack() counts, whose exponents are log(V) + |log R|
    on the mean over the terms; the quotient, log1p (2 ulp) and the result add 6u.
    """
    x, _, t, th = make_logits(T, rows, vocab, name, rows * 7 + vocab, lift=False)
    rng = np.random.default_rng(rows)
    th = np.resize([0, vocab - 1, vocab // 2, vocab - vocab % 8 - 1, vocab * 5 // 7], rows).clip(0, vocab - 1)
    t = T.tensor(th).cuda()
    pick = T.arange(rows).cuda()
    lift = T.tensor(rng.uniform(1.0, 30.0, rows)).cuda()
    x[pick, t] = (x.double().logsumexp(1) + lift).to(x.dtype)
    xh = x.cpu().double().numpy()
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
    r = losses.token_logprobs(x, t, with_entropy=True)
    check(r.logp, logp, rel * miss + 6 * U * np.abs(logp) + 1e-37, "logp")
    # every -p log p moves by its p's error and by the log's, which is of R's relative size for the target and rel for others
    check(r.entropy, ent, 2 * rel * (ent + miss) + 1e-37, "entropy")
    adv = rng.normal(size=rows).astype(np.float32)
    f = losses.policy_loss_logits(x, t, T.tensor(adv).cuda(), cu_seqlens=T.arange(rows + 1, dtype=T.int32).cuda(), reduction="sum")
    check(f.logp, logp, rel * miss + 6 * U * np.abs(logp) + 1e-37, "fused logp")
    want = -adv.astype(np.float64) * miss
    check(f.dlogits[pick, t].double(), want, np.abs(want) * (LO.EPS[name] * 1.01 + rel + 8 * U) + LO.TINY[name], "fused gradient")


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("name", TYPES)
def test_backward(losses, T, name, rows, vocab):
    x, xh, t, th = make_logits(T, rows, vocab, name, rows * 17 + vocab)
    rng = np.random.default_rng(vocab)
    g = rng.normal(size=rows).astype(np.float32)
    c = (rng.normal(size=rows) * 0.1).astype(np.float32)
    if rows > 2:
        g[1], c[1] = 0.0, 0.0
        th = th.copy()
        th[2] = -1
        t = T.tensor(th).cuda()
    for temperature, with_c in ((1.0, False), (0.6, True)):
        r = losses.token_logprobs(x, t, temperature=temperature, with_entropy=True)
        lse, ent = host(r.lse), host(r.entropy)
        gt, ct = T.tensor(g).cuda(), T.tensor(c).cuda()
        kw = dict(entropy=r.entropy, dentropy=ct) if with_c else {}
        got = losses.token_logprobs_backward(x, t, r.lse, gt, temperature=temperature, **kw)
        d, size = LO.rows_grad(xh, th, temperature, lse, g, ent, c if with_c else None)
        # p = exp(z - lse) from the given lse: the temperature's reciprocal (u |z|), one rounding of the difference and
        # one of its product with log2 e (2u |lp|), the exponential (2u) and the products (4u)
        zmax = LO.finite_max(xh / temperature)
        with np.errstate(all="ignore"):
            lp = np.abs(xh / temperature - lse[:, None])
        rel = U * (2 * zmax[:, None] + 3 * np.minimum(lp, 200.0) + 12)
        check(got, d, LO.grad_bound(name, d, size, rel), "%s %dx%d" % (name, rows, vocab))
        again = x.clone()
        assert losses.token_logprobs_backward(again, t, r.lse, gt, temperature=temperature, out=again, **kw) is again
        assert T.equal(again, got)                  # over the logits: the same bits


def test_views_of_logits(losses, T):
    """Rows of every layout that is promised, against the contiguous copy: the same bits."""
    base = (T.randn(6, 5, 1003, generator=T.Generator().manual_seed(5)) * 2).half().cuda()
    t = T.randint(0, 500, (6, 5), generator=T.Generator().manual_seed(6)).cuda()
    views = {"shifted": (base[:, :-1], t[:, :-1].contiguous()),
             "columns": (base[:, :, 3:902], t),
             "swapped": (base.transpose(0, 1), t.t().contiguous()),
             "every other row": (base[::2], t[::2].contiguous()),
             "every other position": (base[:, ::2], t[:, ::2].contiguous()),
             "one row": (base[3:4, 2:3], t[3:4, 2:3].contiguous()),
             "one column of rows": (base[:, 4], t[:, 4].contiguous())}
    for what, (x, tt) in views.items():
        a = losses.token_logprobs(x, tt, with_entropy=True)
        b = losses.token_logprobs(x.contiguous(), tt, with_entropy=True)
        for u, v in zip(a, b):
            assert T.equal(u, v), what
        g = T.randn(tt.shape, generator=T.Generator().manual_seed(7)).cuda()
        want = losses.token_logprobs_backward(x.contiguous(), tt, b.lse, g)
        assert T.equal(losses.token_logprobs_backward(x, tt, b.lse, g), want), what
        copy = base.clone()
        into = copy.as_strided(x.shape, x.stride(), x.storage_offset())
        losses.token_logprobs_backward(into, tt, b.lse, g, out=into)
        assert T.equal(into, want), what
        touched = T.zeros_like(copy, dtype=T.bool)
        touched.as_strided(x.shape, x.stride(), x.storage_offset()).fill_(True)
        assert T.equal(copy[~touched], base[~touched]), what + ": written outside the rows"
    x4 = base.reshape(6, 5, 17, 59)[:, ::2, ::2]
    with pytest.raises(ValueError, match="contiguous"):
        losses.token_logprobs(x4, T.zeros(x4.shape[:-1], dtype=T.int64, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        losses.token_logprobs(base[:, :, ::2], t)
    with pytest.raises(losses.B.RlxError):
        losses.token_logprobs(base[0, 0].expand(4, 1003), t[0, :4].contiguous())


@pytest.mark.parametrize("name", TYPES)
def test_starts_of_rows(losses, T, name):
    """Every alignment of a row's first element, of input and output."""
    vocab = 2051
    flat = (T.randn(3 * 2100, generator=T.Generator().manual_seed(1)) * 2).to(getattr(T, name)).cuda()
    t = T.tensor([0, 2050, 777]).cuda()
    g = T.tensor([1.0, -0.5, 0.25]).cuda()
    for start in range(9):
        x = flat[start:].as_strided((3, vocab), (vocab + start % 3, 1), start)
        r = losses.token_logprobs(x, t, with_entropy=True)
        want = losses.token_logprobs(x.contiguous(), t, with_entropy=True)
        assert all(T.equal(a, b) for a, b in zip(r, want))
        d = losses.token_logprobs_backward(x.contiguous(), t, r.lse, g)
        room = T.full((3 * 2100,), 7.0, dtype=flat.dtype, device="cuda")
        out = room.as_strided((3, vocab), (vocab + 5, 1), 8 - start)
        assert T.equal(losses.token_logprobs_backward(x, t, r.lse, g, out=out), d)
        out.fill_(7.0)
        assert (room == 7.0).all()


def broken_rows(T, name, rows, vocab):
    """Rows with masked, lowest, infinite and NaN logits, ignored and bad targets; the kind of each, logits and targets (host)."""
    dt = getattr(T, name)
    lowest = T.finfo(dt).min
    x = (T.randn(rows, vocab, generator=T.Generator().manual_seed(rows)) * 2).to(dt)
    t = T.randint(0, 1000, (rows,), generator=T.Generator().manual_seed(3))
    kinds = {0: "banned -inf", 1: "banned lowest", 2: "all lowest", 3: "all -inf", 4: "a NaN", 5: "+inf", 6: "ignored",
             7: "bad target", 8: "target -inf", 9: "one left", 10: "all equal", 11: "ignored -100"}
    kind = [i % 12 if rows > 1 else 2 for i in range(rows)]
    for i, k in enumerate(kind):
        if k == 0:
            x[i, 1000:] = -math.inf
        elif k == 1:
            x[i, 1000:] = lowest
        elif k == 2:
            x[i] = lowest
        elif k == 3:
            x[i] = -math.inf
        elif k == 4:
            x[i, 1234] = math.nan
        elif k == 5:
            x[i, 17] = math.inf
        elif k in (6, 11):
            x[i, ::2] = math.nan
            t[i] = -1 if k == 6 else -100
        elif k == 7:
            t[i] = vocab if i % 2 else 1 << 40
        elif k == 8:
            x[i, t[i]] = -math.inf
        elif k == 9:
            x[i] = -math.inf
            x[i, t[i]] = 1.5
        elif k == 10:
            x[i] = 3.25
    return kinds, kind, x, t


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 3001), (40, 3001), (700, 3001), (1, 50001), (43, 50001), (130, 50001)])
def test_masked_and_broken_rows(losses, T, name, rows, vocab):
    kinds, kind, x, t = broken_rows(T, name, rows, vocab)
    xh, th = x.double().numpy(), t.numpy()
    x, t = x.cuda(), t.cuda()
    r = losses.token_logprobs(x, t, with_entropy=True)
    logp, lse, ent = LO.rows(xh, th, 1.0)
    z = LO.finite_max(xh)
    nz = lambda a: np.nan_to_num(a, nan=0.0, neginf=0.0)  # noqa: E731
    check(r.logp, logp, LO.slack(vocab, z, nz(logp)), "logp")
    check(r.lse, lse, LO.slack(vocab, np.where(np.abs(nz(lse)) > 1e30, np.abs(nz(lse)), z), nz(lse)), "lse")
    check(r.entropy, ent, 2 * LO.slack(vocab, z, np.log(vocab) + nz(ent)), "entropy")
    # gradients of the rows that have one: finite where the formula is, and untouched by what their neighbours hold
    g = T.ones(rows).cuda()
    got = host(losses.token_logprobs_backward(x, t, r.lse, g))
    for i, k in enumerate(kind):
        if k in (6, 11):
            assert (got[i] == 0).all()
        elif k in (3, 4, 5, 7):
            assert np.isnan(got[i]).all() or k == 5 or k == 4
        elif k != 2:                                  # lse of an all-lowest row holds no log V
            d, size = LO.rows_grad(xh[i:i + 1], th[i:i + 1], 1.0, host(r.lse)[i:i + 1], np.ones(1))
            assert (np.abs(got[i] - d[0]) <= LO.grad_bound(name, d, size, U * 800)[0]).all(), kinds[k]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,vocab", [(40, 3001), (1, 50001), (43, 50001), (130, 50001), (13, 160003), (100, 160003)])
@pytest.mark.parametrize("over", [False, True])
def test_masked_and_broken_rows_in_the_loss(losses, T, name, rows, vocab, over):
    """The loss straight from such logits, a sequence per row: with old_logp absent and the plain sum, dlogits = -A (1[j = t] - p)."""
    kinds, kind, x, t = broken_rows(T, name, rows, vocab)
    xh, th = x.double().numpy(), t.numpy()
    x, t = x.cuda(), t.cuda()
    adv = np.random.default_rng(rows).normal(size=rows).astype(np.float32)
    cu = T.arange(rows + 1, dtype=T.int32).cuda()
    r = losses.policy_loss_logits(x, t, T.tensor(adv).cuda(), cu_seqlens=cu, reduction="sum", with_entropy=True,
                                  out=x if over else None)
    logp, _, ent = LO.rows(xh, th, 1.0)
    z, nz = LO.finite_max(xh), lambda a: np.nan_to_num(a, nan=0.0, neginf=0.0)
    check(r.logp, logp, LO.slack(vocab, z, nz(logp)), "logp")
    check(r.entropy, ent, 2 * LO.slack(vocab, z, np.log(vocab) + nz(ent)), "entropy")
    got = host(r.dlogits)
    for i, k in enumerate(kind):
        if k in (6, 11):
            assert (got[i] == 0).all()
        elif k in (3, 4, 5, 7):
            assert np.isnan(got[i]).all(), kinds[k]
        else:
            # of logits less their maximum: beside a lowest value of 1e38 even 64 bits hold no log V
            off = xh[i:i + 1] - xh[i].max()
            own = np.log(np.exp(off).sum(1))
            d, size = LO.rows_grad(off, th[i:i + 1], 1.0, own, -adv[i:i + 1])
            rel = LO.slack(vocab, z[i], np.log(vocab) + np.abs(nz(off - own)).clip(0, 200))
            assert (np.abs(got[i] - d[0]) <= LO.grad_bound(name, d, size, rel)[0]).all(), kinds[k]


@pytest.mark.parametrize("name,size,temperature", [("float16", 60000.0, 1.0), ("float16", 100.0, 1e-3),
                                                   ("bfloat16", 1e30, 1.0), ("float32", 3e8, 1.0), ("float32", 1e20, 2.0),
                                                   ("float32", 1e9, 0.5), ("float32", 1e-30, 1.0)])
def test_extreme_sizes(losses, T, name, size, temperature):
    dt = getattr(T, name)
    x = (T.rand(5, 1777, generator=T.Generator().manual_seed(8)) * 2 - 1).double() * size
    x[1] = -x[1].abs()
    x[2, :-1] = -size
    x = x.to(dt)
    t = x.argmax(1)
    t[4] = 5
    xh, th = x.double().numpy(), t.numpy()
    check_forward(losses, T, x.cuda(), xh, t.cuda(), th, temperature, "%s %g" % (name, size))


def test_rows_beyond_32_bits(losses, T):
    """Row starts past 2^31 and 2^32 elements."""
    vocab, stride = 1500, (1 << 32) // 2 + 12345
    room = T.empty(2 * stride + vocab, dtype=T.float16, device="cuda")
    x = room.as_strided((3, vocab), (stride, 1))
    x.copy_(T.randn(3, vocab, generator=T.Generator().manual_seed(9)))
    t = T.tensor([3, 1499, 700]).cuda()
    a, b = losses.token_logprobs(x, t), losses.token_logprobs(x.contiguous(), t)
    assert T.equal(a.logp, b.logp) and T.equal(a.lse, b.lse)
    g = T.ones(3).cuda()
    want = losses.token_logprobs_backward(x.contiguous(), t, b.lse, g)
    assert T.equal(losses.token_logprobs_backward(x, t, b.lse, g, out=x), want)
    adv = T.ones(1).cuda()
    x.copy_(T.randn(3, vocab, generator=T.Generator().manual_seed(9)))
    want = losses.policy_loss_logits(x.contiguous(), t, adv, cu_seqlens=T.tensor([0, 3], dtype=T.int32).cuda())
    got = losses.policy_loss_logits(x, t, adv, cu_seqlens=T.tensor([0, 3], dtype=T.int32).cuda(), out=x)
    assert T.equal(got.dlogits, want.dlogits) and T.equal(got.stats, want.stats)


# --- policy loss --------------------------------------------------------------------------------------------------------

CU = [[0, 1], [0, 5], [0, 0, 3, 3, 10], [2, 2, 700, 1500, 1500], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11],
      [5, 20000], [0] + list(np.cumsum([1 + (i * 37) % 91 for i in range(900)])), [0, 0, 0], [0, 300, 40000, 41000]]


def policy_inputs(torch, tokens, n_seqs, per_token, seed):
    rng = np.random.default_rng(seed)
    lp = -rng.exponential(1.0, tokens)
    d = {"logp": lp, "old_logp": lp - rng.normal(0, 0.15, tokens), "ref_logp": lp + rng.normal(0, 0.4, tokens),
         "entropy": rng.random(tokens) * 3, "advantages": rng.normal(0, 1, tokens if per_token else n_seqs)}
    d = {k: v.astype(np.float32) for k, v in d.items()}
    if not per_token and n_seqs > 2:
        d["advantages"][1] = 0.0
    return d, {k: torch.tensor(v).cuda() for k, v in d.items()}, rng


def check_policy(r, want, tokens, what, moved=0.0):
    """moved: how far the log-probabilities themselves may be off (where they are computed).  Each term carries the
    exponential's 2u, the difference's u and up to four more roundings; sums are in 64 bits and rounded once."""
    stats, n, dlogp, dent, size, terms, moves = want
    assert int(r.tokens) == n, what
    bound = terms * 12 * U + np.abs(stats) * U * 1.01 + moves * moved + 1e-37
    check(r.stats, stats, bound, what + " stats")
    return dlogp, dent, size


@pytest.mark.parametrize("cu", CU, ids=lambda c: "%d-%d" % (len(c) - 1, c[-1]))
@pytest.mark.parametrize("reduction", ["sequence", "token", "sum"])
def test_policy_loss(losses, T, cu, reduction):
    tokens, n_seqs = cu[-1] + (3 if len(cu) % 2 else 0), len(cu) - 1
    seq = LO.sequences(tokens, cu)
    cu_t = T.tensor(np.array(cu, np.int32)).cuda()
    for variant in range(4):
        per_token = variant % 2 == 1
        h, d, rng = policy_inputs(T, tokens, n_seqs, per_token, variant + tokens)
        mask = rng.random(tokens) < (0.0 if variant == 3 else 0.7)
        mask_t = T.tensor(mask).cuda() if variant else None
        counts = mask if variant else np.ones(tokens, bool)
        kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05 * variant, reduction=reduction,
                  entropy_coef=0.01 * (variant % 2), norm=0.5 if reduction == "sum" else 1.0, grad_scale=8.0)
        use = dict(old_logp=d["old_logp"], ref_logp=d["ref_logp"], entropy=d["entropy"]) if variant < 3 else {}
        if variant and variant < 3:                            # what masked tokens hold is not used
            for k in ("logp", "old_logp", "ref_logp", "entropy"):
                d[k][~mask_t] = math.nan if variant == 1 else math.inf
        if variant == 3:
            kw["entropy_coef"] = 0.0
        r = losses.policy_loss(d["logp"], d["advantages"], mask=mask_t, cu_seqlens=cu_t, **use, **kw)
        hu = dict(old=h["old_logp"], ref=h["ref_logp"], entropy=h["entropy"]) if variant < 3 else {}
        want = LO.policy(h["logp"], h["advantages"], seq, n_seqs, counts, **hu, **kw)
        dlogp, dent, size = check_policy(r, want, tokens, "variant %d" % variant)
        check(r.dlogp, dlogp, size * 12 * U + 1e-37, "dlogp")
        if kw["entropy_coef"]:
            check(r.dentropy, dent, np.abs(dent) * 4 * U + 1e-37, "dentropy")
        else:
            assert r.dentropy is None
        again = losses.policy_loss(d["logp"], d["advantages"], mask=mask_t, cu_seqlens=cu_t, **use, **kw)
        assert T.equal(again.stats, r.stats) and T.equal(again.dlogp, r.dlogp)


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 2047, 2049])
@pytest.mark.parametrize("n_seqs", [1, 3, 1024, 5000])
@pytest.mark.parametrize("reduction", ["sequence", "token"])
def test_policy_loss_of_few_tokens_and_many_sequences(losses, T, tokens, n_seqs, reduction):
    rng = np.random.default_rng(tokens + n_seqs)
    cu = np.sort(rng.integers(0, tokens + 1, n_seqs + 1))
    cu[0], cu[-1] = 0, tokens
    h, d, rng = policy_inputs(T, tokens, n_seqs, False, 7)
    mask = rng.random(tokens) < 0.9
    kw = dict(kl_coef=0.1, reduction=reduction)
    r = losses.policy_loss(d["logp"], d["advantages"], old_logp=d["old_logp"], ref_logp=d["ref_logp"],
                           mask=T.tensor(mask).cuda(), cu_seqlens=T.tensor(cu.astype(np.int32)).cuda(), **kw)
    seq = LO.sequences(tokens, cu)
    # the oracle tells advantages per token and per sequence apart by their number
    adv = h["advantages"] if n_seqs == tokens else h["advantages"][seq]
    want = LO.policy(h["logp"], adv, seq, n_seqs, mask, old=h["old_logp"], ref=h["ref_logp"], **kw)
    dlogp, _, size = check_policy(r, want, tokens, "few tokens")
    check(r.dlogp, dlogp, size * 12 * U + 1e-37, "dlogp")
    if n_seqs > 1:                                             # the same offsets as pairs
        cu2 = cu if n_seqs % 2 == 0 else np.append(cu, tokens)
        p = losses.preference_loss(d["logp"], ref_logp=d["ref_logp"], mask=T.tensor(mask).cuda(),
                                   cu_seqlens=T.tensor(cu2.astype(np.int32)).cuda(), beta=0.3)
        stats, rewards, dl = LO.preference(h["logp"], LO.sequences(tokens, cu2), (len(cu2) - 1) // 2, mask,
                                           ref=h["ref_logp"], beta=0.3)
        check(p.rewards, rewards, np.abs(rewards) * 2 * U + 1e-12, "rewards")
        check(p.dlogp, dl, np.abs(dl) * 2 * U + 1e-37, "pairs dlogp")
        check(p.stats, stats, np.abs(stats) * 2 * U + 1e-12, "pairs stats")


def test_policy_loss_padded_batch(losses, T):
    h, d, rng = policy_inputs(T, 6 * 111, 6, False, 4)
    mask = rng.random((6, 111)) < 0.6
    mask[2] = False                                   # a sequence whose mask leaves nothing
    sq = {k: (v if k == "advantages" else v.reshape(6, 111)) for k, v in d.items()}
    r = losses.policy_loss(sq["logp"], sq["advantages"], old_logp=sq["old_logp"], ref_logp=sq["ref_logp"],
                           mask=T.tensor(mask).cuda(), kl_coef=0.1)
    want = LO.policy(h["logp"], h["advantages"], LO.sequences(666, n_seqs=6), 6, mask.reshape(-1), old=h["old_logp"],
                     ref=h["ref_logp"], kl_coef=0.1)
    dlogp, _, size = check_policy(r, want, 666, "padded")
    check(r.dlogp.reshape(-1), dlogp, size * 12 * U + 1e-37, "dlogp")
    one = losses.policy_loss(d["logp"], T.ones(1).cuda())        # one sequence without offsets, on-policy
    assert np.allclose(host(one.stats), [-1.0, -1.0, 0, 0, 0, 1.0], rtol=1e-6) and int(one.tokens) == 666
    assert T.allclose(one.dlogp, T.full_like(one.dlogp, -1.0 / 666), rtol=1e-6)


def test_policy_loss_edges(losses, T):
    """Ratios out of range, an advantage of 0, differences near and far from 0 in the KL term, the clip's borders."""
    f = np.float32
    lo, hi = math.log1p(-float(f(0.2))), math.log1p(float(f(0.2)))
    up = lambda x: np.nextafter(f(x), f(9))       # noqa: E731
    dn = lambda x: np.nextafter(f(x), f(-9))      # noqa: E731
    old = np.array([-100, 100, -100, 0, 0, 0, 0, 0, 0, 0, 0, -100], f)
    logp = np.array([0, 0, 0, dn(dn(hi)), up(up(hi)), up(up(lo)), dn(dn(lo)), 1e-3, 0, 0, 0, 0], f)
    ref = np.array([0, 0, 0, 0, 0, 0, 0, 2e-3, 1e-6, 60, -60, 0], f)
    adv = np.array([1, 1, 0, 1, 1, -1, -1, 1, -1, 1, 1, -1], f)
    n = len(old)
    r = losses.policy_loss(T.tensor(logp).cuda(), T.tensor(adv).cuda(), old_logp=T.tensor(old).cuda(),
                           ref_logp=T.tensor(ref).cuda(), cu_seqlens=T.tensor([0, n], dtype=T.int32).cuda(),
                           kl_coef=0.5, reduction="sum")
    g = host(r.dlogp)
    em1 = np.expm1(ref.astype(np.float64) - logp)
    slope = [0, 0, 0, None, 0, None, 0, None, None, None, None, math.inf]
    for i in range(n):
        if slope[i] == math.inf:
            assert g[i] > 1e38                       # A < 0 is not clipped upwards: the formula's own overflow
            continue
        ratio = math.exp(float(logp[i]) - float(old[i])) if slope[i] is None else 0.0
        want = (-float(adv[i]) * ratio) - 0.5 * em1[i]
        if i == 1:                                   # rho = e^-100, not clipped for A >= 0
            want = -math.exp(-100.0) - 0.5 * em1[i]
        assert abs(g[i] - want) <= 12 * U * (abs(adv[i]) * ratio + abs(0.5 * em1[i])) + 1e-37, i
    # the KL term near 0 keeps its relative precision
    for d in (1e-6, -1e-4, 3e-3, -0.1, 0.49999, 0.5, 0.7, -3.0, 20.0):
        one = losses.policy_loss(T.zeros(1).cuda(), T.zeros(1).cuda(), ref_logp=T.tensor([f(d)]).cuda(), kl_coef=1.0)
        x = float(f(d))
        want = math.expm1(x) - x if abs(x) > 1e-2 else x * x / 2 * (1 + x / 3 + x * x / 12 + x ** 3 / 60)
        assert abs(float(one.stats[2]) - want) <= 30 * U * want, d


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 5), (7, 33), (3, 4099), (40, 1000), (700, 515), (11, 50257), (2, 151936),
                                        (530, 8200), (5, 200001)])
def test_policy_loss_logits(losses, T, name, rows, vocab):
    x, xh, t, th = make_logits(T, rows, vocab, name, rows + 3 * vocab)
    cu = sorted({0, rows // 3, rows // 2, rows - rows // 7})
    cu = [0, 0] + cu[1:] if len(cu) > 1 else [0, rows]
    n_seqs = len(cu) - 1
    seq = LO.sequences(rows, cu)
    for variant in range(3):
        temperature = (1.0, 0.7, 1.3)[variant]
        logp, lse, ent = LO.rows(xh, th, temperature)
        rng = np.random.default_rng(variant)
        # ratios that no rounding of a log-probability carries over the clip's borders
        lr = rng.normal(0, 0.15, rows)
        for border in (math.log1p(-0.2), math.log1p(0.3)):
            lr = np.where(np.abs(lr - border) < 0.01, border + 0.02, lr)
        old = (logp - lr).astype(np.float32)
        ref = (logp + rng.normal(0, 0.3, rows)).astype(np.float32)
        per_token = variant == 1
        adv = rng.normal(0, 1, rows if per_token else n_seqs).astype(np.float32)
        mask = rng.random(rows) < 0.8
        tt = th.copy()
        if rows > 4:
            tt[4] = -1
        xv = x.clone()
        xv[T.tensor(~mask).cuda()] = math.nan           # prompt rows are not read
        mask_t = T.tensor(mask).cuda()
        kw = dict(clip_low=0.2, clip_high=0.3, kl_coef=0.05, entropy_coef=0.02 if variant == 2 else 0.0,
                  reduction=("sequence", "token", "sum")[variant], norm=0.5, grad_scale=64.0)
        args = dict(old_logp=T.tensor(old).cuda(), ref_logp=T.tensor(ref).cuda(), mask=mask_t,
                    cu_seqlens=T.tensor(np.array(cu, np.int32)).cuda(), temperature=temperature, with_entropy=True)
        tg, ag = T.tensor(tt).cuda(), T.tensor(adv).cuda()
        r = losses.policy_loss_logits(xv, tg, ag, **args, **kw)
        counts = mask & (tt >= 0) & (seq >= 0)
        want = LO.policy(logp, adv, seq, n_seqs, counts, old=old, ref=ref, entropy=ent, **kw)
        zmax = LO.finite_max(xh / temperature)
        moved = LO.slack(vocab, zmax, logp)
        dlogp, dent, size = check_policy(r, want, rows, "variant %d" % variant,
                                         moved=float(moved[counts].max()) if counts.any() else 0.0)
        check(r.logp, np.where(counts, logp, 0.0), moved, "logp")
        check(r.entropy, np.where(counts, ent, 0.0), 2 * LO.slack(vocab, zmax, np.log(vocab) + ent), "entropy")
        d, dsize = LO.rows_grad(xh, np.where(counts, tt, -1), temperature, lse, dlogp, ent,
                                dent if kw["entropy_coef"] else None)
        # the row's factor moves with its log-probability (d rho = rho d logp, d e^d likewise, and 12u of its own);
        # a probability is off by its own log-probability's slack
        _, gsize = LO.rows_grad(xh, np.where(counts, tt, -1), temperature, lse, size + 0.1 * 64.0 * 0.05)
        with np.errstate(all="ignore"):
            lp = np.minimum(np.abs(xh / temperature - lse[:, None]), 200.0)
        rel = U * (4 * zmax[:, None] + 8 * lp + vocab / 256 + 60)
        w = np.abs(gsize) * (2 * moved[:, None] + 12 * U)
        check(r.dlogits, d, LO.grad_bound(name, d, dsize, rel) + w, "dlogits")
        again = losses.policy_loss_logits(xv, tg, ag, out=xv, **args, **kw)        # over the logits
        assert again.dlogits is xv and T.equal(xv, r.dlogits) and T.equal(again.stats, r.stats)


def test_policy_loss_logits_equals_the_separate_operators(losses, T):
    """One call against token_logprobs -> policy_loss -> token_logprobs_backward on a padded, shifted batch."""
    b, s, vocab = 5, 41, 3001
    full = (T.randn(b, s + 1, vocab, generator=T.Generator().manual_seed(2)) * 2).cuda()
    x = full[:, :-1]
    t = T.randint(0, vocab, (b, s), generator=T.Generator().manual_seed(3)).cuda()
    mask = (T.rand(b, s, generator=T.Generator().manual_seed(4)) < 0.7).cuda()
    adv = T.randn(b, generator=T.Generator().manual_seed(5)).cuda()
    f = losses.token_logprobs(x, t, with_entropy=True)
    noise = (T.rand(b, s, generator=T.Generator().manual_seed(6)) * 0.2 - 0.1).cuda()    # inside the clip
    kw = dict(kl_coef=0.1, entropy_coef=0.01, reduction="token")
    old, ref = f.logp - noise, f.logp + 2 * noise
    p = losses.policy_loss(f.logp, adv, old_logp=old, ref_logp=ref, entropy=f.entropy, mask=mask, **kw)
    d = losses.token_logprobs_backward(x, t, f.lse, p.dlogp, entropy=f.entropy, dentropy=p.dentropy)
    r = losses.policy_loss_logits(x, t, adv, old_logp=old, ref_logp=ref, mask=mask, **kw)
    assert int(r.tokens) == int(mask.sum()) == int(p.tokens)
    assert T.allclose(r.stats, p.stats, rtol=1e-5, atol=1e-7)
    assert (r.dlogits - d).norm() <= 1e-5 * d.norm()
    assert (r.dlogits[~mask] == 0).all()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("vocab", [24000, 24575, 33001, 50257, 64007, 65536, 80001, 98304, 110001, 128256, 151936, 155657])
def test_every_shape_of_a_row(losses, T, name, vocab):
    """Rows of each size that is held in registers, masked and partly banned, against the separate operators in FP32.

    Both have the same logits; what differs is the type that the gradient is rounded to (half a step relative to itself) and
    the two computations' own errors, each within slack(); values below the type's smallest step are off by half of one.
    """
    rows = 97
    g = T.Generator(device="cuda").manual_seed(vocab)
    x = (T.randn(rows, vocab, generator=g, device="cuda") * 2.5).to(getattr(T, name))
    x[:, vocab // 3:vocab // 3 + 40] = -math.inf
    t = T.randint(0, vocab // 3, (rows,), generator=g, device="cuda")
    t[5], t[6], t[7] = vocab - 1, 0, -1
    adv = T.randn(rows, generator=g, device="cuda")
    cu = T.arange(rows + 1, dtype=T.int32, device="cuda")
    x32 = x.float()
    f = losses.token_logprobs(x32, t, with_entropy=True)
    for ec in (0.0, 0.5):
        r = losses.policy_loss_logits(x, t, adv, cu_seqlens=cu, reduction="sum", entropy_coef=ec, with_entropy=True)
        dh = T.full_like(adv, -ec) if ec else None
        d = losses.token_logprobs_backward(x32, t, f.lse, -adv, entropy=f.entropy if ec else None, dentropy=dh)
        lp = (x32 - f.lse[:, None]).abs().nan_to_num(posinf=0.0)
        zmax = 16.0                                     # of 1.6e7 normal values times 2.5
        rel = 2 * U * (4 * zmax + 6 * lp + vocab / 256 + 40 + 8)
        p = T.exp(x32 - f.lse[:, None]) * (t >= 0)[:, None]
        size = adv.abs()[:, None] * p + ec * p * (lp + f.entropy[:, None] + 1)
        size[T.arange(rows).cuda()[t >= 0], t[t >= 0]] += adv.abs()[t >= 0]
        bound = d.abs() * (LO.EPS[name] * 1.01) + size * rel + LO.TINY[name]
        assert x32.isfinite().logical_not().sum() == rows * 40 and x32.nan_to_num(neginf=0.0).abs().max() <= zmax
        assert bool(((r.dlogits.float() - d).abs() <= bound).all()), "entropy_coef %g" % ec
        assert T.allclose(r.logp, f.logp, rtol=1e-5, atol=2e-5) and T.allclose(r.entropy, f.entropy, rtol=2e-5, atol=2e-5)


def test_gradient_of_the_logits_against_differences(losses, T):
    """Differences of the loss itself (in 64 bits) in some of the logits."""
    rows, vocab = 6, 37
    x, xh, t, th = make_logits(T, rows, vocab, "float32", 77)
    rng = np.random.default_rng(0)
    cu, seq = [0, 2, 6], LO.sequences(rows, [0, 2, 6])
    lp0 = LO.rows(xh, th, 0.9)[0]
    old, ref = (lp0 - rng.uniform(-0.1, 0.1, rows)).astype(np.float32), (lp0 + 0.2).astype(np.float32)
    adv = rng.normal(size=2).astype(np.float32)
    kw = dict(kl_coef=0.3, entropy_coef=0.2)

    def loss(z):
        logp, _, ent = LO.rows(z, th, 0.9)
        return LO.policy(logp, adv, seq, 2, np.ones(rows, bool), old=old, ref=ref, entropy=ent, **kw)[0][0]

    r = losses.policy_loss_logits(x, t, T.tensor(adv).cuda(), old_logp=T.tensor(old).cuda(), ref_logp=T.tensor(ref).cuda(),
                                  cu_seqlens=T.tensor(cu, dtype=T.int32).cuda(), temperature=0.9, **kw)
    got = host(r.dlogits)
    for i in range(rows):
        for j in list(rng.integers(0, vocab, 6)) + [th[i]]:
            step = np.zeros_like(xh)
            step[i, j] = 1e-5
            diff = (loss(xh + step) - loss(xh - step)) / 2e-5
            # central differences: h^2 times a third derivative of about 1, and FP64 cancellation over h
            assert abs(diff - got[i, j]) <= 1e-8 + 2e-6 * abs(diff) + 4e-7


def test_bad_target_in_a_batch(losses, T):
    x, _, t, _ = make_logits(T, 6, 100, "float16", 3)
    t[2] = 100
    r = losses.policy_loss_logits(x, t, T.ones(1).cuda(), cu_seqlens=T.tensor([0, 6], dtype=T.int32).cuda())
    bad = T.tensor([0, 0, 1, 0, 0, 0], dtype=T.bool).cuda()
    assert r.dlogits[bad].isnan().all() and r.dlogits[~bad].isfinite().all()
    assert r.logp[bad].isnan().all() and r.logp[~bad].isfinite().all() and r.stats[0].isnan()


# --- preference loss ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cu", [[0, 1, 2], [0, 0, 3], [0, 5, 5, 5, 5], [3, 40, 700, 1400, 1401],
                                [0] + list(np.cumsum([1 + (i * 53) % 301 for i in range(1200)])),
                                [0, 30000, 30001, 90000, 150000]], ids=lambda c: "%d-%d" % (len(c) - 1, c[-1]))
def test_preference_loss(losses, T, cu):
    tokens, pairs = cu[-1] + 2, (len(cu) - 1) // 2
    seq = LO.sequences(tokens, cu)
    cu_t = T.tensor(np.array(cu, np.int32)).cuda()
    for variant in range(4):
        rng = np.random.default_rng(variant + tokens)
        lp = -rng.exponential(1.0, tokens).astype(np.float32)
        ref = (lp + rng.normal(0, 0.3, tokens)).astype(np.float32) if variant != 1 else None
        mask = rng.random(tokens) < (0.7, 1.0, 0.5, 0.0)[variant]
        kw = dict(beta=(0.1, 2.0, 0.5, 0.1)[variant], margin=0.3 * variant, average=variant % 2 == 1, grad_scale=4.0)
        ls = (0.0, 0.1, 1.0, 0.0)[variant]
        lp_t, mask_t = T.tensor(lp).cuda(), T.tensor(mask).cuda()
        ref_t = T.tensor(ref).cuda() if ref is not None else None
        lp_t[~mask_t] = math.nan
        r = losses.preference_loss(lp_t, ref_logp=ref_t, mask=mask_t, cu_seqlens=cu_t, label_smoothing=ls, **kw)
        stats, rewards, dlogp = LO.preference(lp, seq, pairs, mask, ref=ref, smoothing=ls, **kw)
        # sums are in 64 bits: what is left is each result's own rounding
        check(r.rewards, rewards, np.abs(rewards) * 2 * U + 1e-12, "rewards")
        check(r.stats, stats, np.abs(stats) * 2 * U + 1e-12, "stats")
        check(r.dlogp, dlogp, np.abs(dlogp) * 2 * U + 1e-37, "dlogp")
        again = losses.preference_loss(lp_t, ref_logp=ref_t, mask=mask_t, cu_seqlens=cu_t, label_smoothing=ls, **kw)
        assert T.equal(again.dlogp, r.dlogp) and T.equal(again.stats, r.stats)


def test_preference_loss_far_apart(losses, T):
    """x of +-1e4: the loss grows linearly, the gradient stays at its limits."""
    lp = T.tensor([[0.0], [-1e4], [-1e4], [0.0]]).cuda()        # pair 0: 0 against -1e4, pair 1: -1e4 against 0
    r = losses.preference_loss(lp, beta=1.0)
    assert host(r.stats).tolist() == [5000.0, 0.5, 0.0, -5000.0, -5000.0]
    assert host(r.dlogp).reshape(-1).tolist() == [0.0, -0.5, 0.0, 0.5]
    with pytest.raises(ValueError, match="even"):
        losses.preference_loss(lp[:3].contiguous())


# --- empty input, refusals, streams, graphs ----------------------------------------------------------------------------------

def test_empty_input(losses, T):
    x = T.empty(0, 100, dtype=T.float16, device="cuda")
    t = T.empty(0, dtype=T.int64, device="cuda")
    r = losses.token_logprobs(x, t, with_entropy=True)
    assert r.logp.shape == (0,)
    assert losses.token_logprobs_backward(x, t, r.lse, r.logp).shape == (0, 100)
    cu = T.zeros(1, dtype=T.int32, device="cuda")
    none = T.empty(0, device="cuda")
    for out in (losses.policy_loss(none, none, cu_seqlens=cu), losses.policy_loss_logits(x, t, none, cu_seqlens=cu)):
        assert host(out.stats).tolist() == [0.0] * 6 and int(out.tokens) == 0
    assert host(losses.preference_loss(none, cu_seqlens=cu).stats).tolist() == [0.0] * 5


def test_python_refusals(losses, T):
    x, t = T.zeros(4, 10, device="cuda"), T.zeros(4, dtype=T.int64, device="cuda")
    adv, cu = T.zeros(2, device="cuda"), T.tensor([0, 1, 4], dtype=T.int32, device="cuda")
    bad = [lambda: losses.token_logprobs(x.double(), t), lambda: losses.token_logprobs(x, t.short()),
           lambda: losses.token_logprobs(x, t[:3]), lambda: losses.token_logprobs(x, t.cpu()),
           lambda: losses.token_logprobs(x[0], t[0]),
           lambda: losses.token_logprobs_backward(x, t, adv, adv),
           lambda: losses.token_logprobs_backward(x, t, x[:, 0].contiguous(), x[:, 1]),
           lambda: losses.token_logprobs_backward(x, t, x[:, 0].contiguous(), None),
           lambda: losses.token_logprobs_backward(x, t, x[:, 0].contiguous(), x[:, 0].contiguous(), out=x.half()),
           lambda: losses.policy_loss(x[:, 0].contiguous(), adv),
           lambda: losses.policy_loss(x[:, 0].contiguous(), adv, cu_seqlens=cu.long()),
           lambda: losses.policy_loss(x, adv, cu_seqlens=cu),
           lambda: losses.policy_loss(x[:, 0].contiguous(), adv, cu_seqlens=cu, reduction="mean"),
           lambda: losses.policy_loss(x[:, 0].contiguous(), adv, cu_seqlens=cu, mask=x[:, 0].contiguous()),
           lambda: losses.policy_loss(x[:, 0].contiguous(), adv, cu_seqlens=cu, entropy_coef=0.1),
           lambda: losses.preference_loss(x[:, 0].contiguous())]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail("call %d was not refused" % i)
    with pytest.raises(losses.B.RlxError):
        losses.token_logprobs(x, t, temperature=0.0)
    wide = T.zeros(4, 12, device="cuda")
    with pytest.raises(losses.B.RlxError):               # overlaps the logits in another layout
        losses.token_logprobs_backward(wide[:, :10], t, x[:, 0].contiguous(), x[:, 0].contiguous(),
                                       out=wide.as_strided((4, 10), (11, 1)))


@pytest.mark.parametrize("rows,vocab", [(3, 40000), (900, 2000)])
def test_other_streams_and_recorded_graphs(losses, T, rows, vocab):
    """A call on a side stream, and two recorded graphs of the whole chain that are replayed in turn on new inputs,
    with eager work of the same kind in between: always the eager bits."""
    x, _, t, _ = make_logits(T, rows, vocab, "bfloat16", 5)
    adv, cu = T.tensor([0.7, -0.4]).cuda(), T.tensor([0, rows // 2, rows], dtype=T.int32).cuda()
    mask = (T.rand(rows, generator=T.Generator().manual_seed(1)) < 0.8).cuda()
    ref = T.full((rows,), -3.0).cuda()
    kw = dict(mask=mask, cu_seqlens=cu)

    def chain(x):
        f = losses.token_logprobs(x, t, with_entropy=True)
        p = losses.policy_loss(f.logp, adv, ref_logp=ref, entropy=f.entropy, kl_coef=0.01, entropy_coef=0.01,
                               reduction="token", **kw)
        d = losses.token_logprobs_backward(x, t, f.lse, p.dlogp, entropy=f.entropy, dentropy=p.dentropy)
        q = losses.policy_loss_logits(x, t, adv, ref_logp=ref, kl_coef=0.01, **kw)
        w = losses.preference_loss(f.logp, ref_logp=ref, **kw)
        return [f.logp, f.lse, f.entropy, p.stats, p.dlogp, d, q.stats, q.dlogits, w.stats, w.dlogp]

    want = [o.clone() for o in chain(x)]
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        got = chain(x)
    T.cuda.current_stream().wait_stream(side)
    assert all(T.equal(a, b) for a, b in zip(got, want))
    held = [x.clone(), x.clone()]
    graphs, outs = [], []
    for k in range(2):
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            outs.append(chain(held[k]))
        graphs.append(g)
    for turn in range(4):
        new = [(x.float() * (1.0 + 0.1 * turn + 0.05 * k)).to(x.dtype) for k in range(2)]
        for k in range(2):
            held[k].copy_(new[k])
            graphs[k].replay()
        eager = [[o.clone() for o in chain(v)] for v in new]
        T.cuda.synchronize()
        for k in range(2):
            assert all(T.equal(a, b) for a, b in zip(outs[k], eager[k])), "replay %d of graph %d" % (turn, k)


def test_calls_at_once_on_two_streams(losses, T):
    """The same chain on two streams at the same time, large enough to overlap, each with other inputs: the bits of either
    one alone."""
    rows, vocab = 900, 9001
    inputs = [make_logits(T, rows, vocab, "float16", seed) for seed in (1, 2)]
    adv = T.tensor([0.5, -0.5, 1.0]).cuda()

    def chain(x, t):
        f = losses.token_logprobs(x, t, with_entropy=True)
        q = losses.policy_loss_logits(x.view(3, rows // 3, vocab), t.view(3, -1), adv, reduction="token")
        few = losses.policy_loss_logits(x[:40].reshape(4, -1), t[:4], adv[:1])
        p = losses.policy_loss(f.logp.view(3, -1), adv, entropy=f.entropy.view(3, -1), entropy_coef=0.1)
        w = losses.preference_loss(f.logp.view(4, -1))
        return [f.logp, f.lse, f.entropy, q.stats, q.dlogits, few.stats, few.dlogits, p.stats, p.dlogp, w.stats, w.dlogp]

    want = [[o.clone() for o in chain(x, t)] for x, _, t, _ in inputs]
    streams = [T.cuda.Stream(), T.cuda.Stream()]
    T.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (x, _, t, _) in zip(streams, inputs):
            with T.cuda.stream(s):
                got.append(chain(x, t))
        T.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(T.equal(u, v) for u, v in zip(a, b))


# --- the operators in the framework's own step ----------------------------------------------------------------------------

@pytest.mark.parametrize("fused", [False, True])
def test_policy_step(losses, L, host, O, T, fused):
    """host.policy_step on a one-layer model (an output projection): its step equals the same micro-batches done by
    hand (loss from the oracle, gradient products in FP32), clip and update included."""
    import test_gpu_losses as here
    hidden, vocab, rows, n_micro = 16, 257, 24, 3
    specs = [L.TensorSpec("lm_head", vocab * hidden, L.DTYPE_F32, L.NO_DECAY, hidden)]
    out = []
    g = T.Generator().manual_seed(0)
    w0 = T.randn(vocab, hidden, generator=g) * 0.3
    acts = [T.randn(rows, hidden, generator=g).cuda() for _ in range(n_micro)]
    targets = [T.randint(0, vocab, (rows,), generator=g).cuda() for _ in range(n_micro)]
    adv = [T.randn(3, generator=g).cuda() for _ in range(n_micro)]
    mask = (T.rand(rows, generator=g) < 0.7).cuda()
    cu = T.tensor([0, 7, 15, 24], dtype=T.int32).cuda()
    ref = [T.full((rows,), -5.0).cuda() for _ in range(n_micro)]

    st = host.ParamStore(specs, "cuda:0")
    st.param(0).copy_(w0.reshape(-1))
    opt = host.AdamWOptimizer(st, lr=1e-2)
    st.fill("g", 4, 0.0, 1.0)                          # stale gradients that the step must clear first

    def forward(k):
        return dict(logits=acts[k] @ st.param(0).view(vocab, hidden).t(), targets=targets[k], advantages=adv[k],
                    ref_logp=ref[k])

    def backward(k, dlogits):
        st.grad(0).view(vocab, hidden).add_(dlogits.t() @ acts[k])

    loss, norm, results = host.policy_step(opt, forward, backward, n_micro, 0.01, fused_clip=fused, mask=mask,
                                           cu_seqlens=cu, kl_coef=0.1)
    T.cuda.synchronize()
    # by hand, in 64 bits
    seq, counts = LO.sequences(rows, cu.tolist()), mask.cpu().numpy()
    w64, grad, total = w0.double().numpy(), np.zeros((vocab, hidden)), 0.0
    for k in range(n_micro):
        a, th = here.host(acts[k]), targets[k].cpu().numpy()
        z = a @ w64.T
        logp, lse, ent = LO.rows(z, th, 1.0)
        stats, n, dlogp, *_ = LO.policy(logp, here.host(adv[k]), seq, 3, counts, ref=here.host(ref[k]), kl_coef=0.1,
                                        norm=1.0 / n_micro)
        d, _ = LO.rows_grad(z, np.where(counts, th, -1), 1.0, lse, dlogp)
        grad += d.T @ a
        total += stats[0]
        assert int(results[k].tokens) == n and results[k].dlogits is None
    # FP32 products of 16 terms feed the softmax: 1e-5 relative covers them many times over
    assert abs(loss - total) <= 1e-5 * max(1.0, abs(total))
    assert abs(norm - np.linalg.norm(grad)) <= 1e-5 * np.linalg.norm(grad) and norm > 0.01
    scale = 0.01 / (norm + 1e-6)
    got = here.host(st.grad(0)).reshape(vocab, hidden)
    assert np.abs(got - grad * (1.0 if fused else scale)).max() <= 2e-5 * np.abs(grad).max()
    # the first AdamW step moves every weight by lr times the sign of its gradient, where that is well above eps
    moved = here.host(st.param(0)).reshape(vocab, hidden) - w64
    big = np.abs(grad) * scale > 1e-6
    assert big.any() and np.allclose(moved[big], -1e-2 * np.sign(grad[big]), rtol=2e-2)
    with pytest.raises(ValueError):
        host.policy_step(opt, forward, backward, 0, 1.0)
    with pytest.raises(ValueError):
        host.policy_step(opt, forward, backward, 1, 1.0, norm=0.5)
    # the same step on a stream of its own
    st2 = host.ParamStore(specs, "cuda:0")
    st2.param(0).copy_(w0.reshape(-1))
    opt2 = host.AdamWOptimizer(st2, lr=1e-2)
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    loss2, norm2, _ = host.policy_step(
        opt2, lambda k: dict(forward(k), logits=acts[k] @ st2.param(0).view(vocab, hidden).t()),
        lambda k, d: st2.grad(0).view(vocab, hidden).add_(d.t() @ acts[k]), n_micro, 0.01, fused_clip=fused,
        stream=side.cuda_stream, mask=mask, cu_seqlens=cu, kl_coef=0.1)
    T.cuda.synchronize()
    assert (loss2, norm2) == (loss, norm) and T.equal(st2.param(0), st.param(0))


def test_cpp_host_losses(torch_gpu):
    """tests/cpp/test_losses_host.cpp: the C++ wrappers and OptimStep::policy_step against loops in double."""
    import os
    import subprocess
    folder = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
    subprocess.run(["make", "-C", folder, "-s", "test_losses_host.bin"], check=True)
    res = subprocess.run([os.path.join(folder, "test_losses_host.bin")], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.count("[PASS]") == 6 and "[FAIL]" not in res.stdout
