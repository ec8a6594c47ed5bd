"""Refusals of the loss operators' C ABI and of their Python functions (no device needed), and their oracle against
finite differences and torch."""
import ctypes as C
import importlib
import os

import numpy as np
import pytest

import loss_oracle as LO

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000           # an aligned address that is never followed: every call here is refused on the host
Q = 0x900000000


@pytest.fixture(scope="module")
def losses(pkg):
    return importlib.import_module(pkg.__name__ + ".losses")


def logits(B, data=P, rows=4, vocab=100, row_stride=100, group_rows=0, group_stride=0, dtype=0, reserved=0):
    return B.Logits(data, rows, vocab, row_stride, group_rows, group_stride, dtype, reserved)


def logprob(B, x, targets=P, index=0, temp=1.0, logp=P, lse=P, ent=None, ws=P, nbytes=1 << 40):
    return B.load().rlx_token_logprob(C.byref(x), targets, index, temp, logp, lse, ent, ws, nbytes, None)


def test_struct_layouts(B, tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "rlx_adamw.h"\nint main(void){return !(sizeof(rlx_logits) == %d && sizeof(rlx_policy_args) '
                   '== %d && sizeof(rlx_policy_stats) == 32 && sizeof(rlx_preference_args) == %d && '
                   'sizeof(rlx_preference_stats) == 20);}\n'
                   % (C.sizeof(B.Logits), C.sizeof(B.PolicyArgs), C.sizeof(B.PreferenceArgs)))
    exe = tmp_path / "t"
    assert os.system("gcc -std=c99 -Wall -Werror -I%s/include -o %s %s" % (ROOT, exe, src)) == 0
    assert os.system(str(exe)) == 0


def test_logits_are_checked(B):
    bad = B.ERR_INVALID_ARG
    assert logprob(B, logits(B, rows=0, data=None)) == B.OK
    for kw in (dict(data=None), dict(rows=-1), dict(vocab=0), dict(row_stride=99), dict(row_stride=-100), dict(dtype=3),
               dict(reserved=1), dict(group_rows=-1), dict(group_rows=2, group_stride=150),
               dict(group_rows=2, group_stride=99, row_stride=300), dict(row_stride=1 << 61)):
        assert logprob(B, logits(B, **kw)) == bad, kw
    assert logprob(B, logits(B, data=P + 1)) == B.ERR_MISALIGNED
    assert logprob(B, logits(B, data=P + 2, dtype=1)) == B.ERR_MISALIGNED
    assert logprob(B, logits(B, vocab=(1 << 30) + 1, row_stride=1 << 31)) == B.ERR_TOO_LARGE
    assert logprob(B, logits(B, rows=1 << 31)) == B.ERR_TOO_LARGE
    assert B.load().rlx_token_logprob(None, P, 0, 1.0, P, P, None, None, 0, None) == bad
    x = logits(B)
    assert logprob(B, x, targets=None) == bad and logprob(B, x, index=2) == bad
    assert logprob(B, x, targets=P + 4, index=1) == B.ERR_MISALIGNED
    assert logprob(B, x, logp=None) == bad and logprob(B, x, lse=None) == bad
    assert logprob(B, x, ent=P + 2) == B.ERR_MISALIGNED
    for t in (0.0, -1.0, float("inf"), float("nan"), 1e-45):
        assert logprob(B, x, temp=t) == B.ERR_BAD_HYPER
    assert logprob(B, x, ws=P + 8) == B.ERR_MISALIGNED
    for lib_fn in (B.load().rlx_token_logprob_workspace,):
        assert lib_fn(C.byref(x)) >= 0 and lib_fn(C.byref(logits(B, vocab=0))) == -1


def backward(B, x, dx, **kw):
    a = dict(targets=P, index=0, temp=1.0, lse=P, ent=None, dlogp=P, dent=None)
    a.update(kw)
    return B.load().rlx_token_logprob_backward(C.byref(x), a["targets"], a["index"], a["temp"], a["lse"], a["ent"],
                                               a["dlogp"], a["dent"], C.byref(dx), None)


def test_gradient_memory_is_checked(B):
    x = logits(B)
    bad = B.ERR_INVALID_ARG
    for kw in (dict(rows=5), dict(vocab=99), dict(dtype=2), dict(data=None)):
        assert backward(B, x, logits(B, **{"data": Q, **kw})) == bad, kw
    assert backward(B, x, logits(B, row_stride=101)) == bad                  # the same start, other strides
    assert backward(B, x, logits(B, data=P + 200)) == bad                    # overlap
    assert backward(B, x, logits(B, data=P + 2 * 399)) == bad                # overlap by one element
    assert backward(B, x, logits(B, data=Q), lse=None) == bad
    assert backward(B, x, logits(B, data=Q), dlogp=None) == bad
    assert backward(B, x, logits(B, data=Q), ent=P) == bad
    assert backward(B, x, logits(B, data=Q), dent=P) == bad
    assert backward(B, x, logits(B, data=Q), dlogp=P + 1) == B.ERR_MISALIGNED
    assert backward(B, x, logits(B, data=Q), temp=0.0) == B.ERR_BAD_HYPER


def policy_args(B, **kw):
    a = dict(old_logp=P, ref_logp=P, advantages=P, entropy=None, mask=P, cu_seqlens=P, n_seqs=2, clip_low=0.2,
             clip_high=0.2, kl_coef=0.1, entropy_coef=0.0, norm=1.0, grad_scale=1.0, reduction=0,
             advantage_per_token=0)
    a.update(kw)
    return B.PolicyArgs(*[a[f[0]] for f in B.PolicyArgs._fields_])


def policy(B, args, logp=P, tokens=10, dlogp=P, dent=None, stats=P, ws=P, nbytes=1 << 40):
    return B.load().rlx_policy_loss(logp, tokens, C.byref(args) if args else None, dlogp, dent, stats, ws, nbytes, None)


REFUSED = [dict(advantages=None), dict(n_seqs=-1), dict(n_seqs=0), dict(cu_seqlens=None, n_seqs=3), dict(reduction=3),
           dict(reduction=-1)]
BAD_HYPER = [dict(clip_low=-0.1), dict(clip_low=1.1), dict(clip_high=-0.1), dict(kl_coef=float("nan")),
             dict(entropy_coef=float("inf")), dict(norm=float("nan")), dict(grad_scale=float("inf")),
             dict(clip_high=float("inf"))]


def test_policy_arguments_are_checked(B):
    bad = B.ERR_INVALID_ARG
    assert policy(B, None) == bad
    for kw in REFUSED:
        assert policy(B, policy_args(B, **kw)) == bad, kw
    for kw in BAD_HYPER:
        assert policy(B, policy_args(B, **kw)) == B.ERR_BAD_HYPER, kw
    ok = policy_args(B)
    many = 100000                                          # tokens of a batch that needs scratch memory
    for kw in (dict(logp=None), dict(dlogp=None), dict(stats=None), dict(tokens=-1), dict(tokens=many, nbytes=8),
               dict(tokens=many, ws=None)):
        assert policy(B, ok, **kw) == bad, kw
    assert policy(B, policy_args(B, entropy_coef=0.1), dent=P) == bad            # needs entropy
    assert policy(B, policy_args(B, entropy_coef=0.1, entropy=P)) == bad         # needs dentropy
    for kw in (dict(logp=P + 1), dict(dlogp=P + 2), dict(stats=P + 4), dict(ws=P + 4)):
        assert policy(B, ok, **kw) == B.ERR_MISALIGNED, kw
    for kw in (dict(old_logp=P + 1), dict(cu_seqlens=P + 2), dict(advantages=P + 3), dict(entropy=P + 2)):
        assert policy(B, policy_args(B, **kw)) == B.ERR_MISALIGNED, kw
    assert policy(B, ok, tokens=1 << 31) == B.ERR_TOO_LARGE
    lib = B.load()
    assert lib.rlx_policy_loss_workspace(-1, 1) == -1 and lib.rlx_policy_loss_workspace(1, -1) == -1
    assert lib.rlx_policy_loss_workspace(many, 3) > 8


def fused(B, args, x, dx, targets=P, index=0, temp=1.0, logp=P, ent=None, stats=P, ws=P, nbytes=1 << 40):
    return B.load().rlx_policy_loss_logits(C.byref(x), targets, index, temp, C.byref(args), logp, ent, C.byref(dx), stats,
                                           ws, nbytes, None)


def test_policy_logits_arguments_are_checked(B):
    bad = B.ERR_INVALID_ARG
    x, dx, ok = logits(B), logits(B, data=Q), policy_args(B)
    for kw in REFUSED:
        assert fused(B, policy_args(B, **kw), x, dx) == bad, kw
    for kw in BAD_HYPER:
        assert fused(B, policy_args(B, **kw), x, dx) == B.ERR_BAD_HYPER, kw
    assert fused(B, policy_args(B, entropy=P), x, dx) == bad
    assert fused(B, ok, x, logits(B, data=P + 200)) == bad
    assert fused(B, ok, x, dx, targets=None) == bad and fused(B, ok, x, dx, index=7) == bad
    assert fused(B, ok, x, dx, logp=None) == bad and fused(B, ok, x, dx, stats=None) == bad
    assert fused(B, ok, x, dx, nbytes=8) == bad and fused(B, ok, x, dx, ws=None) == bad
    assert fused(B, ok, x, dx, temp=-1.0) == B.ERR_BAD_HYPER
    assert fused(B, ok, x, dx, stats=P + 4) == B.ERR_MISALIGNED
    assert B.load().rlx_policy_loss_logits_workspace(C.byref(logits(B, vocab=0)), 1) == -1
    assert B.load().rlx_policy_loss_logits_workspace(C.byref(x), -1) == -1


def test_preference_arguments_are_checked(B):
    lib, bad = B.load(), B.ERR_INVALID_ARG

    def call(tokens=8, logp=P, dlogp=P, rewards=P, stats=P, ws=P, nbytes=1 << 40, **kw):
        a = dict(ref_logp=P, mask=P, cu_seqlens=P, n_pairs=2, beta=0.1, label_smoothing=0.0, margin=0.0, grad_scale=1.0,
                 average=0, reserved=0)
        a.update(kw)
        args = B.PreferenceArgs(*[a[f[0]] for f in B.PreferenceArgs._fields_])
        return lib.rlx_preference_loss(logp, tokens, C.byref(args), dlogp, rewards, stats, ws, nbytes, None)

    for kw in (dict(tokens=-1), dict(logp=None), dict(dlogp=None), dict(stats=None), dict(tokens=100000, ws=None),
               dict(tokens=100000, nbytes=8), dict(n_pairs=-1), dict(n_pairs=0), dict(reserved=1), dict(cu_seqlens=None, tokens=7)):
        assert call(**kw) == bad, kw
    for kw in (dict(beta=float("nan")), dict(label_smoothing=-0.1), dict(label_smoothing=1.5), dict(margin=float("inf")),
               dict(grad_scale=float("nan"))):
        assert call(**kw) == B.ERR_BAD_HYPER, kw
    for kw in (dict(logp=P + 1), dict(dlogp=P + 1), dict(rewards=P + 2), dict(stats=P + 2), dict(ws=P + 4),
               dict(ref_logp=P + 1), dict(cu_seqlens=P + 1)):
        assert call(**kw) == B.ERR_MISALIGNED, kw
    assert call(n_pairs=1 << 30) == B.ERR_TOO_LARGE
    assert call(n_pairs=(1 << 22) + 1, nbytes=1 << 40) == B.ERR_TOO_LARGE      # more than one launch holds
    assert B.load().rlx_preference_loss_workspace(0, (1 << 22) + 1) == -1
    assert lib.rlx_preference_loss(P, 8, None, P, P, P, P, 1 << 40, None) == bad
    assert lib.rlx_preference_loss_workspace(-1, 1) == -1 and lib.rlx_preference_loss_workspace(100000, 4) > 8


def test_python_functions_refuse_host_tensors(losses):
    import torch
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        losses.token_logprobs(x, t)
    with pytest.raises(ValueError, match="GPU"):
        losses.policy_loss(torch.zeros(4), torch.zeros(1))
    with pytest.raises(ValueError, match="GPU"):
        losses.preference_loss(torch.zeros(2, 4))


# --- the oracle itself ------------------------------------------------------------------------------------------------

def test_oracle_rows_against_torch():
    import torch
    rng = np.random.default_rng(1)
    x = rng.normal(0, 3, (7, 33))
    t = rng.integers(0, 33, 7)
    logp, lse, ent = LO.rows(x, t, 0.8)
    z = torch.tensor(x / 0.8, requires_grad=True)
    lq = torch.log_softmax(z, 1)
    want = lq[torch.arange(7), torch.tensor(t)]
    h = torch.distributions.Categorical(logits=z).entropy()
    assert np.allclose(logp, want.detach(), atol=1e-12) and np.allclose(ent, h.detach(), atol=1e-12)
    assert np.allclose(lse, torch.logsumexp(z, 1).detach(), atol=1e-12)
    g, c = rng.normal(size=7), rng.normal(size=7)
    (want * torch.tensor(g)).sum().add((h * torch.tensor(c)).sum()).backward()
    d, _ = LO.rows_grad(x, t, 0.8, lse, g, ent, c)
    assert np.allclose(d, z.grad.numpy() / 0.8, atol=1e-12)


@pytest.mark.parametrize("reduction", ["sequence", "token", "sum"])
def test_oracle_policy_gradient_against_differences(reduction):
    rng = np.random.default_rng(2)
    t, cu = 24, [2, 9, 9, 20]
    seq = LO.sequences(t, cu)
    counts = rng.random(t) < 0.7
    lp, old, ref = -rng.random(t) * 3, None, None
    old, ref = lp - rng.normal(0, 0.2, t), lp + rng.normal(0, 0.3, t)
    adv, h = rng.normal(size=3), rng.random(t)
    kw = dict(old=old, ref=ref, clip_high=0.3, kl_coef=0.25, entropy_coef=0.5, reduction=reduction, norm=0.5)

    def loss(lp, h):
        return LO.policy(lp, adv, seq, 3, counts, entropy=h, **kw)[0][0]

    _, n, dlogp, dent, *_ = LO.policy(lp, adv, seq, 3, counts, entropy=h, **kw)
    assert n == (counts & (seq >= 0)).sum()
    e = 1e-6
    for i in range(t):
        step = np.zeros(t)
        step[i] = e
        assert abs((loss(lp + step, h) - loss(lp - step, h)) / (2 * e) - dlogp[i]) < 1e-7
        assert abs((loss(lp, h + step) - loss(lp, h - step)) / (2 * e) - dent[i]) < 1e-7


@pytest.mark.parametrize("average", [False, True])
def test_oracle_preference_gradient_against_differences(average):
    rng = np.random.default_rng(3)
    t, cu = 30, [1, 6, 6, 15, 28]
    seq = LO.sequences(t, cu)
    counts = rng.random(t) < 0.8
    lp, ref = -rng.random(t), -rng.random(t)
    kw = dict(ref=ref, beta=0.7, smoothing=0.1, margin=0.2, average=average)
    dlogp = LO.preference(lp, seq, 2, counts, **kw)[2]
    for i in range(t):
        step = np.zeros(t)
        step[i] = 1e-6
        diff = (LO.preference(lp + step, seq, 2, counts, **kw)[0][0] - LO.preference(lp - step, seq, 2, counts, **kw)[0][0])
        assert abs(diff / 2e-6 - dlogp[i]) < 1e-8


def test_backward_with_log_probabilities_is_checked(B):
    """The form that also takes logp refuses what the other one does, and a misaligned logp."""
    x, dx = logits(B), logits(B, data=Q)

    def call(logp=P, targets=P, index=0, temp=1.0, lse=P, ent=None, dlogp=P, dent=None, x=x, dx=dx):
        return B.load().rlx_token_logprob_backward_logp(C.byref(x), targets, index, temp, lse, ent, logp, dlogp, dent,
                                                        C.byref(dx), None)

    assert call(x=logits(B, rows=0, data=None), dx=logits(B, rows=0, data=None)) == B.OK
    for kw in (dict(lse=None), dict(dlogp=None), dict(ent=P), dict(dent=P), dict(targets=None), dict(index=2),
               dict(dx=logits(B, data=P + 200))):
        assert call(**kw) == B.ERR_INVALID_ARG, kw
    assert call(logp=P + 2) == B.ERR_MISALIGNED and call(temp=0.0) == B.ERR_BAD_HYPER


@pytest.mark.parametrize("side", [None, 77])
def test_policy_step_works_on_the_optimizers_device(pkg, losses, monkeypatch, side):
    """Every part of a step runs with the optimizer's device as the current one, and on that device's stream."""
    import torch
    host = importlib.import_module(pkg.__name__ + ".host")
    now, seen = ["cuda:0"], []

    class Device:
        def __init__(self, device):
            self.device = str(device)

        def __enter__(self):
            now.append(self.device)

        def __exit__(self, *exc):
            now.pop()

    class Stream(Device):
        def __enter__(self):
            now.append(self.device + " 77")

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda stream, device: Stream(device))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
    monkeypatch.setattr(host, "_stream", lambda: 77 if now[-1].endswith(" 77") else now[-1])
    monkeypatch.setattr(host, "training_step", lambda *a, **kw: seen.append(("step", now[-1])) or 2.0)

    def loss(**kw):
        seen.append(("loss", now[-1]))
        return losses.PolicyLossLogits(torch.ones(6), torch.tensor(1), None, None, kw["logits"])

    monkeypatch.setattr(losses, "policy_loss_logits", loss)

    class Store:
        device = torch.device("cuda:1")

        def zero_grads(self, st):
            seen.append(("clear on %s" % st, now[-1]))

    class Optimizer:
        store = Store()

    def forward(k):
        seen.append(("forward", now[-1]))
        return dict(logits=torch.zeros(1))

    r = host.policy_step(Optimizer(), forward, lambda k, d: seen.append(("backward", now[-1])), 2, 1.0, stream=side)
    assert r[:2] == (2.0, 2.0) and now == ["cuda:0"]
    where = "cuda:1" if side is None else "cuda:1 77"
    assert seen == [("clear on %s" % ("cuda:1" if side is None else 77), where)] + [
        (what, where) for what in ("forward", "loss", "backward") * 2] + [("step", where)]
