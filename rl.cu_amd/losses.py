"""Loss operators on torch-allocated device memory: token log-probabilities of logits and their gradient, the clipped
policy loss with a KL term (from log-probabilities or straight from the logits) and the preference loss.

They stand where the reference's trainers launch their loss kernels (include/training/GRPO_trainer.h:452-517 for the
policy loss), in front of the backward pass and of host.training_step; host.policy_step runs them in that order.
torch is used for device memory and streams only; all arithmetic happens in librlx_adamw.so, whose header states the
formulas and what is done with masked, empty and out-of-range input.

Arguments are device tensors of one GPU; work goes to that GPU's current stream and nothing is waited for.  Every call
takes its scratch memory and its outputs from torch's allocator, so calls on several streams and calls recorded
into graphs never share any.  Gradients are explicit: nothing here takes part in torch's autograd.  It is told of tensors that
are written over, though: if an operation kept the logits for its own backward pass (a tanh does), out=logits makes
that pass raise torch's error, and the gradient has to go elsewhere.  Per-token tensors are contiguous; logits may be any
view whose last dimension is contiguous and whose other dimensions step through memory in at most two strides
(logits[:, :-1] of a padded batch).
"""
import ctypes as C
from collections import namedtuple

import torch

from . import binding as B

TokenLogprobs = namedtuple("TokenLogprobs", "logp lse entropy")
# stats: float32 [loss, policy, kl, entropy, clip_fraction, ratio]; tokens: int64 scalar, how many count
PolicyLoss = namedtuple("PolicyLoss", "stats tokens dlogp dentropy")
PolicyLossLogits = namedtuple("PolicyLossLogits", "stats tokens logp entropy dlogits")
# stats: float32 [loss, accuracy, reward_margin, chosen_reward, rejected_reward]; rewards: float32 [2 * pairs]
PreferenceLoss = namedtuple("PreferenceLoss", "stats rewards dlogp")

_DTYPES = {torch.float16: B.DTYPE_F16, torch.float32: B.DTYPE_F32, torch.bfloat16: B.DTYPE_BF16}
_REDUCTIONS = {"sequence": B.LOSS_SEQUENCE_MEAN, "token": B.LOSS_TOKEN_MEAN, "sum": B.LOSS_SUM}


# handle of a GPU's current stream; torch's own short cut where it has one (the public way costs 2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class _Here:
    """Stands for torch.cuda.device(...) where that device is the current one already."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return None


_HERE = _Here()


def _on(device):
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _on_gpu(name, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a tensor on a GPU" % name)
    return t.device


def _ptr(name, t, device, dtype, shape):
    """Address of a contiguous tensor of the given type and shape; None for None."""
    if t is None:
        return None
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous():
        return t.data_ptr()
    if _on_gpu(name, t) != device:
        raise ValueError("%s is on %s, the other tensors on %s" % (name, t.device, device))
    if t.dtype != dtype:
        raise ValueError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have the shape %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    raise ValueError("%s must be contiguous" % name)


def _logits(name, x):
    """The rows of a [..., vocab] tensor as the library takes them."""
    _on_gpu(name, x)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError("%s must be float16, bfloat16 or float32, not %s" % (name, x.dtype))
    shape, strides = x.shape, x.stride()
    if len(shape) < 2 or shape[-1] < 1:
        raise ValueError("%s must have the shape [..., vocab]" % name)
    vocab = shape[-1]
    if vocab > 1 and strides[-1] != 1:
        raise ValueError("the last dimension of %s must be contiguous" % name)
    if len(shape) == 2:
        rows = shape[0]
        return B.Logits(x.data_ptr(), rows, vocab, strides[0] if rows > 1 else vocab, 0, 0, dtype, 0)
    # leading dimensions from the last one outwards, merged where one continues the other
    dims, rows = [], 1
    for n, step in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        rows *= n
        if n == 1:
            continue
        if dims and step == dims[-1][0] * dims[-1][1]:
            dims[-1][0] *= n
        else:
            dims.append([n, step])
    if rows == 0 or not dims:
        return B.Logits(x.data_ptr(), rows, vocab, vocab, 0, 0, dtype, 0)
    if len(dims) > 2:
        raise ValueError("the rows of %s lie in more than two strides: make it contiguous" % name)
    if len(dims) == 1:
        return B.Logits(x.data_ptr(), rows, vocab, dims[0][1], 0, 0, dtype, 0)
    return B.Logits(x.data_ptr(), rows, vocab, dims[0][1], dims[0][0], dims[1][1], dtype, 0)


def _targets(targets, device, shape):
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64):
        raise ValueError("targets must be an int32 or int64 tensor")
    return (_ptr("targets", targets, device, targets.dtype, shape),
            B.INDEX_I64 if targets.dtype == torch.int64 else B.INDEX_I32)


# tells autograd that a tensor's values have changed
_changed = torch.autograd.graph.increment_version


def _gradient(logits, x, out):
    """The gradient's tensor (a new one unless given) and its rows; x: those of the logits."""
    if out is logits:
        return out, x
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the shape, type and device of logits")
    return out, _logits("out", out)


def _workspace(nbytes, device, where):
    """(tensor to keep alive, address) of scratch memory."""
    if nbytes <= 0:
        if nbytes < 0:
            raise B.RlxError(B.ERR_INVALID_ARG, where)
        return None, None
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr()


def _address(t):
    return None if t is None else t.data_ptr()


def _floats(like):
    """A contiguous FP32 tensor in the shape of a contiguous per-token tensor."""
    return torch.empty_like(like, dtype=torch.float32)


def _batch(shape, device, mask, cu_seqlens):
    """Mask and offset addresses and the number of sequences of per-token tensors of this shape: packed tokens with
    offsets, or one sequence per row of a padded batch."""
    mask_ptr = None
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError("mask must be bool or uint8, not %s" % mask.dtype)
        mask_ptr = _ptr("mask", mask, device, mask.dtype, shape)
    if cu_seqlens is None:
        if len(shape) > 2:
            raise ValueError("per-token tensors must be [tokens] or [sequences, length]")
        return mask_ptr, None, (shape[0] if len(shape) == 2 else 1)
    if len(shape) != 1:
        raise ValueError("cu_seqlens goes with packed tokens: per-token tensors must be [tokens]")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be [sequences + 1]")
    return mask_ptr, _ptr("cu_seqlens", cu_seqlens, device, torch.int32, cu_seqlens.shape), cu_seqlens.numel() - 1


def token_logprobs(logits, targets, temperature=1.0, with_entropy=False):
    """Log-probability of targets[...] under softmax(logits / temperature), the log-sum-exp and, if asked, the
    entropy of every row.  Rows with a negative target are ignored (outputs 0)."""
    x = _logits("logits", logits)
    device, shape = logits.device, logits.shape[:-1]
    target_ptr, index_type = _targets(targets, device, shape)
    lib = B.load()
    with _on(device):
        logp, lse, entropy = _floats(targets), _floats(targets), _floats(targets) if with_entropy else None
        nbytes = lib.rlx_token_logprob_workspace(C.byref(x))
        ws, ws_ptr = _workspace(nbytes, device, "rlx_token_logprob")
        B.check(lib.rlx_token_logprob(C.byref(x), target_ptr, index_type, temperature, logp.data_ptr(),
                                      lse.data_ptr(), _address(entropy), ws_ptr, nbytes, _raw_stream(device.index)),
                "rlx_token_logprob")
    return TokenLogprobs(logp, lse, entropy)


def token_logprobs_backward(logits, targets, lse, dlogp, temperature=1.0, entropy=None, dentropy=None, out=None,
                            logp=None):
    """Gradient of the logits from the gradients of token_logprobs' logp and (with its entropy) entropy.
    out=logits writes it over the logits.  With token_logprobs' logp the gradients of likely targets keep the relative
    precision of 1 - p; an lse alone leaves them off by a few times 2^-24 |lse| / (1 - p) of themselves."""
    x = _logits("logits", logits)
    device, shape = logits.device, logits.shape[:-1]
    target_ptr, index_type = _targets(targets, device, shape)
    if (entropy is None) != (dentropy is None):
        raise ValueError("entropy and dentropy go together")
    f32 = torch.float32
    lse_p, dlogp_p = _ptr("lse", lse, device, f32, shape), _ptr("dlogp", dlogp, device, f32, shape)
    ent_p, dent_p = _ptr("entropy", entropy, device, f32, shape), _ptr("dentropy", dentropy, device, f32, shape)
    logp_p = _ptr("logp", logp, device, f32, shape)
    if lse_p is None or dlogp_p is None:
        raise ValueError("lse and dlogp are needed")
    given = out
    with _on(device):
        out, dx = _gradient(logits, x, out)
        B.check(B.load().rlx_token_logprob_backward_logp(C.byref(x), target_ptr, index_type, temperature, lse_p, ent_p,
                                                         logp_p, dlogp_p, dent_p, C.byref(dx),
                                                         _raw_stream(device.index)), "rlx_token_logprob_backward")
    if given is not None:
        _changed(given)
    return out


def _policy_args(shape, device, advantages, old_logp, ref_logp, entropy, mask, cu_seqlens, clip_low, clip_high,
                 kl_coef, entropy_coef, reduction, norm, grad_scale):
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'sequence', 'token' or 'sum'")
    f32 = torch.float32
    mask_p, cu_p, n_seqs = _batch(shape, device, mask, cu_seqlens)
    _on_gpu("advantages", advantages)
    per_sequence = advantages.dim() == 1 and advantages.numel() == n_seqs
    adv_p = _ptr("advantages", advantages, device, f32, advantages.shape if per_sequence else shape)
    return B.PolicyArgs(_ptr("old_logp", old_logp, device, f32, shape), _ptr("ref_logp", ref_logp, device, f32, shape),
                        adv_p, _ptr("entropy", entropy, device, f32, shape), mask_p, cu_p, n_seqs, clip_low, clip_high,
                        kl_coef, entropy_coef, norm, grad_scale, _REDUCTIONS[reduction], 0 if per_sequence else 1)


def _policy_memory(nbytes, device, where):
    """(scratch tensor to keep alive, address of an rlx_policy_stats, its parts, address of scratch memory).  The statistics live
    on, so they have an allocation of their own (1 us more than in one with the scratch memory, which they would hold)."""
    scratch, scratch_ptr = _workspace(nbytes, device, where)
    buf = torch.empty(4, dtype=torch.int64, device=device)
    return scratch, buf.data_ptr(), buf.view(torch.float32)[:6], buf[3], scratch_ptr


def policy_loss(logp, advantages, old_logp=None, ref_logp=None, entropy=None, mask=None, cu_seqlens=None,
                clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, reduction="sequence", norm=1.0,
                grad_scale=1.0):
    """Clipped policy loss with a KL term over log-probabilities, its statistics and its gradients.
    Tokens are packed ([tokens] with cu_seqlens, without them one sequence) or padded ([sequences, length]).  advantages:
    [sequences] (as many as sequences means one each), or one per token in logp's shape.  entropy is needed if
    entropy_coef is not 0; dentropy is its gradient then (else None)."""
    device, shape = _on_gpu("logp", logp), logp.shape
    if entropy_coef != 0.0 and entropy is None:
        raise ValueError("entropy_coef needs entropy")
    args = _policy_args(shape, device, advantages, old_logp, ref_logp, entropy, mask, cu_seqlens, clip_low, clip_high,
                        kl_coef, entropy_coef, reduction, norm, grad_scale)
    logp_p = _ptr("logp", logp, device, torch.float32, shape)
    tokens = logp.numel()
    lib = B.load()
    with _on(device):
        dlogp, dentropy = _floats(logp), _floats(logp) if entropy_coef != 0.0 else None
        nbytes = lib.rlx_policy_loss_workspace(tokens, args.n_seqs)
        scratch, stats_ptr, stats, count, ws_ptr = _policy_memory(nbytes, device, "rlx_policy_loss")
        B.check(lib.rlx_policy_loss(logp_p, tokens, C.byref(args), dlogp.data_ptr(), _address(dentropy),
                                    stats_ptr, ws_ptr, nbytes, _raw_stream(device.index)), "rlx_policy_loss")
    return PolicyLoss(stats, count, dlogp, dentropy)


def policy_loss_logits(logits, targets, advantages, old_logp=None, ref_logp=None, mask=None, cu_seqlens=None,
                       temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0,
                       reduction="sequence", norm=1.0, grad_scale=1.0, with_entropy=False, out=None):
    """policy_loss from the logits: loss, log-probabilities and the gradient of the logits in one call.  out=logits
    writes the gradient over the logits.  grad_scale multiplies the gradient only (16-bit gradients of a mean over
    thousands of tokens would fall below their range)."""
    x = _logits("logits", logits)
    device, shape = logits.device, logits.shape[:-1]
    target_ptr, index_type = _targets(targets, device, shape)
    args = _policy_args(shape, device, advantages, old_logp, ref_logp, None, mask, cu_seqlens, clip_low, clip_high,
                        kl_coef, entropy_coef, reduction, norm, grad_scale)
    lib, given = B.load(), out
    with _on(device):
        logp, entropy = _floats(targets), _floats(targets) if with_entropy else None
        out, dx = _gradient(logits, x, out)
        nbytes = lib.rlx_policy_loss_logits_workspace(C.byref(x), args.n_seqs)
        scratch, stats_ptr, stats, count, ws_ptr = _policy_memory(nbytes, device, "rlx_policy_loss_logits")
        B.check(lib.rlx_policy_loss_logits(C.byref(x), target_ptr, index_type, temperature, C.byref(args),
                                           logp.data_ptr(), _address(entropy), C.byref(dx), stats_ptr,
                                           ws_ptr, nbytes, _raw_stream(device.index)), "rlx_policy_loss_logits")
    if given is not None:
        _changed(given)
    return PolicyLossLogits(stats, count, logp, entropy, out)


def preference_loss(logp, ref_logp=None, mask=None, cu_seqlens=None, beta=0.1, label_smoothing=0.0, margin=0.0,
                    average=False, grad_scale=1.0):
    """Preference loss over pairs: the first half of the sequences are the chosen answers, the second half the
    rejected ones in the same order.  Tokens packed or padded as in policy_loss."""
    device, shape = _on_gpu("logp", logp), logp.shape
    mask_p, cu_p, n_seqs = _batch(shape, device, mask, cu_seqlens)
    if n_seqs % 2:
        raise ValueError("preference_loss needs an even number of sequences (chosen, then rejected), not %d" % n_seqs)
    f32 = torch.float32
    args = B.PreferenceArgs(_ptr("ref_logp", ref_logp, device, f32, shape), mask_p, cu_p, n_seqs // 2, beta,
                            label_smoothing, margin, grad_scale, 1 if average else 0, 0)
    logp_p = _ptr("logp", logp, device, f32, shape)
    tokens = logp.numel()
    lib = B.load()
    with _on(device):
        dlogp = _floats(logp)
        rewards = torch.empty(n_seqs, dtype=f32, device=device)
        stats = torch.empty(5, dtype=f32, device=device)
        nbytes = lib.rlx_preference_loss_workspace(tokens, args.n_pairs)
        ws, ws_ptr = _workspace(nbytes, device, "rlx_preference_loss")
        B.check(lib.rlx_preference_loss(logp_p, tokens, C.byref(args), dlogp.data_ptr(), rewards.data_ptr(),
                                        stats.data_ptr(), ws_ptr, nbytes, _raw_stream(device.index)),
                "rlx_preference_loss")
    return PreferenceLoss(stats, rewards, dlogp)
