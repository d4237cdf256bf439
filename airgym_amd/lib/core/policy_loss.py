"""Clipped policy loss with a KL term over rows of logits (csrc/policy_loss.hip): what `fused_ppo_loss` (fused_loss.py) is to a
Gaussian head, for a policy that answers with a choice - a discrete head, a token of a vocabulary.

    lp = log softmax(logits)[action]    r = exp(lp - old_logp)    d = ref_logp - lp
    row = max(-A r, -A clip(r, 1 - e_clip, 1 + e_clip)) + kl_coef (exp(d) - d - 1) - entropy_coef H

averaged over the rows that `mask` counts.  exp(d) - d - 1 is the non-negative estimate of KL(policy || reference) from the action
taken.  One pass writes the loss and its gradient: a forward under autograd already holds d loss / d logits, the backward only scales
it (by nothing at all if the loss is the graph's root; bfloat16 gradients are rounded a second time by any factor that is no power of two).
float16 holds neither the gradients of a mean over many rows nor those of a single row with a large ratio: for such logits the forward
keeps a copy of the logits, and the backward forms the gradient in its place, together with whatever the loss was scaled by."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from airgym_amd import _native as N
from airgym_amd.lib.core.native_call import activation, flags_of, on_device_of, ptr, shape_error, stream_of, wants_gradient

STATS = ("policy_loss", "kl", "entropy", "old_kl", "clip_frac", "rows")
_ARGS = ctypes.sizeof(N.AgTokenLossArgs)
_KEPT = 4 * N.AG_TOKEN_KEPT_ROW_FLOATS


def _launch(logits, actions, old_logp, advantages, ref_logp, mask, coefs, want_grad):
    lib = N.load()
    dev = logits.device
    loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(6, dtype=torch.float32, device=dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
    logits, r0, r1, v, s0, s1 = _table(logits)
    n = lib.ag_token_policy_loss_workspace_bytes(r0 * r1, v)
    keep = r0 * r1 * _KEPT if want_grad and logits.dtype == torch.float16 else 0
    ws = torch.empty(keep + n, dtype=torch.uint8, device=dev)         # the rows that are kept first
    at = ws.data_ptr()
    a = N.AgTokenLossArgs(_ARGS, N.AG_DTYPES[logits.dtype], v, r0, r1, s0, s1, logits.data_ptr(), actions.data_ptr(),
                          old_logp.data_ptr(), advantages.data_ptr(), ptr(ref_logp), ptr(mask), *coefs, loss.data_ptr(),
                          stats.data_ptr(), ptr(grad), at + keep, n, at if keep else None)
    with on_device_of(logits):
        N.check(lib.ag_token_policy_loss(ctypes.byref(a), stream_of(logits)), "ag_token_policy_loss")
    return loss, stats, grad, ws if keep else None


class _TokenPolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantages, ref_logp, mask, coefs, train):
        loss, stats, grad, kept = _launch(logits, actions, old_logp, advantages, ref_logp, mask, coefs, train)
        ctx.save_for_backward(logits, actions, old_logp, advantages, ref_logp, mask)
        ctx.coefs, ctx.grad, ctx.kept = coefs, grad, kept
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        if dloss is None:
            return (None,) * 8
        # the gradient is handed over, not kept: autograd may go on to add to it in place.  A second pass over a retained graph forms
        # it again.
        grad, kept, ctx.grad, ctx.kept = ctx.grad, ctx.kept, None, None
        if grad is None:
            _, _, grad, kept = _launch(*ctx.saved_tensors, ctx.coefs, True)
        lib, dtype = N.load(), N.AG_DTYPES[grad.dtype]
        with on_device_of(grad):
            if kept is None:
                N.check(lib.ag_scale_by(grad.data_ptr(), grad.numel(), dtype, dloss.data_ptr(), stream_of(grad)), "ag_scale_by")
            else:
                N.check(lib.ag_token_policy_grad(grad.data_ptr(), kept.data_ptr(), grad.numel() // grad.shape[-1], grad.shape[-1], dtype,
                                                 dloss.data_ptr(), stream_of(grad)), "ag_token_policy_grad")
        return (grad,) + (None,) * 7


def _rows(logits, actions):
    """logits with dense rows, their leading shape and the actions as dense int64."""
    if not isinstance(logits, torch.Tensor) or logits.dim() < 2 or logits.shape[-1] < 1:
        raise shape_error("logits", logits, "[..., V]")
    lead = logits.shape[:-1]
    logits = activation("logits", logits, logits.shape)
    if not isinstance(actions, torch.Tensor) or actions.dtype != torch.int64 or actions.shape != lead or actions.device != logits.device:
        raise shape_error("actions", actions, f"int64 {list(lead)} on {logits.device}")
    return logits, lead, actions.contiguous()


def _table(logits):
    """logits [..., V] as R0 x R1 rows: a tensor that holds them, R0, R1, V and the two strides."""
    if logits.dim() == 2:
        (r, v), (s, _) = logits.shape, logits.stride()
        return logits, 1, r, v, 0, s
    if logits.dim() > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
    return logits, *logits.shape, *logits.stride()[:2]


def _per_row(name, t, lead, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != lead or t.device != device:
        raise shape_error(name, t, f"float32 {list(lead)} on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: the loss has gradients for the logits only; detach it")
    return t.contiguous()


def policy_loss(logits, actions, old_logp, advantages, *, ref_logp=None, mask=None, e_clip=0.2, kl_coef=0.0, entropy_coef=0.0):
    """logits [..., V] (float32, bfloat16 or float16), actions int64 [...], old_logp, advantages and ref_logp float32 [...], mask bool
    or uint8 [...] (None: every row counts) -> (loss, stats), float32: the loss to call backward() on and
    [policy loss, KL term, entropy, KL of the old policy, fraction of clipped rows, rows counted], each a mean over the rows counted.

    Rows that do not count are not read: whatever their logits, actions and numbers are, they add nothing and get a gradient of zero.
    If no row counts, loss, statistics and gradients are zero.  Logits of -inf are choices that are not available; a row that counts and
    has no other, or an action outside [0, V), gives NaN.  A kl_coef or an advantage of exactly zero takes its term out of loss and
    gradient, also where the term is infinite."""
    logits, lead, actions = _rows(logits, actions)
    dev = logits.device
    old_logp, advantages = _per_row("old_logp", old_logp, lead, dev), _per_row("advantages", advantages, lead, dev)
    if ref_logp is not None:
        ref_logp = _per_row("ref_logp", ref_logp, lead, dev)
    elif kl_coef != 0.0:
        raise ValueError("kl_coef: the KL term needs ref_logp")
    if mask is not None:
        mask = flags_of("mask", mask, lead, dev).contiguous()
    if not e_clip >= 0.0:
        raise ValueError(f"e_clip: {e_clip}")
    if logits.numel() == 0:
        return logits.sum().float(), torch.zeros(6, device=dev)
    return _TokenPolicyLoss.apply(logits, actions, old_logp, advantages, ref_logp, mask, (float(e_clip), float(kl_coef), float(entropy_coef)),
                                  wants_gradient(logits))


def action_logp(logits, actions):
    """log softmax(logits)[action] and the entropy of every row, float32 [...]: what a rollout stores as old_logp and what a reference
    policy's logits give as ref_logp.  No gradients.  An action outside [0, V) and a row of nothing but -inf give NaN."""
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("action_logp has no backward pass: detach the logits (policy_loss trains)")
    logits, lead, actions = _rows(logits, actions)
    logp = torch.empty(lead, dtype=torch.float32, device=logits.device)
    entropy = torch.empty_like(logp)
    if logits.numel():
        logits, r0, r1, v, s0, s1 = _table(logits)
        with on_device_of(logits):
            N.check(N.load().ag_token_logp(logits.data_ptr(), r0, r1, s0, s1, v, N.AG_DTYPES[logits.dtype], actions.data_ptr(),
                                           logp.data_ptr(), entropy.data_ptr(), stream_of(logits)), "ag_token_logp")
    return logp, entropy
