"""The sequence operators restated step by step in float64 on the CPU: causal convolution, selective scan, clipped policy loss.
Differentiable by autograd; test infrastructure only."""
import torch


def _cut(resets, t, b):
    return resets is not None and bool(resets[b, t])


def causal_conv(x, weight, bias, state, silu, lengths=None, resets=None):
    """x [B, T, D], weight [D, W], state [B, W-1, D] or None -> y, state after the last step."""
    B, T, D = x.shape
    W = weight.shape[1]
    ys, lasts = [], []
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        win = [torch.zeros(D, dtype=x.dtype) for _ in range(W - 1)] if state is None else list(state[b])
        row = []
        for t in range(n):
            if _cut(resets, t, b):
                win = [torch.zeros(D, dtype=x.dtype) for _ in range(W - 1)]
            win = win + [x[b, t]]
            p = sum(w * weight[:, k] for k, w in enumerate(win))
            if bias is not None:
                p = p + bias
            row.append(p * torch.sigmoid(p) if silu else p)
            win = win[1:]
        row += [torch.zeros(D, dtype=x.dtype)] * (T - n)
        ys.append(torch.stack(row))
        lasts.append(torch.stack(win))
    return torch.stack(ys), torch.stack(lasts)


def selective_scan(u, delta, A, B, C, D, z, bias, state, softplus=True, lengths=None, resets=None):
    """u, delta, z [b, T, d], A [d, N], B, C [b, T, G, N] -> out, state after the last step."""
    b_, T, d = u.shape
    G = B.shape[2]
    outs, lasts = [], []
    for b in range(b_):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        h = torch.zeros(d, A.shape[1], dtype=u.dtype) if state is None else state[b]
        row = []
        for t in range(n):
            if _cut(resets, t, b):
                h = torch.zeros_like(A)
            dt = delta[b, t] if bias is None else delta[b, t] + bias
            if softplus:
                dt = torch.logaddexp(dt, torch.zeros((), dtype=dt.dtype))
            Bt, Ct = (v[b, t].repeat_interleave(d // G, 0) for v in (B, C))
            h = torch.exp(dt[:, None] * A) * h + (dt * u[b, t])[:, None] * Bt
            y = (h * Ct).sum(-1)
            if D is not None:
                y = y + D * u[b, t]
            if z is not None:
                y = y * z[b, t] * torch.sigmoid(z[b, t])
            row.append(y)
        row += [torch.zeros(d, dtype=u.dtype)] * (T - n)
        outs.append(torch.stack(row))
        lasts.append(h)
    return torch.stack(outs), torch.stack(lasts)


def policy_loss(logits, actions, old_logp, adv, ref_logp, mask, e_clip, kl_coef, entropy_coef):
    """logits [R, V] -> loss, [policy loss, KL term, entropy, KL of the old policy, clipped fraction, rows]."""
    zero = torch.zeros((), dtype=logits.dtype)
    sums, rows = [zero] * 5, 0
    for r in range(logits.shape[0]):
        if mask is not None and not bool(mask[r]):
            continue
        rows += 1
        on = logits[r] > -float("inf")
        top = logits[r][on].max().detach()        # shifts nothing, but log V beside a row of -3e38 is lost in any number format
        x = logits[r][on] - top
        lse = torch.logsumexp(x, 0)
        H = -(torch.exp(x - lse) * (x - lse)).sum()
        lp = (logits[r, actions[r]] - top) - lse
        ratio = torch.exp(lp - old_logp[r])
        pol = torch.maximum(-adv[r] * ratio, -adv[r] * ratio.clamp(1 - e_clip, 1 + e_clip))
        kl = zero
        if ref_logp is not None:
            kl = torch.exp(ref_logp[r] - lp) - (ref_logp[r] - lp) - 1
        terms = (pol, kl, H, ratio - 1 - (lp - old_logp[r]), ((ratio - 1).abs() > e_clip).to(logits.dtype))
        sums = [s + t for s, t in zip(sums, terms)]
    sums = [s / max(rows, 1) for s in sums]
    loss = sums[0] + kl_coef * sums[1] - entropy_coef * sums[2]
    return loss, torch.stack([s.detach() for s in sums] + [torch.tensor(float(rows), dtype=logits.dtype)])
