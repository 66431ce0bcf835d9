"""64-bit definitions of the policy and the preference loss, on the CPU, for the tests.

Written with whole-array torch operations and differentiated by autograd; the
kernels are compared with these at the same (rounded) inputs.
"""

import math

import torch


def token_sequences(shape, cu):
    """Sequence index of every token, -1 for none, and the number of sequences."""
    if cu is None:
        S, T = shape if len(shape) == 2 else (1, shape[0])
        return torch.arange(S).repeat_interleave(T), S
    n = shape[0]
    seq = torch.full((n,), -1)
    for s in range(len(cu) - 1):
        seq[cu[s]:cu[s + 1]] = s
    return seq, len(cu) - 1


def policy(logp, old, adv, ref=None, mask=None, cu=None, clip=0.2, clip_high=None, dual_clip=None, kl_coef=0.0,
           reduction="mean", grad_out=None):
    """dict(loss, grad, kl, clip_fraction, size): size is the sum of the terms'
    magnitudes behind the loss, gsize behind every gradient."""
    shape = logp.shape
    x = logp.detach().reshape(-1).double().requires_grad_(True)
    n = x.numel()
    seq, S = token_sequences(shape, cu)
    on = seq >= 0
    if mask is not None:
        on = on & mask.reshape(-1).bool()
    i = on.nonzero()[:, 0]
    A = adv.reshape(-1).double()
    A = A[i] if adv.shape == shape else A[seq[i]]
    xi = x[i]
    d = xi - (old.reshape(-1)[i].double() if old is not None else xi.detach())
    r = torch.exp(d)
    lo, hi = 1 - clip, 1 + (clip if clip_high is None else clip_high)
    a, b = r * A, torch.clamp(r, lo, hi) * A
    cut = torch.where(A > 0, r > hi, (A < 0) & (r < lo))
    pg = torch.where(cut, b, a)
    if dual_clip is not None:
        far = (A < 0) & (r > dual_clip)
        pg = torch.where(far, dual_clip * A, pg)
        cut = cut | far
    kl = torch.zeros_like(xi)
    gk = torch.zeros_like(xi)
    if ref is not None:
        q = ref.reshape(-1)[i].double() - xi
        kl = torch.expm1(q) - q
        gk = abs(kl_coef) * torch.expm1(q).detach().abs()  # |beta (e^q - 1)|: a magnitude, whatever beta's sign
    tok = -pg + kl_coef * kl
    cnt = max(len(i), 1)
    if reduction == "sequence":
        per = torch.bincount(seq[i], minlength=S).double()
        w = 1.0 / (per[seq[i]] * max(int((per > 0).sum()), 1))
    elif reduction == "mean":
        w = torch.full_like(xi, 1.0 / cnt)
    else:
        w = torch.ones_like(xi)
    size = (tok.detach().abs() * 0 + pg.detach().abs() + abs(kl_coef) * kl.detach()) * w
    gsize = torch.zeros(n, dtype=torch.float64)
    up = torch.ones(()) if grad_out is None else grad_out
    if reduction == "none":
        full = torch.zeros(n, dtype=torch.float64).index_put((i,), tok)
        loss = full.view(shape)
        ui = up.reshape(-1)[i].double() if up.dim() else up.double()
        total = (tok * ui).sum()
        lsize = torch.zeros(n, dtype=torch.float64).index_put((i,), size).view(shape)
    else:
        loss = (tok * w).sum()
        ui = up.double()
        total = loss * ui
        lsize = size.sum()
    grad = torch.autograd.grad(total, [x])[0] if len(i) else torch.zeros_like(x)
    gsize[i] = (a.detach().abs() + gk) * w * ui.abs()
    return dict(loss=loss.detach(), lsize=lsize, grad=grad.view(shape), gsize=gsize.view(shape),
                kl=kl.detach().sum() / cnt, clip_fraction=cut.double().sum() / cnt)


def preference(logp, ref=None, mask=None, cu=None, beta=0.1, margin=0.0, loss_type="sigmoid", label_smoothing=0.0,
               length_normalize=False, reduction="mean", grad_out=None):
    shape = logp.shape
    x = logp.detach().reshape(-1).double().requires_grad_(True)
    seq, S = token_sequences(shape, cu)
    on = seq >= 0
    if mask is not None:
        on = on & mask.reshape(-1).bool()
    i = on.nonzero()[:, 0]
    P = S // 2
    per_token = ref is not None and ref.shape == shape
    d = x[i] - (ref.reshape(-1)[i].double() if per_token else 0.0)
    D = torch.zeros(S, dtype=torch.float64).index_add(0, seq[i], d)
    # a 32-bit difference per token, 64-bit sums
    dsize = torch.zeros(S, dtype=torch.float64).index_add(0, seq[i], d.detach().abs())
    if ref is not None and not per_token:
        D = D - ref.double()
    if length_normalize:
        c = torch.bincount(seq[i], minlength=S).clamp(min=1).double()
        D, dsize = D / c, dsize / c
    gap = D[:P] - D[P:]
    h = beta * gap - margin
    if loss_type == "sigmoid":
        loss = -(1 - label_smoothing) * torch.nn.functional.logsigmoid(h) \
            - label_smoothing * torch.nn.functional.logsigmoid(-h)
    elif loss_type == "hinge":
        loss = torch.relu(1 - h)
    else:
        loss = (gap - 1 / (2 * beta)) ** 2
    pairs = loss
    if reduction == "mean":
        loss = loss.sum() / max(P, 1)
    elif reduction == "sum":
        loss = loss.sum()
    up = torch.ones(()) if grad_out is None else grad_out
    total = (loss * up.double()).sum()
    grad = torch.autograd.grad(total, [x])[0] if x.numel() and P else torch.zeros_like(x)
    return dict(loss=loss.detach(), pairs=pairs.detach(), grad=grad.view(shape), chosen=beta * D.detach()[:P],
                rejected=beta * D.detach()[P:], gap=gap.detach(), dsize=dsize)


def cuts(n, S, gen, first=0, last=0):
    """Offsets of S sequences, some empty, that leave `first` and `last` tokens to none."""
    at = torch.randint(first, n - last + 1, (S + 1,), generator=gen).sort().values
    at[0], at[-1] = first, n - last
    if S >= 4:
        at[2] = at[1]  # an empty sequence
    return at.tolist()


def half_steps(dtype, value):
    """Half a rounding step of `dtype` at `value` (below the normal range: of the smallest step)."""
    info = torch.finfo(dtype)
    return info.eps / 2 * torch.clamp(value.abs(), min=info.tiny)


INF, NAN = math.inf, math.nan
