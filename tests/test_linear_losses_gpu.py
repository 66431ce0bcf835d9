"""GPU tests of the losses on a head's log-probabilities against 64 bits.

Tolerances are bounds of the arithmetic, element by element, with u = 2^-24 (half
a float32 step), h half a step of the input type, and B = max over the logits of
sum_k |e_k c_k|:

* a logit: tensor cores add products of 16 at a time rounding towards zero (2u);
  of 16-bit inputs 16 such steps per segment, then one float32 addition per 256
  products: dz = (16 * 2u + ceil(D / 256) u) B (bfloat16 runs 32 steps per segment
  and is held to the same bound but for long vocabularies); of float32 inputs, each the sum of
  two float16 parts to 2^-22 (4u) and the parts' smallest product left out (4u),
  8 steps per segment and three additions per 128 columns: dz = (8 * 2u +
  3 * (ceil(D / 128) + 1) u + 12u) B; the bias and the temperature 2u |z| more;
* a log-probability: the target's logit and the log-sum-exp move by dz each;
  exp2 and its argument (|z - max| < 40) and the logarithm: within 2^-18;
* a dlogit w, a difference of softmax and teacher values times the row's
  cotangent d: those values carry 2 dz + 2^-18 relative each; w is rounded to the
  input type (h; float32 inputs: to two float16 parts, as e and c, h = 12u);
  float16 parts are in units of 2^-14 of the largest d's power of two, so half
  their smallest step is 2^-39 of it;
* a gradient sum_v w_v c_v: those relative errors times sum_v |w_v c_v|, and the
  accumulation's: 2u per 16 terms, u per segment, chunk and K split added;
  the result is rounded to the input type (eps / 2).
"""

import gc
import math

import pytest
import torch

import mlx_cce
import token_loss_ref as R
from mlx_cce import _ext

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def head(N, D, V, dtype, seed, bias=None, peak=6.0):
    g = torch.Generator().manual_seed(seed)
    c = torch.randn(V, D, generator=g) * D ** -0.5
    e = torch.randn(N, D, generator=g)
    t = torch.randint(0, V, (N,), generator=g)
    ct = c[t]
    e = e + peak * ct / (ct * ct).sum(1, keepdim=True).clamp(min=0.05)
    b = None if bias is None else (torch.randn(V, generator=g) * 0.5).to(bias)
    return e.to(dtype), c.to(dtype), b, t, g


class Bounds:
    """The bounds above for one head."""

    def __init__(self, e, c, b, T=1.0):
        N, D = e.shape
        big = float((e.double().abs() @ c.double().abs().t()).max()) if N else 0.0
        f32 = e.dtype == torch.float32
        steps = 8 * 2 + 3 * (math.ceil(D / 128) + 1) + 12 if f32 else 16 * 2 + math.ceil(D / 256)
        z = big + (0.0 if b is None else float(b.double().abs().max()))
        self.dz = (steps * U * big + 2 * U * z) / T
        self.dlogp = 2 * self.dz + 2.0 ** -18
        self.h = 12 * U if f32 else torch.finfo(e.dtype).eps / 2
        self.tiny = 0.0 if e.dtype == torch.bfloat16 else 2.0 ** -39


def leaves(e, c, b):
    return [x.cuda().requires_grad_(True) for x in (e, c)] + ([] if b is None else [b.cuda().requires_grad_(True)])


def check_grads(B, grads, e, c, b, w, mag, d):
    """w: 64-bit dlogits [N, V] (by the logits before any temperature), each the
    difference of parts whose magnitudes sum to mag d (d: the rows' cotangents): a
    softmax value q next to 1 in q - 1 leaves an error of q's size, not of w's."""
    extra = mag * d[:, None] * (2 * B.dz + 2.0 ** -18)
    wa = w.abs() + extra
    e64, c64 = e.double(), c.double()
    for got, want, left, other, add, what in (
            (grads[0], w @ c64, wa, c64, extra @ c64.abs(), "grad_e"),
            (grads[1], w.t() @ e64, wa.t(), e64, extra.t() @ e64.abs(), "grad_c")):
        got = got.cpu()
        tol = add + (left @ other.abs()) * (B.h + (left.shape[1] / 16 + 64) * 2 * U)
        tol = tol + 2.0 ** math.ceil(math.log2(max(float(d.max()), 1e-30))) * B.tiny * other.abs().sum(0)
        if got.dtype != torch.float32:
            tol = tol + R.half_steps(got.dtype, want.abs() + tol)
        bad = (got.double() - want).abs() > tol + 1e-37
        assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])
    if b is not None:
        tol = extra.sum(0) + wa.sum(0) * (e.shape[0] + 64) * U + 1e-37
        if b.dtype != torch.float32:
            tol = tol + R.half_steps(b.dtype, w.sum(0).abs() + tol)
        assert torch.all((grads[2].cpu().double() - w.sum(0)).abs() <= tol), "grad_bias"


# ---------------------------------------------------------------------------
# log-probabilities
# ---------------------------------------------------------------------------

def check_log_probs(N, D, V, dtype, bias=None, ignore=0.3, seed=0, int32=False):
    e, c, b, t, g = head(N, D, V, dtype, seed + N + D + V, bias)
    t = torch.where(torch.rand(N, generator=g) < ignore, torch.full_like(t, -100), t)
    go = torch.randn(N, generator=g)
    xs = leaves(e, c, b)
    logp = mlx_cce.linear_log_probs(xs[0], xs[1], (t.int() if int32 else t).cuda(), *xs[2:])
    grads = torch.autograd.grad(logp, xs, go.cuda())
    z = e.double() @ c.double().t() + (0 if b is None else b.double())
    lq = torch.log_softmax(z, 1)
    on = t >= 0
    want = torch.where(on, lq.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    B = Bounds(e, c, b)
    assert logp.dtype == torch.float32
    assert torch.all((logp.detach().cpu().double() - want).abs() <= B.dlogp)
    w = torch.zeros(N, V, dtype=torch.float64)
    w[on] = -lq[on].exp()
    w[on, t[on]] += 1
    mag = torch.where(on[:, None], lq.exp(), 0.0)
    check_grads(B, grads, e, c, b, w * go.double()[:, None], mag, (go * on).abs().double())
    _ext.device_status()


SHAPES = [(1, 64, 40), (128, 64, 256), (130, 72, 1000), (257, 136, 2049), (300, 520, 5000), (40, 2048, 777)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,V", SHAPES)
def test_log_probs(N, D, V, dtype):
    check_log_probs(N, D, V, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D,V", [(33, 50, 700), (70, 7, 129), (5, 1, 2), (20, 12, 33)])
def test_log_probs_odd_widths(N, D, V, dtype):
    check_log_probs(N, D, V, dtype, bias=torch.float32)


@pytest.mark.parametrize("bias", DTYPES)
def test_log_probs_bias_types(bias):
    check_log_probs(200, 128, 1500, torch.bfloat16, bias=bias, int32=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_in_several_chunks(dtype, monkeypatch):
    monkeypatch.setenv("CCE_BWD_CHUNK_ROWS", "512")
    check_log_probs(200, 96, 2000, dtype, bias=torch.float32)


def test_log_probs_rows_left_out():
    e, c, b, t, g = head(260, 64, 500, torch.bfloat16, 3)
    for keep in (0, 1, 128, 129, 260):
        tt = t.clone()
        tt[torch.randperm(260, generator=g)[keep:]] = -100
        bad = e.clone()
        bad[tt < 0] = R.NAN  # rows left out are not looked at
        xs = leaves(bad, c, None)
        logp = mlx_cce.linear_log_probs(xs[0], xs[1], tt.cuda())
        ge, gc = torch.autograd.grad(logp.sum(), xs)
        ys = leaves(e[tt >= 0], c, None)
        want = mlx_cce.linear_log_probs(ys[0], ys[1], tt[tt >= 0].cuda())
        we, wc = torch.autograd.grad(want.sum(), ys)
        on = (tt >= 0).cuda()
        assert torch.equal(logp[on], want) and torch.all(logp[~on] == 0)
        assert torch.equal(ge[on], we) and torch.all(ge[~on] == 0) and torch.equal(gc, wc)
    empty = mlx_cce.linear_log_probs(e[:0].cuda().requires_grad_(True), c.cuda(), t[:0].cuda())
    assert empty.shape == (0,)
    empty.sum().backward()


def test_log_probs_ignore_index_and_shapes():
    e, c, _, t, _ = head(24, 64, 300, torch.bfloat16, 4)
    x, w, tt = e.cuda().view(4, 6, 64), c.cuda(), t.cuda().view(4, 6)
    flat = mlx_cce.linear_log_probs(e.cuda(), w, t.cuda(), ignore_index=None)
    assert torch.equal(mlx_cce.linear_log_probs(x, w, tt, ignore_index=None).view(-1), flat)
    zeroed = mlx_cce.linear_log_probs(x, w, torch.zeros_like(tt), ignore_index=0)
    assert torch.all(zeroed == 0)
    # a transposed view, and e one element behind an aligned address
    xt = x.transpose(0, 1)
    assert torch.equal(mlx_cce.linear_log_probs(xt, w, tt.t()), flat.view(4, 6).t())
    buf = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    buf[1:].copy_(e.view(-1))
    assert torch.equal(mlx_cce.linear_log_probs(buf[1:].view(24, 64), w, t.cuda()), flat)


def test_log_probs_are_not_biased():
    """Two-level accumulation: over many rows with large logits the mean error is
    far below a tensor core's one-directional 1e-5 (its rounding towards zero)."""
    e, c, _, t, _ = head(512, 4096, 512, torch.bfloat16, 5, peak=14.0)
    lp = mlx_cce.linear_log_probs(e.cuda(), c.cuda(), t.cuda()).cpu().double()
    want = torch.log_softmax(e.double() @ c.double().t(), 1).gather(1, t[:, None])[:, 0]
    # 16 segments, each at most 16 steps of 2u towards zero on a partial logit of about 2 (14 / 8
    # segments' worth and noise): below 16 * 16 * 2u * 2 / 2 on average
    assert float((lp - want).mean().abs()) < 256 * 2 * U
    assert float((lp - want).abs().max()) < Bounds(e, c, None).dlogp


# ---------------------------------------------------------------------------
# policy and preference loss of a head
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum", "none"])
def test_linear_policy_is_the_two_operators(dtype, reduction):
    e, c, b, t, g = head(300, 64, 700, dtype, 20, bias=torch.float32)
    t = torch.where(torch.rand(300, generator=g) < 0.3, torch.full_like(t, -100), t).cuda()
    cu = torch.tensor([3, 60, 60, 200, 290], dtype=torch.int32, device="cuda")
    old, ref = (-torch.rand(300, generator=g) * 5).cuda(), (-torch.rand(300, generator=g) * 5).cuda()
    adv = torch.randn(4, generator=g).cuda()
    kw = dict(ref_logp=ref, cu_seqlens=cu, kl_coef=0.1, clip=0.3, reduction=reduction, return_stats=True)
    xs = leaves(e, c, b)
    loss, stats = mlx_cce.linear_policy_loss(xs[0], xs[1], t, old, adv, xs[2], **kw)
    ys = leaves(e, c, b)
    logp = mlx_cce.linear_log_probs(ys[0], ys[1], t, ys[2])
    want, wstats = mlx_cce.policy_loss(logp, old, adv, mask=t >= 0, **kw)
    assert torch.equal(loss, want) and all(torch.equal(a, w) for a, w in zip(stats, wstats))
    for a, w in zip(torch.autograd.grad(loss.sum(), xs), torch.autograd.grad(want.sum(), ys)):
        assert torch.equal(a, w)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("padded", [True, False])
def test_linear_preference_is_the_two_operators(dtype, padded):
    e, c, b, t, g = head(240, 64, 700, dtype, 21)
    t = torch.where(torch.rand(240, generator=g) < 0.3, torch.full_like(t, -100), t).cuda()
    ref = (-torch.rand(240, generator=g) * 5).cuda()
    shape = (6, 40) if padded else (240,)
    kw = dict(beta=0.2, label_smoothing=0.1, return_rewards=True)
    if not padded:
        kw["cu_seqlens"] = torch.tensor([0, 30, 90, 90, 150, 200, 240], device="cuda")
    xs, ys = leaves(e, c, b), leaves(e, c, b)
    loss, rew = mlx_cce.linear_preference_loss(xs[0].view(*shape, 64), xs[1], t.view(shape), ref.view(shape), **kw)
    logp = mlx_cce.linear_log_probs(ys[0], ys[1], t).view(shape)
    want, wrew = mlx_cce.preference_loss(logp, ref.view(shape), mask=t.view(shape) >= 0, **kw)
    assert torch.equal(loss, want) and torch.equal(rew.chosen, wrew.chosen)
    for a, w in zip(torch.autograd.grad(loss, xs), torch.autograd.grad(want, ys)):
        assert torch.equal(a, w)


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------

def teacher(e, c, b, K, g, sharp=1.1):
    z = e.float() @ c.float().t() + (0 if b is None else b.float())
    z = sharp * z + 0.5 * torch.randn(z.shape, generator=g)
    lp, ids = z.log_softmax(1).topk(K, dim=1)
    p = torch.rand(ids.shape, generator=g).argsort(1)  # any order
    return lp.gather(1, p), ids.gather(1, p)


def distill64(e, c, b, ids, tlp, T=1.0, tail=False, mask=None, reduction="mean", go=None):
    """(loss, per-row size of its terms, 64-bit dlogits by the raw logits)"""
    N, V = e.shape[0], c.shape[0]
    raw = (e.double() @ c.double().t() + (0 if b is None else b.double())).requires_grad_(True)
    lq = torch.log_softmax(raw / T, 1)
    there = (ids >= 0) & (ids < V)
    t = tlp.double()
    if tail:
        p = torch.where(there, t.exp(), 0.0)
    else:
        s = torch.where(there, t / T, -math.inf)
        none = torch.isinf(s).all(1, keepdim=True)
        p = torch.where(none, 0.0, torch.softmax(torch.where(none, 0.0, s), 1))
    full = torch.zeros(N, V, dtype=torch.float64).scatter_add(1, ids.clamp(0, V - 1), torch.where(there, p, 0.0))
    member = torch.zeros(N, V, dtype=torch.bool)
    i, k = there.nonzero(as_tuple=True)
    member[i, ids[i, k]] = True
    lqs = torch.where(full > 0, lq, 0.0)
    rows = (torch.special.xlogy(full, full) - full * lqs).sum(1)
    size = (torch.special.xlogy(full, full).abs() + full * lqs.abs()).sum(1).detach()
    has = there.any(1)
    if tail:
        rest = torch.where(has & ~member.all(1), (1 - full.sum(1)).clamp(min=0), 0.0)
        out = torch.where(member, -math.inf, lq).logsumexp(1)
        out = torch.where(member.all(1), 0.0, out)
        term = torch.special.xlogy(rest, rest) - rest * out
        rows = rows + term
        size = size + (torch.special.xlogy(rest, rest).abs() + rest * out.abs()).detach()
    else:
        has = has & (full.sum(1) > 0)
    on = has if mask is None else has & mask
    rows = torch.where(on, rows, 0.0)
    if reduction == "mean":
        loss = rows.sum() / max(int(on.sum()), 1)
    else:
        loss = rows.sum() if reduction == "sum" else rows
    total = (loss * (1.0 if go is None else go.double())).sum()
    (w,) = torch.autograd.grad(total, [raw])
    return loss.detach(), torch.where(on, size, 0.0), w, on


def check_distill(e, c, b, ids, tlp, T=1.0, tail=False, mask=None, reduction="mean", go=None, int32=False):
    xs = leaves(e, c, b)
    loss = mlx_cce.linear_distillation_loss(xs[0], xs[1], (ids.int() if int32 else ids).cuda(), tlp.cuda(), *xs[2:],
                                            temperature=T, tail=tail, mask=None if mask is None else mask.cuda(),
                                            reduction=reduction)
    grads = torch.autograd.grad(loss, xs, None if go is None else go.cuda())
    want, size, w, on = distill64(e, c, b, ids, tlp, T, tail, mask, reduction, go)
    B = Bounds(e, c, b, T)
    # teacher probabilities: expf, the sum and its division: 2^-19 of every term
    row = torch.where(on, B.dlogp + 2.0 ** -19 * (1 + size), 0.0)
    n = max(int(on.sum()), 1)
    tol = row if reduction == "none" else row.sum() / (n if reduction == "mean" else 1)
    assert loss.dtype == torch.float32
    assert torch.all((loss.detach().cpu().double() - want).abs() <= tol + 2 * U * want.abs()), (loss, want)
    # dlogits are differences whole q - p: the errors of both sides, each at most
    # the row's cotangent times 2 dz + 2^-18 relative
    d = (torch.ones(()) if go is None else go.double().abs()) * on / (n if reduction == "mean" else 1) / T
    lq = torch.log_softmax((e.double() @ c.double().t() + (0 if b is None else b.double())) / T, 1)
    V = c.shape[0]
    there = (ids >= 0) & (ids < V)
    p = torch.where(there, tlp.double().exp() if tail else
                    torch.nan_to_num(torch.softmax(torch.where(there, tlp.double() / T, -math.inf), 1)), 0.0)
    full = torch.zeros(e.shape[0], V, dtype=torch.float64).scatter_add(1, ids.clamp(0, V - 1), p)
    mag = lq.exp() + full
    if tail:
        member = torch.zeros(e.shape[0], V, dtype=torch.bool)
        i, k = there.nonzero(as_tuple=True)
        member[i, ids[i, k]] = True
        rest = (1 - full.sum(1)).clamp(min=0)
        out = torch.where(member, -math.inf, lq)
        mag = mag + torch.nan_to_num(torch.softmax(out, 1)) * rest[:, None]
        # r = 1 - sum p is held in 64 bits and rounded: u; q_r and r differ by those errors
    check_grads(B, grads, e, c, b, w, mag, d)
    _ext.device_status()
    return loss.detach(), grads


DISTILL = [(1, 64, 40, 1), (128, 64, 256, 2), (130, 72, 1000, 7), (257, 136, 2049, 33), (300, 520, 5000, 64),
           (20, 64, 3001, 1024), (64, 72, 300, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("N,D,V,K", DISTILL)
def test_distillation(N, D, V, K, tail, dtype):
    e, c, b, _, g = head(N, D, V, dtype, N + K)
    tlp, ids = teacher(e, c, b, K, g)
    check_distill(e, c, b, ids, tlp, T=1.0 if tail else 2.0, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_masks_bias_and_absent_entries(tail, reduction, dtype):
    e, c, b, _, g = head(200, 64, 1200, dtype, 41, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 20, g)
    ids = torch.where(torch.rand(ids.shape, generator=g) < 0.2, torch.full_like(ids, -1), ids)
    ids[3] = -1                # a row without any entry
    ids[4, ::2] = 1200 + 5     # past the vocabulary: absent too
    tlp[5, ::2] = -R.INF       # entries without mass
    if not tail:
        tlp[6] = -R.INF        # nor any in the row
    mask = torch.rand(200, generator=g) < 0.8
    bad = torch.where(mask[:, None], e.float(), R.NAN).to(dtype)
    go = torch.randn(200, generator=g) if reduction == "none" else torch.tensor(2.0)
    kw = dict(T=1.5, tail=tail, mask=mask, reduction=reduction, go=go)
    loss, grads = check_distill(e, c, b, ids, tlp, int32=True, **kw)
    assert torch.all(grads[0][~mask.cuda()] == 0) and torch.all(grads[0][3] == 0)
    # what masked rows hold is not looked at
    tn = torch.where(mask[:, None], tlp, R.NAN)
    xs = leaves(bad, c, b)
    again = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids.cuda(), tn.cuda(), xs[2], temperature=1.5, tail=tail,
                                             mask=mask.cuda(), reduction=reduction)
    got = torch.autograd.grad(again, xs, go.cuda())
    assert torch.equal(again, loss) and all(torch.equal(a, w) for a, w in zip(got, grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_same_id_twice(tail, dtype):
    e, c, b, _, g = head(70, 64, 600, dtype, 42)
    tlp, ids = teacher(e, c, b, 12, g)
    ids[:, 5] = ids[:, 0]
    ids[:, 7] = ids[:, 0]
    tlp = tlp - 1.0  # (so that repeated entries leave some mass over)
    check_distill(e, c, b, ids, tlp, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_odd_widths_and_chunks(dtype, monkeypatch):
    e, c, b, _, g = head(90, 50, 1100, dtype, 43, bias=torch.bfloat16)
    tlp, ids = teacher(e, c, b, 9, g)
    check_distill(e, c, b, ids, tlp, T=0.7)
    monkeypatch.setenv("CCE_BWD_CHUNK_ROWS", "256")
    e, c, b, _, g = head(140, 64, 1100, dtype, 44, bias=torch.float16)
    tlp, ids = teacher(e, c, b, 9, g)
    check_distill(e, c, b, ids, tlp, tail=True)


def test_distillation_tiny_tail_keeps_its_digits():
    """A student whose mass outside of the entries is 1e-9: 1 - sum q would be 0."""
    g = torch.Generator().manual_seed(45)
    V, D, N = 400, 64, 32
    c = torch.randn(V, D, generator=g) * 0.1
    b = torch.full((V,), -30.0)
    ids = torch.arange(8).repeat(N, 1)
    b[:8] = 0.0
    e = torch.randn(N, D, generator=g)
    tlp = torch.log_softmax(torch.randn(N, 8, generator=g), 1) + math.log(0.999)
    check_distill(e.bfloat16(), c.bfloat16(), b, ids, tlp, tail=True)


def test_distillation_without_rows():
    e, c, b, _, g = head(150, 64, 300, torch.bfloat16, 46)
    tlp, ids = teacher(e, c, b, 4, g)
    xs = leaves(e, c, None)
    loss = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids.cuda(), tlp.cuda(), mask=torch.zeros(150).bool().cuda())
    grads = torch.autograd.grad(loss, xs)
    assert float(loss) == 0 and all(torch.all(x == 0) for x in grads)
    loss = mlx_cce.linear_distillation_loss(xs[0][:0], xs[1], ids[:0].cuda(), tlp[:0].cuda())
    grads = torch.autograd.grad(loss, xs)
    assert float(loss) == 0 and all(torch.all(x == 0) for x in grads)


def test_only_the_gradients_asked_for():
    e, c, b, t, g = head(140, 64, 300, torch.bfloat16, 47, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 4, g)
    f = lambda x, w, v: mlx_cce.linear_distillation_loss(x, w, ids.cuda(), tlp.cuda(), v)
    h = lambda x, w, v: mlx_cce.linear_log_probs(x, w, t.cuda(), v).sum()
    for fn in (f, h):
        xs = leaves(e, c, b)
        want = torch.autograd.grad(fn(*xs), xs)
        for k in range(3):
            ys = [x.detach().requires_grad_(i == k) for i, x in enumerate(xs)]
            (got,) = torch.autograd.grad(fn(*ys), [ys[k]])
            assert torch.equal(got, want[k])


def test_gradients_against_differences():
    """Central differences of the kernel's own loss along a direction, float32
    inputs: error h^2/6 |L'''| + rounding. Directions of norm 1, h = 2^-5."""
    e, c, b, t, g = head(24, 32, 90, torch.float32, 48, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 6, g)
    f = lambda x, w, v: mlx_cce.linear_distillation_loss(x, w, ids.cuda(), tlp.cuda(), v, temperature=1.3)
    xs = leaves(e, c, b)
    grads = torch.autograd.grad(f(*xs), xs)
    h = 2.0 ** -5
    for k in range(3):
        d = torch.randn(xs[k].shape, generator=g).cuda()
        d = d / d.norm()
        plus = [x.detach() + h * d if i == k else x.detach() for i, x in enumerate(xs)]
        minus = [x.detach() - h * d if i == k else x.detach() for i, x in enumerate(xs)]
        diff = (float(f(*plus)) - float(f(*minus))) / (2 * h)
        # |z| changes by at most |d| max(|c|, |e|) per unit: L''' <= 6 (that)^3; the loss carries 2^-18
        reach = max(float(e.norm(dim=1).max()), float(c.norm(dim=1).max())) / 1.3 if k < 2 else 1.0
        mean = 1 / 24 if k < 2 else 1.0  # a unit direction in e or c moves few of the mean's rows far
        assert abs(diff - float((grads[k] * d).sum())) <= h * h * reach ** 3 * mean + 2.0 ** -18 / h


def test_second_derivatives_are_an_error_and_changed_weights_are_noticed():
    e, c, b, t, g = head(40, 64, 300, torch.bfloat16, 51)
    tlp, ids = teacher(e, c, b, 4, g)
    xs = leaves(e, c, None)
    for fn in (lambda: mlx_cce.linear_distillation_loss(xs[0], xs[1], ids.cuda(), tlp.cuda()),
               lambda: mlx_cce.linear_log_probs(xs[0], xs[1], t.cuda()).sum(),
               lambda: mlx_cce.linear_preference_loss(xs[0].view(4, 10, 64), xs[1], t.view(4, 10).cuda())):
        ge, gc = torch.autograd.grad(fn(), xs, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            ge.float().sum().backward()
        loss = fn()
        with torch.no_grad():
            xs[1].mul_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_results_do_not_change_between_runs():
    e, c, b, t, g = head(700, 128, 3000, torch.bfloat16, 49, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 16, g)

    def run():
        xs = leaves(e, c, b)
        loss = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids.cuda(), tlp.cuda(), xs[2], tail=True)
        loss = loss + mlx_cce.linear_log_probs(xs[0], xs[1], t.cuda(), xs[2]).sum()
        return [loss.detach(), *torch.autograd.grad(loss, xs)]

    a = run()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(a, run()))


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------

def _mixed(e, c, ids, tlp, t, old, adv, cu):
    """On-policy distillation: a policy loss and a distillation loss of one head."""
    loss = mlx_cce.linear_policy_loss(e, c, t, old, adv, cu_seqlens=cu, reduction="sequence")
    return loss + 0.5 * mlx_cce.linear_distillation_loss(e, c, ids, tlp, temperature=2.0, mask=t >= 0)


def _mixed_inputs(seed):
    e, c, _, t, g = head(300, 128, 2000, torch.bfloat16, seed)
    tlp, ids = teacher(e, c, None, 8, g)
    t = torch.where(torch.rand(300, generator=g) < 0.3, torch.full_like(t, -100), t)
    cu = torch.tensor([0, 100, 180, 300], dtype=torch.int32)
    old, adv = -torch.rand(300, generator=g), torch.randn(3, generator=g)
    return [x.cuda() for x in (e, c, ids, tlp, t, old, adv, cu)]


def _grads(args):
    e, c = (x.detach().requires_grad_(True) for x in args[:2])
    loss = _mixed(e, c, *args[2:])
    return [loss.detach(), *torch.autograd.grad(loss, [e, c])]


def test_two_streams_at_once():
    ins = [_mixed_inputs(60 + k) for k in range(2)]
    want = [_grads(a) for a in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(_grads(ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(x, y) for x, y in zip(r, want[k]))


def test_captured_and_replayed():
    args = _mixed_inputs(70)
    e, c = (x.detach().requires_grad_(True) for x in args[:2])

    def step():
        loss = _mixed(e, c, *args[2:])
        return [loss, *torch.autograd.grad(loss, [e, c])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for scale in (1.0, 0.5):
        with torch.no_grad():
            e.mul_(scale)
        want = [x.detach().clone() for x in step()]
        for gr, _ in graphs + graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(x.detach(), y) for x, y in zip(out, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_with_other_rows_than_replayed(dtype):
    """The rows that count, and so the row tiles and K splits, are the replay's."""
    e, c, b, t, g = head(700, 64, 3000, dtype, 95, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 8, g)
    tlp, ids = tlp.cuda(), ids.cuda()
    xs = leaves(e, c, b)
    targets, mask = t.cuda(), torch.ones(700, dtype=torch.bool, device="cuda")

    def step():
        logp = mlx_cce.linear_log_probs(xs[0], xs[1], targets, xs[2])
        loss = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids, tlp, xs[2], mask=mask)
        return [logp, loss, *torch.autograd.grad(logp.sum() + loss, xs)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for keep in (700, 0, 1, 130, 700):
        targets.copy_(torch.where(torch.arange(700) < keep, t, torch.full_like(t, -100)))
        mask.copy_(torch.arange(700) >= 700 - keep)
        want = [x.detach().clone() for x in step()]
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.detach(), y) for x, y in zip(out, want))


def test_capture_beside_a_live_eager_graph_is_refused():
    """Refused before anything of the backward pass runs; without the eager graph the
    same capture works."""
    args = _mixed_inputs(71)
    e, c = (x.detach().requires_grad_(True) for x in args[:2])
    eager = _mixed(e, c, *args[2:])
    gr = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="delete its loss first"):
        with torch.cuda.graph(gr):
            _mixed(e, c, *args[2:]).backward()
    eager.backward()
    want = [e.grad.clone(), c.grad.clone()]
    del eager, gr
    gc.collect()  # (the refused call's frames hold its loss)
    e.grad = c.grad = None
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        loss = _mixed(e, c, *args[2:])
        loss.backward()
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(e.grad, want[0]) and torch.equal(c.grad, want[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_not_finite_stay_alone(dtype):
    """A NaN or infinite row that counts, or an infinite upstream gradient, costs its own
    row: the others get the bits they get beside a row of zeros."""
    e, c, b, t, g = head(150, 64, 700, dtype, 90)
    up = torch.randn(150, generator=g).cuda()
    def run(bad, g3):
        e1 = e.clone()
        e1[3] = 0
        e1[3, 5:7] = bad
        e1 = e1.cuda().requires_grad_(True)
        logp = mlx_cce.linear_log_probs(e1, c.cuda(), t.cuda())
        u = up.clone()
        u[3] = g3
        return logp.detach(), torch.autograd.grad(logp, [e1], u)[0]
    rest = torch.arange(150, device="cuda") != 3
    want = run(0.0, 0.0)
    assert torch.isfinite(want[1]).all()
    for bad, g3 in ((float("nan"), 1.0), (float("inf"), 1.0), (0.0, float("inf")), (0.0, float("nan"))):
        got = run(bad, g3)
        assert torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[1][rest], want[1][rest])
        assert not torch.isfinite(got[1][3]).any() or bad == 0.0


def test_a_run_of_all_operators_together():
    """A padded batch of pairs with a reference, distilled from a teacher besides:
    one loss, one backward pass, against 64 bits."""
    e, c, b, t, g = head(160, 64, 500, torch.float32, 80, bias=torch.float32)
    tlp, ids = teacher(e, c, b, 10, g)
    t = t.view(4, 40).clone()
    t[:, :7] = -100
    t[3, 20:] = -100
    ref = -torch.rand(4, 40, generator=g) * 6
    xs = leaves(e, c, b)
    x4 = xs[0].view(4, 40, 64)
    loss = mlx_cce.linear_preference_loss(x4, xs[1], t.cuda(), ref.cuda(), xs[2], beta=0.1) \
        + mlx_cce.linear_distillation_loss(x4, xs[1], ids.view(4, 40, 10).cuda(), tlp.view(4, 40, 10).cuda(), xs[2],
                                           mask=(t >= 0).cuda())
    grads = torch.autograd.grad(loss, xs)
    on = (t >= 0).view(-1)
    z = e.double() @ c.double().t() + b.double()
    lq = torch.log_softmax(z, 1)
    logp = torch.where(on, lq.gather(1, t.view(-1).clamp(min=0)[:, None])[:, 0], 0.0)
    q = R.preference(logp.view(4, 40), ref, mask=t >= 0)
    dl, _, w, _ = distill64(e, c, b, ids, tlp, mask=on)
    w = w - q["grad"].reshape(-1, 1) * lq.exp()
    w[on, t.view(-1)[on]] += q["grad"].reshape(-1)[on]
    assert abs(float(loss) - float(q["loss"] + dl)) < 2e-5
    for got, want in zip(grads, (w @ c.double(), w.t() @ e.double(), w.sum(0))):
        assert torch.all((got.cpu().double() - want).abs() <= 2e-5 * want.abs().max())


def _free(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def test_offsets_past_32_bits_rows():
    """N D and N V beyond 2^31: the last rows are those of a call of their own."""
    _free(60)
    N, D, V = 540_001, 4096, 4200
    g = torch.Generator(device="cuda").manual_seed(100)
    e = torch.randn(N, D, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    c = (torch.randn(V, D, generator=g, device="cuda") * 0.03).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[5:-300] = torch.where(torch.rand(N - 305, generator=g, device="cuda") < 0.1, -100, t[5:-300])
    logp = mlx_cce.linear_log_probs(e, c, t)
    up = torch.ones(N, device="cuda")
    (grad,) = torch.autograd.grad(logp, [e], up)
    tail = e.detach()[-300:].clone().requires_grad_(True)
    want = mlx_cce.linear_log_probs(tail, c, t[-300:])
    assert torch.equal(logp.detach()[-300:], want.detach())
    (gt,) = torch.autograd.grad(want, [tail], up[:300])
    # the K splits differ with the number of rows: float32 sums in another order, then one rounding each
    w = torch.softmax(tail.detach().float() @ c.float().t(), 1)
    w[torch.arange(300, device="cuda"), t[-300:]] -= 1
    tol = (w.abs() @ c.float().abs()) * ((V / 16 + 64) * 2 * U) + R.half_steps(torch.bfloat16, gt.float()).float() * 2
    assert torch.all((grad[-300:].float() - gt.float()).abs() <= tol * 1.01)
    assert (grad[5:-300][t[5:-300] == -100] == 0).all()
    _ext.device_status()


@pytest.mark.parametrize("D", [4096, 4104])
def test_offsets_past_32_bits_vocabulary(D):
    """V D beyond 2^31, in place and on the padded copy of c: against 64 bits."""
    _free(60)
    N, V = 400, 530_001
    g = torch.Generator(device="cuda").manual_seed(101)
    e = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    c = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    for v in range(0, V, 1 << 16):
        c[v:v + (1 << 16)] = torch.randn(min(1 << 16, V - v), D, generator=g, device="cuda") * 0.03
    t = torch.randint(V - 200, V, (N,), generator=g, device="cuda")
    c.requires_grad_(True)
    logp = mlx_cce.linear_log_probs(e, c, t)
    (grad,) = torch.autograd.grad(logp, [c], torch.ones(N, device="cuda"))
    e64, last = e.double(), c.detach()[-200:].double()
    lse = torch.full((N,), -math.inf, dtype=torch.float64, device="cuda")
    big = 0.0
    for v in range(0, V, 20_000):
        part = c.detach()[v:v + 20_000].double()
        lse = torch.logaddexp(lse, torch.logsumexp(e64 @ part.t(), 1))
        big = max(big, float((e64.abs() @ part.abs().t()).max()))
    lq = e64 @ last.t() - lse[:, None]
    dz = ((32 * 2 + math.ceil(D / 512)) * U) * big   # bfloat16: 32 steps a segment
    want = lq.gather(1, (t - (V - 200))[:, None])[:, 0]
    assert torch.all((logp.detach().double() - want).abs() <= 2 * dz + 2.0 ** -18)
    w = -lq.exp()
    extra = w.abs() * (2 * dz + 2.0 ** -18)
    w[torch.arange(N, device="cuda"), t - (V - 200)] += 1
    wa = w.abs() + extra
    want = w.t() @ e64
    tol = extra.t() @ e64.abs() + (wa.t() @ e64.abs()) * (2.0 ** -8 + (N / 16 + 64) * 2 * U)
    tol = tol + R.half_steps(torch.bfloat16, want.abs().cpu() + tol.cpu()).to("cuda")
    assert torch.all((grad[-200:].double() - want).abs() <= tol)
    _ext.device_status()
