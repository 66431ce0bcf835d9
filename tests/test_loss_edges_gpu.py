"""GPU tests of the losses on a head's log-probabilities at the edges of their range:
NaN and infinite operands, values of very different sizes, shapes that could be read
two ways, failing calls.  Tolerances are those of ``test_linear_losses_gpu``."""

import math

import pytest
import torch

import mlx_cce
import token_loss_ref as R
from mlx_cce import _ext
from test_loss_edges_cpu import SEGMENTS, drift_bound, drift_inputs
from test_linear_losses_gpu import DTYPES, U, Bounds, distill64, head, leaves, teacher

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


# ---------------------------------------------------------------------------
# NaN in the classifier and the bias
# ---------------------------------------------------------------------------

# (V, columns): alone behind a full tile, a whole 32-column chunk at the start of a
# 128-column half, a whole half, the last chunk of a half, one in the middle
NAN_COLUMNS = [(129, range(128, 129)), (257, range(256, 257)), (300, range(0, 32)), (300, range(128, 256)),
               (400, range(352, 384)), (64, range(0, 64)), (300, range(17, 18))]


def _nan_head(V, cols, where, dtype):
    e, c, b, t, g = head(40, 64, V, dtype, V, bias=torch.float32)
    if where == "c":
        c[list(cols)] = NAN
    else:
        b[list(cols)] = NAN
    return e.cuda(), c.cuda(), b.cuda(), t.cuda(), g


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["c", "bias"])
@pytest.mark.parametrize("V,cols", NAN_COLUMNS)
def test_a_nan_column_is_in_every_rows_sum(V, cols, where, dtype):
    e, c, b, t, g = _nan_head(V, cols, where, dtype)
    assert torch.isnan(mlx_cce.linear_log_probs(e, c, t, b)).all()
    adv = torch.ones(1, device="cuda")
    assert torch.isnan(mlx_cce.linear_policy_loss(e, c, t, None, adv, b))
    assert torch.isnan(mlx_cce.linear_preference_loss(e.view(2, 20, 64), c, t.view(2, 20), None, b))
    # NaN columns among the listed ones, among the others, and beside columns of -infinity
    listed = torch.tensor([cols[0], (cols[-1] + 1) % V], device="cuda").expand(40, 2)
    others = torch.tensor([v for v in range(V) if v not in cols][:2] or [0, 1], device="cuda").expand(40, 2)
    tlp = torch.full((40, 2), math.log(0.25), device="cuda")
    masked = torch.where(torch.isnan(b), b, -INF)
    for tail in (False, True):
        for ids in (listed, others):
            rows = mlx_cce.linear_distillation_loss(e, c, ids, tlp, b, tail=tail, reduction="none")
            assert torch.isnan(rows).all(), (tail, rows)
    if where == "bias":
        assert torch.isnan(mlx_cce.linear_log_probs(e, c, t, masked)).all()
    _ext.device_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_columns_of_minus_infinity_are_still_no_columns(dtype):
    """A bias of -infinity takes its column out, whole chunks and halves of them too."""
    e, c, b, t, _ = head(40, 64, 500, dtype, 7, bias=torch.float32)
    gone = torch.zeros(500, dtype=torch.bool)
    gone[:32] = gone[128:256] = gone[300:310] = True
    t = torch.where(gone[t], torch.full_like(t, 499), t)
    left = torch.nonzero(~gone)[:, 0]
    want = torch.log_softmax(e.double() @ c[left].double().t() + b[left].double(), 1)
    at = torch.searchsorted(left, t)
    got = mlx_cce.linear_log_probs(e.cuda(), c.cuda(), t.cuda(), torch.where(gone, -INF, b).cuda())
    assert torch.all((got.cpu().double() - want.gather(1, at[:, None])[:, 0]).abs() <= Bounds(e, c, b).dlogp)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", ["c", "bias"])
@pytest.mark.parametrize("V,cols", NAN_COLUMNS)
def test_a_nan_column_is_in_the_cross_entropy(V, cols, where, dtype):
    e, c, b, t, _ = _nan_head(V, cols, where, dtype)
    assert torch.isnan(mlx_cce.linear_cross_entropy(e, c, t, b, reduction="none")).all()
    assert torch.isnan(mlx_cce.linear_cross_entropy(e, c, t, torch.where(torch.isnan(b), b, -INF))).all() or where == "c"
    _ext.device_status()


# ---------------------------------------------------------------------------
# rows of very different cotangents
# ---------------------------------------------------------------------------

def _check_rows_apart(grads, e, c, b, w, mag, d, B, floor):
    """As check_grads, but each row's floor is its own: a dlogit of row i is held to
    ``floor`` dd_i (dd: the power of two above its cotangent's bound) beside its
    relative error.  grad_c takes row i's e in units of the largest dd: what that
    leaves of e_i is 2 floor max|e| D / dd_i, weighted by the row's dlogits."""
    extra = mag * d[:, None] * (2 * B.dz + 2.0 ** -18)
    wa = w.abs() + extra
    dd = 2.0 ** torch.ceil(torch.log2((d * mag.max(1).values.clamp(min=1)).clamp(min=1e-300)))
    e64, c64 = e.double(), c.double()
    N, V = w.shape
    half = R.half_steps if e.dtype != torch.float32 else lambda t, x: 0.0

    def off(got, want, tol):
        """Errors; 0 for an infinity of the right sign where the value may round to one
        (float16: from 65520, half a step above its largest number)."""
        err = (got.cpu().double() - want).abs()
        if e.dtype == torch.float16:
            err = torch.where((want.abs() + tol >= 65520) & torch.isinf(got.cpu()) & (got.cpu() * want > 0), 0.0, err)
        return err

    want = w @ c64
    tol = extra @ c64.abs() + (wa @ c64.abs()) * (B.h + (V / 16 + 64) * 2 * U) + floor * dd[:, None] * c64.abs().sum(0)
    tol = tol + half(e.dtype, want.abs() + tol)
    err = off(grads[0], want, tol)
    assert torch.all(err <= tol), ("grad_e", (err / tol).max())
    want = w.t() @ e64
    tol = extra.t() @ e64.abs() + (wa.t() @ e64.abs()) * (2 * B.h + (N / 16 + 64) * 2 * U)
    tol = tol + floor * (dd[:, None] * e64.abs()).sum(0)
    tol = tol + (wa / dd[:, None]).sum(0)[:, None] * 2 * floor * e64.abs().max() * dd.max()
    tol = tol + half(c.dtype, want.abs() + tol)
    err = off(grads[1], want, tol)
    assert torch.all(err <= tol), ("grad_c", (err / tol).max())
    if b is not None:
        tol = extra.sum(0) + wa.sum(0) * (N + 64) * U
        assert torch.all((grads[2].cpu().double() - w.sum(0)).abs() <= tol), "grad_bias"


# half the smallest step of a float16 part, 2^-25, in units of 2^-14 of dd; float32's
# second part is in units of 2^-11 of the first's: 2^-50, and where that part, up to
# 2^-25, is all there is, its product with the other operand's second part, 2^-12 of
# it, is missing: 2^-51 more
FLOORS = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -39, torch.float32: 1.5 * 2.0 ** -50}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("chunks", [1, 6])
def test_one_cotangent_far_above_the_others(dtype, chunks, monkeypatch):
    """An unbounded policy ratio: one row's cotangent 2^30 times the others'.  The other
    rows keep their gradients, tails included."""
    if chunks > 1:
        monkeypatch.setenv("CCE_BWD_CHUNK_ROWS", "512")
    e, c, b, t, g = head(200, 64, 3000, dtype, 11, bias=torch.float32)
    e = (e.float() * 0.5).to(dtype)
    go = torch.randn(200, generator=g) * 2.0 ** -14
    go[7] = 2.0 ** 16
    go[8] = 0.0
    go[9] = 1e-30
    xs = leaves(e, c, b)
    logp = mlx_cce.linear_log_probs(xs[0], xs[1], t.cuda(), xs[2])
    grads = torch.autograd.grad(logp, xs, go.cuda())
    lq = torch.log_softmax(e.double() @ c.double().t() + b.double(), 1)
    w = -lq.exp()
    w[torch.arange(200), t] += 1
    d = go.double()
    B = Bounds(e, c, b)
    _check_rows_apart(grads, e, c, b, w * d[:, None], lq.exp(), d.abs(), B, FLOORS[dtype])
    assert torch.all(grads[0][8] == 0)
    _ext.device_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_bits_again_and_from_a_graph_kept(dtype):
    e, c, b, t, g = head(500, 96, 2500, dtype, 14, bias=torch.float32)
    go = (torch.randn(500, generator=g) * 2.0 ** torch.randint(-12, 12, (500,), generator=g)).cuda()
    tlp, ids = (v.cuda() for v in teacher(e, c, b, 12, g))
    xs = leaves(e, c, b)

    def run():
        logp = mlx_cce.linear_log_probs(xs[0], xs[1], t.cuda(), xs[2])
        rows = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids, tlp, xs[2], tail=True, reduction="none")
        return [(logp + rows).detach(), *torch.autograd.grad((logp, rows), xs, (go, go.flip(0)), retain_graph=True),
                *torch.autograd.grad((logp, rows), xs, (go, go.flip(0)))]

    first = run()
    assert all(torch.equal(x, y) for x, y in zip(first[1:4], first[4:]))
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, run()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_teacher_probabilities_above_one(dtype, reduction):
    """With a tail the teacher's values are used as they are: a sum of 40 must not
    overflow the float16 dlogits."""
    e, c, b, t, g = head(60, 64, 900, dtype, 12)
    tlp, ids = teacher(e, c, b, 8, g)
    tlp = tlp - torch.logsumexp(tlp, 1, keepdim=True)
    tlp[::2] += math.log(40.0)
    tlp[1::2] += math.log(0.6)
    go = torch.randn(60, generator=g) * 2.0 ** 10 if reduction == "none" else torch.tensor(2.0 ** 16)
    xs = leaves(e, c, b)
    loss = mlx_cce.linear_distillation_loss(xs[0], xs[1], ids.cuda(), tlp.cuda(), tail=True, reduction=reduction)
    grads = torch.autograd.grad(loss, xs, go.cuda())
    want, size, w, on = distill64(e, c, b, ids, tlp, tail=True, reduction=reduction, go=go)
    assert torch.all((loss.detach().cpu().double() - want).abs() <= 1e-4 * want.abs() + 1e-4 * size.max())
    q = torch.log_softmax(e.double() @ c.double().t(), 1).exp()
    p = torch.zeros_like(q).scatter_add(1, ids, tlp.double().exp())
    whole = p.sum(1).clamp(min=1)[:, None]
    d = (go.double().abs() if reduction == "none" else go.double().abs().expand(60) / 60).clone()
    if reduction == "mean":  # (one scale for all rows, that of the largest sum)
        d64 = torch.full_like(d, float(d[0]))
        floor = FLOORS[dtype] * float(whole.max())
    else:
        d64, floor = d, FLOORS[dtype]
    B = Bounds(e, c, b)
    # the tail's coefficient is a difference: whole q_r - r, errors of both
    _check_rows_apart(grads, e, c, b, w, whole * q + p + 1, d64, B, floor)
    _ext.device_status()


def _log_probs_of_rest(e, c, b, t, go, row, col):
    """Log-probabilities and gradients of all rows but one, whose e is far above the
    others' and whose cotangent is 0; the classifier's column ``col`` is as far above
    and masked.  What 22-bit parts with a common scale leave of the other values
    besides is 1.5 2^-50 of the power of two above the tensor's largest (FLOORS)."""
    rest = torch.arange(e.shape[0]) != row
    cols = torch.arange(c.shape[0]) != col
    xs = leaves(e, c, b)
    logp = mlx_cce.linear_log_probs(xs[0], xs[1], t.cuda(), xs[2])
    grads = torch.autograd.grad(logp, xs, go.cuda())
    e1, c1, b1, t1 = e[rest], c[cols], b[cols], t[rest] - (t[rest] > col).long()
    lq = torch.log_softmax(e1.double() @ c1.double().t() + b1.double(), 1)
    B = Bounds(e1, c1, b1)
    floor = 2 * FLOORS[e.dtype] if e.dtype == torch.float32 else 0.0
    lost = floor * float(e.abs().max() * c1.abs().sum(1).max() + c.abs().max() * e1.abs().sum(1).max())
    B.dz += lost
    B.dlogp += 2 * lost
    n = e1.shape[0]
    want = lq.gather(1, t1[:, None])[:, 0]
    assert torch.all((logp.detach().cpu().double()[rest] - want).abs() <= B.dlogp)
    w = -lq.exp()
    w[torch.arange(n), t1] += 1
    d = go[rest].double()
    w = w * d[:, None]
    mag = lq.exp()
    extra = mag * d.abs()[:, None] * (2 * B.dz + 2.0 ** -18)
    wa = w.abs() + extra
    h = R.half_steps if e.dtype != torch.float32 else lambda dt, x: 0.0
    for got, left, other, add, big in ((grads[0].cpu()[rest], w, c1.double(), extra @ c1.double().abs(), float(c.abs().max())),
                                       (grads[1].cpu()[cols], w.t(), e1.double(), extra.t() @ e1.double().abs(),
                                        float(e.abs().max()))):
        want = left @ other
        la = wa if left is w else wa.t()
        tol = add + (la @ other.abs()) * (2 * B.h + (left.shape[1] / 16 + 64) * 2 * U)
        tol = tol + floor * big * la.sum(1, keepdim=True)
        tol = tol + FLOORS[e.dtype] * 2 * float(d.abs().max()) * other.abs().sum(0)
        tol = tol + h(e.dtype, want.abs() + tol)
        err = (got.double() - want).abs()
        assert torch.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 192])
def test_values_far_above_the_others(dtype, D):
    """One row of e and one masked column of c 2^24 above the rest of the tensors: the
    other rows keep their digits."""
    e, c, b, t, g = head(200, D, 1500, dtype, 13, bias=torch.float32)
    t = torch.where(t == 5, torch.full_like(t, 6), t)
    e[11] *= 2.0 ** 24
    c[5] *= 2.0 ** 24
    b[5] = -INF
    go = torch.randn(200, generator=g)
    go[11] = 0.0
    _log_probs_of_rest(e, c, b, t, go, 11, 5)
    _ext.device_status()


# ---------------------------------------------------------------------------
# torch's transforms
# ---------------------------------------------------------------------------

def _transformed():
    """(name, a function of one tensor around each loss, its argument)"""
    g = torch.Generator().manual_seed(61)
    x, old = -torch.rand(4, 50, generator=g).cuda(), -torch.rand(4, 50, generator=g).cuda()
    adv = torch.randn(4, generator=g).cuda()
    e, c, _, t, g = head(200, 64, 300, torch.bfloat16, 62)
    tlp, ids = (v.cuda() for v in teacher(e, c, None, 4, g))
    e, c, t = e.cuda(), c.cuda(), t.cuda()
    return [("policy", lambda v: mlx_cce.policy_loss(v * 1.5, old, adv) * 2, x),
            ("preference", lambda v: mlx_cce.preference_loss(v * 1.5, old) * 2, x),
            ("log_probs", lambda v: mlx_cce.linear_log_probs(v * 1.5, c, t).sum() * 2, e),
            ("linear_policy", lambda v: mlx_cce.linear_policy_loss((v * 1.5).view(4, 50, 64), c, t.view(4, 50), old, adv) * 2,
             e),
            ("linear_preference", lambda v: mlx_cce.linear_preference_loss((v * 1.5).view(4, 50, 64), c, t.view(4, 50)) * 2,
             e),
            ("distillation", lambda v: mlx_cce.linear_distillation_loss(v * 1.5, c, ids, tlp) * 2, e)]


@pytest.mark.parametrize("k", range(6))
def test_compiled_functions_break_their_graph_at_the_losses(k):
    _, f, x = _transformed()[k]
    out = []
    for fn in (f, torch.compile(f, backend="aot_eager")):
        torch._dynamo.reset()
        y = x.clone().requires_grad_(True)
        loss = fn(y)
        out.append((loss.detach(), torch.autograd.grad(loss, [y])[0]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    torch._dynamo.reset()
    with pytest.raises(Exception, match="traced graph|Observed exception"):
        torch.compile(f, backend="eager", fullgraph=True)(x)
    torch._dynamo.reset()


@pytest.mark.parametrize("k", range(6))
def test_traces_and_transforms_are_refused_or_right(k):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    _, f, x = _transformed()[k]
    with pytest.raises(RuntimeError, match="cannot be traced"):  # (a trace would hold buffers and no kernel)
        make_fx(f)(x)
    xs = torch.stack([x, 0.5 * x])
    assert torch.equal(torch.func.vmap(f)(xs), torch.stack([f(v) for v in xs]))  # (one call for each)
    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.grad(f)(x)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp is not implemented"):
        f(forward_ad.make_dual(x, torch.ones_like(x)))
    y = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="one gradient at a time"):
        torch.autograd.grad(f(y), [y], torch.ones(2, device="cuda"), is_grads_batched=True)
    _ext.device_status()


# ---------------------------------------------------------------------------
# the tensor cores' rounding towards zero
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_drift_of_a_large_logit(dtype):
    """The mean error of log-probabilities beside a logit of 14, which one accumulator
    would leave 7e-5 off (test_the_drift_bound_tells_one_accumulator_from_several)."""
    e, c, peak, target = drift_inputs(dtype)
    lp = mlx_cce.linear_log_probs(e.cuda(), c.cuda(), target.cuda()).cpu().double()
    want = torch.log_softmax(e.double() @ c.double().t(), 1).gather(1, target[:, None])[:, 0]
    err = float((lp - want).mean())
    assert abs(err) < drift_bound(e, c, peak, target, *SEGMENTS[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("place", ["first", "last"])
def test_drift_of_a_logit_that_one_channel_carries(place, dtype):
    """A logit of 14 in the first step of its segment is cut in each of the S steps that
    follow, half a last place, 2^-21, each on average; in the last step it is cut
    once.  k 2^-23 of it are added back for both: a mean error in between."""
    seg, k = SEGMENTS[dtype]
    steps = seg // 16
    g = torch.Generator().manual_seed(6)
    N, D, V = 256, 2048, 512
    e = torch.randn(N, D, generator=g)
    c = torch.randn(V, D, generator=g) * D ** -0.5
    ch = 3 * seg + (0 if place == "first" else seg - 1)
    c[:, ch] = 0.0
    e[:, ch], c[0, ch] = 7.0, 2.0
    e, c = e.to(dtype), c.to(dtype)
    target = torch.arange(N) % (V - 1) + 1
    z = e.double() @ c.double().t()
    e, z = e[z[:, 0] > 8.5], z[z[:, 0] > 8.5]  # (one binade)
    e, z = e[z[:, 0] < 15.5], z[z[:, 0] < 15.5]
    target = target[:len(e)]
    lp = mlx_cce.linear_log_probs(e.cuda(), c.cuda(), target.cuda()).cpu().double()
    err = float((lp - torch.log_softmax(z, 1).gather(1, target[:, None])[:, 0]).mean())
    back = k * 2.0 ** -23 * 14
    # (the error of the log-sum-exp, negated: what was added back and what was cut, to
    # an eighth, and 2^-20 for everything after the sum)
    assert -1.125 * back - 2.0 ** -20 <= err <= 1.125 * (steps * 2.0 ** -21 - back) + 2.0 ** -20
