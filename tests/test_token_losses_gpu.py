"""GPU tests of the policy and preference losses against their 64-bit definitions.

Tolerances.  A half step of float32 is u = 2^-24.  A token's term is built from
d (rounded once: |d| u on the ratio, |d| <= 4 here), expf (2 ulp = 4 u), the
product with A (u) and the KL term: expm1f (1 ulp = 2 u), at most four times
more after the subtraction of q, its weight and the sum (2 u).  That is at most
16 u of the terms' magnitudes; sums are held in 64 bits and rounded once (u).
Gradients carry the same terms and three more products (weight, upstream,
sequence weight).  EPS = 2^-19 = 32 u covers both.  A gradient of a smaller
type is rounded once more, by half a step of it.
"""

import pytest
import torch

import mlx_cce
import token_loss_ref as R

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -19
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
REDUCTIONS = ["mean", "sequence", "sum", "none"]


def near(x, g, width):
    return torch.clamp(x + width * torch.randn(x.shape, generator=g), max=0.0, min=-8.0)


def batch(n, S, seed, dtype=torch.float32, packed=True, first=0, last=0):
    g = torch.Generator().manual_seed(seed)
    shape = (n,) if packed else (S, n // S)
    n = n if packed else n // S * S
    logp = -(torch.rand(n, generator=g) ** 4 * 6).view(shape)
    old = near(logp, g, 0.3)
    ref = near(logp, g, 0.5)
    mask = torch.rand(shape, generator=g) < 0.7
    cu = R.cuts(n, S, g, first, last) if packed else None
    return dict(logp=logp.to(dtype), old=old.to(dtype), ref=ref.to(dtype), mask=mask, cu=cu, g=g, shape=shape, S=S)


def cuda_cu(cu):
    return None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")


def run_policy(b, adv, grad_out=None, **kw):
    dev = "cuda"
    x = b["logp"].to(dev).requires_grad_(True)
    old, ref = b["old"], b["ref"]
    loss, stats = mlx_cce.policy_loss(x, None if old is None else old.to(dev), adv.to(dev),
                                      ref_logp=None if ref is None else ref.to(dev),
                                      mask=None if b["mask"] is None else b["mask"].to(dev), cu_seqlens=cuda_cu(b["cu"]),
                                      return_stats=True, **kw)
    (grad,) = torch.autograd.grad(loss, [x], None if grad_out is None else grad_out.to(dev))
    assert grad.dtype == x.dtype and loss.dtype == torch.float32
    return loss.detach().cpu().double(), grad.cpu(), stats.kl.item(), stats.clip_fraction.item()


def check_policy(b, adv, grad_out=None, **kw):
    loss, grad, kl, cf = run_policy(b, adv, grad_out, **kw)
    r = R.policy(b["logp"], b["old"], adv, b["ref"], b["mask"], b["cu"], grad_out=grad_out, **kw)
    assert loss.shape == r["loss"].shape
    assert torch.all((loss - r["loss"]).abs() <= EPS * r["lsize"] + 1e-37)
    tol = EPS * r["gsize"] + R.half_steps(grad.dtype, r["grad"]) * (grad.dtype != torch.float32)
    bad = (grad.double() - r["grad"]).abs() > tol + 1e-37
    assert not bad.any(), (grad[bad][:4], r["grad"][bad][:4])
    assert abs(kl - float(r["kl"])) <= EPS * float(r["kl"])
    assert abs(cf - float(r["clip_fraction"])) <= 2.0 ** -23
    return grad


@pytest.mark.parametrize("reduction", REDUCTIONS)
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("n,S", [(1, 1), (5, 2), (1023, 7), (1024, 1), (1025, 4), (2048, 2), (5003, 40), (70001, 3)])
def test_policy_sizes(n, S, packed, reduction):
    b = batch(n, S, seed=n + S, packed=packed)
    adv = torch.randn(S, generator=b["g"])
    go = torch.randn(b["shape"], generator=b["g"]) if reduction == "none" else None
    check_policy(b, adv, go, kl_coef=0.05, reduction=reduction)


@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_policy_large_batch(reduction):
    """Enough tokens for blocks of four steps; sequences longer and shorter than a block."""
    n = 2 * 148 * 8 * 1024 + 1500
    b = batch(n, 37, seed=77, first=3, last=5000)
    b["cu"][5] = b["cu"][4] + 1 if b["cu"][4] + 1 <= b["cu"][6] else b["cu"][5]
    adv = torch.randn(37, generator=b["g"])
    go = torch.randn(b["shape"], generator=b["g"]) if reduction == "none" else None
    check_policy(b, adv, go, kl_coef=0.05, reduction=reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_policy_types_and_token_advantages(dtype, reduction):
    b = batch(3001, 9, seed=3, dtype=dtype, first=17, last=600)
    adv = torch.randn(b["shape"], generator=b["g"])
    go = torch.randn(b["shape"], generator=b["g"]) if reduction == "none" else torch.tensor(3.0)
    grad = check_policy(b, adv, go, kl_coef=0.1, reduction=reduction)
    assert torch.all(grad[:17] == 0) and torch.all(grad[-600:] == 0)  # tokens of no sequence


@pytest.mark.parametrize("kw", [dict(clip=0.1, clip_high=0.4), dict(clip=0.0), dict(clip=1.0, clip_high=R.INF),
                                dict(dual_clip=1.5), dict(dual_clip=3.0, clip_high=0.0), dict(kl_coef=-0.2)])
def test_policy_clips(kw):
    b = batch(4099, 6, seed=11)
    adv = torch.randn(b["shape"], generator=b["g"])
    adv[::50] = 0.0
    check_policy(b, adv, **kw)


def test_policy_on_its_own_samples_and_without_reference():
    b = batch(2500, 5, seed=12)
    b["old"] = b["ref"] = b["mask"] = None
    check_policy(b, torch.randn(5, generator=b["g"]), reduction="sequence")


def test_policy_border_is_decided_exactly():
    """Tokens whose ratio is a few 64-bit steps beside the border: each has its own side's gradient."""
    import math
    hi, lo = math.log(1.2), math.log(0.8)
    old = -torch.rand(4000, generator=torch.Generator().manual_seed(0)) * 3 - 1
    d = torch.tensor([hi, lo], dtype=torch.float64).repeat(2000)
    logp = (old.double() + d).float()          # off the border by the rounding of logp alone
    adv = torch.tensor([1.0, -1.0]).repeat(2000)
    b = dict(logp=logp, old=old, ref=None, mask=None, cu=None, shape=logp.shape)
    grad = check_policy(b, adv, reduction="sum")
    assert 500 < int((grad == 0).sum()) < 3500  # both sides occur


@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_policy_masked_values_are_not_used(reduction):
    b = batch(3000, 6, seed=5)
    off = ~b["mask"]
    for name, bad in (("logp", -R.INF), ("old", R.NAN), ("ref", R.INF)):
        b[name] = torch.where(off, torch.full_like(b[name], bad), b[name])
    adv = torch.randn(3000, generator=b["g"])
    adv = torch.where(off, torch.full_like(adv, R.NAN), adv)
    go = torch.where(off, R.INF, 1.0).float() if reduction == "none" else None
    clean = dict(b, **{k: torch.where(off, torch.zeros_like(b[k]), b[k]) for k in ("logp", "old", "ref")})
    loss, grad, _, _ = run_policy(b, adv, go, kl_coef=0.1, reduction=reduction)
    adv0 = torch.where(off, torch.zeros_like(adv), adv)
    go0 = None if go is None else torch.where(off, torch.zeros_like(go), go)
    want = run_policy(clean, adv0, go0, kl_coef=0.1, reduction=reduction)
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
    assert torch.all(grad[off] == 0)


@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_policy_without_tokens(reduction):
    b = batch(700, 3, seed=6)
    b["mask"] = torch.zeros(700, dtype=torch.bool)
    adv = torch.ones(3)
    go = torch.ones(700) if reduction == "none" else None
    loss, grad, kl, cf = run_policy(b, adv, go, reduction=reduction, kl_coef=1.0)
    assert torch.all(loss == 0) and torch.all(grad == 0) and kl == 0 and cf == 0
    empty = dict(logp=torch.zeros(0), old=torch.zeros(0), ref=None, mask=None, cu=[0, 0, 0], shape=(0,))
    loss, grad, _, _ = run_policy(empty, torch.ones(2), torch.ones(0) if reduction == "none" else None,
                                  reduction=reduction)
    assert float(loss.sum()) == 0 and grad.numel() == 0


def test_policy_nan_in_a_token_that_counts_shows():
    b = batch(100, 2, seed=7)
    b["mask"] = None
    b["logp"][3] = R.NAN
    loss, _, _, _ = run_policy(b, torch.ones(2))
    assert torch.isnan(loss)


def test_policy_strided_and_unaligned_inputs():
    b = batch(5000, 8, seed=8)
    adv = torch.randn(5000, generator=b["g"])
    want = run_policy(b, adv, kl_coef=0.1)
    dev = "cuda"

    def odd(t):  # contiguous, but 1 element behind an aligned address
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)
        buf[1:].copy_(t)
        return buf[1:]

    def wide(t):  # every second element of a wider tensor
        buf = torch.empty(t.numel(), 2, dtype=t.dtype, device=dev)
        buf[:, 0].copy_(t)
        return buf[:, 0]

    for f in (odd, wide):
        x = f(b["logp"]).detach().requires_grad_(True)
        loss = mlx_cce.policy_loss(x, f(b["old"]), f(adv), ref_logp=f(b["ref"]), mask=f(b["mask"]),
                                   cu_seqlens=f(torch.tensor(b["cu"], dtype=torch.int32)), kl_coef=0.1)
        (grad,) = torch.autograd.grad(loss, [x])
        # (block sums are the same whichever way a block's values were loaded)
        assert float(loss) == float(want[0]) and torch.equal(grad.cpu(), want[1])


def test_policy_gradient_against_differences():
    """Central differences of the kernel's own per-token loss, away from the
    clipping borders: error h^2/6 |l'''| + rounding 2 EPS |l| / (2 h)."""
    g = torch.Generator().manual_seed(9)
    x = -torch.rand(512, generator=g) - 0.5
    old = x + 0.05 * torch.randn(512, generator=g)
    ref = x + 0.3 * torch.randn(512, generator=g)
    adv = torch.randn(512, generator=g)
    h = 2.0 ** -7

    def f(v):
        return mlx_cce.policy_loss(v, old.cuda(), adv.cuda(), ref_logp=ref.cuda(), clip=0.5, kl_coef=0.2,
                                   reduction="none")

    xc = x.cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(f(xc).sum(), [xc])
    with torch.no_grad():
        diff = ((f(xc + h).double() - f(xc - h).double()) / (2 * h)).cpu()
    mag = 2.0 * (adv.abs() * 1.5 + 1.0)  # bounds |l| and |l'''|: r < 1.5, e^q < 4
    assert torch.all((diff - grad.cpu().double()).abs() <= mag * (h * h / 6 + 2 * EPS / (2 * h)))


def test_policy_results_do_not_change_between_runs():
    b = batch(300001, 500, seed=13)
    adv = torch.randn(500, generator=b["g"])
    a = run_policy(b, adv, kl_coef=0.1, reduction="sequence")
    for _ in range(3):
        c = run_policy(b, adv, kl_coef=0.1, reduction="sequence")
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


# ---------------------------------------------------------------------------
# preference loss
# ---------------------------------------------------------------------------

def run_preference(b, ref, grad_out=None, **kw):
    dev = "cuda"
    x = b["logp"].to(dev).requires_grad_(True)
    loss, rew = mlx_cce.preference_loss(x, None if ref is None else ref.to(dev),
                                        mask=None if b["mask"] is None else b["mask"].to(dev),
                                        cu_seqlens=cuda_cu(b["cu"]), return_rewards=True, **kw)
    (grad,) = torch.autograd.grad(loss, [x], None if grad_out is None else grad_out.to(dev))
    assert grad.dtype == x.dtype and loss.dtype == torch.float32
    return loss.detach().cpu().double(), grad.cpu(), rew.chosen.cpu().double(), rew.rejected.cpu().double()


def check_preference(b, ref, grad_out=None, **kw):
    loss, grad, chosen, rejected = run_preference(b, ref, grad_out, **kw)
    r = R.preference(b["logp"], ref, b["mask"], b["cu"], grad_out=grad_out, **kw)
    beta = kw.get("beta", 0.1)
    P = r["gap"].numel()
    # D: a rounding u per token difference, then 64 bits; rewards rounded once
    u = 2.0 ** -24
    dD = u * r["dsize"]
    dgap = dD[:P] + dD[P:]
    assert torch.all((chosen - r["chosen"]).abs() <= beta * dD[:P] + 2 * u * r["chosen"].abs() + 1e-37)
    assert torch.all((rejected - r["rejected"]).abs() <= beta * dD[P:] + 2 * u * r["rejected"].abs() + 1e-37)
    # the loss's slope by gap is at most beta (sigmoid, hinge) or 2 |gap - 1/(2 beta)|
    slope = 2 * (r["gap"] - 0.5 / beta).abs() + 2 * dgap if kw.get("loss_type") == "ipo" else torch.full((P,), beta)
    err = slope * dgap + 2 * u * r["pairs"].abs()
    red = kw.get("reduction", "mean")
    total = err if red == "none" else err.sum() / (P if red == "mean" else 1) + 2 * u * r["loss"].abs()
    assert torch.all((loss - r["loss"]).abs() <= total + 1e-37)
    # the gradient: the slope's own change by dgap (its derivative: beta^2 / 4, or 2) and roundings
    curve = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kw.get("loss_type", "sigmoid")]
    seq, S = R.token_sequences(b["logp"].shape, b["cu"])
    scale = torch.ones(P, dtype=torch.float64) if grad_out is None else grad_out.double().abs() * torch.ones(P)
    change = (curve * dgap * scale / (P if red == "mean" else 1)).repeat(2)[seq.clamp(min=0)].view(b["logp"].shape)
    tol = change + 4 * u * r["grad"].abs() + R.half_steps(grad.dtype, r["grad"]) * (grad.dtype != torch.float32)
    bad = (grad.double() - r["grad"]).abs() > tol + 1e-37
    assert not bad.any(), (grad[bad][:4], r["grad"][bad][:4])
    return grad


@pytest.mark.parametrize("loss_type", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("n,pairs", [(2, 1), (64, 4), (1024, 1), (1025, 3), (4097, 70), (90001, 2)])
def test_preference_sizes(n, pairs, packed, loss_type):
    b = batch(n, 2 * pairs, seed=n + pairs, packed=packed)
    check_preference(b, b["ref"], loss_type=loss_type)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_preference_large_batch(dtype):
    b = batch(2 * 148 * 8 * 1024 + 1500, 2 * 301, seed=78, dtype=dtype, first=9, last=4000)
    check_preference(b, b["ref"], loss_type="ipo", beta=0.01)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_preference_types(dtype, reduction):
    b = batch(6007, 22, seed=21, dtype=dtype, first=5, last=900)
    go = torch.randn(11, generator=b["g"]) if reduction == "none" else torch.tensor(-2.0)
    grad = check_preference(b, b["ref"], go, reduction=reduction, beta=0.3)
    assert torch.all(grad[:5] == 0) and torch.all(grad[-900:] == 0)


@pytest.mark.parametrize("kw", [dict(label_smoothing=0.2), dict(margin=0.7), dict(length_normalize=True, beta=2.0),
                                dict(length_normalize=True, loss_type="ipo"), dict(beta=5.0)])
def test_preference_options(kw):
    b = batch(3003, 10, seed=22)
    check_preference(b, b["ref"], **kw)


def test_preference_reference_sums_and_none():
    b = batch(3003, 10, seed=23)
    check_preference(b, None, beta=0.01)
    check_preference(b, torch.randn(10, generator=b["g"]) * 30 - 100, beta=0.01)


def test_preference_masked_values_and_empty_sides():
    b = batch(2000, 8, seed=24)
    off = ~b["mask"]
    off[b["cu"][0]:b["cu"][1]] = True  # a chosen sequence without a token that counts
    b["mask"] = ~off
    clean = dict(b)
    want = check_preference(clean, b["ref"])
    bad = dict(b, logp=torch.where(off, torch.full_like(b["logp"], -R.INF), b["logp"]))
    ref = torch.where(off, torch.full_like(b["ref"], R.NAN), b["ref"])
    assert torch.equal(run_preference(bad, ref)[1], want)
    nothing = dict(b, mask=torch.zeros(2000, dtype=torch.bool))
    loss, grad, chosen, _ = run_preference(nothing, b["ref"])
    assert abs(float(loss) - 0.6931471805599453) < 1e-7 and torch.all(grad == 0) and torch.all(chosen == 0)


def test_preference_empty_batches():
    dev = "cuda"
    x = torch.zeros(0, device=dev, requires_grad=True)
    cu = torch.zeros(81, dtype=torch.int32, device=dev)  # 40 pairs, no token: two launches' sizes
    loss = mlx_cce.preference_loss(x, x.detach(), cu_seqlens=cu)
    loss.backward()
    assert abs(float(loss) - 0.6931471805599453) < 1e-7 and x.grad.numel() == 0
    y = torch.randn(5, device=dev, requires_grad=True)
    loss = mlx_cce.preference_loss(y, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=dev))  # no pair
    loss.backward()
    assert float(loss) == 0 and torch.all(y.grad == 0)


# ---------------------------------------------------------------------------
# streams, graphs, several calls at once
# ---------------------------------------------------------------------------

def test_calls_on_two_streams_at_once():
    bs = [batch(200000 + 7 * k, 50, seed=30 + k) for k in range(2)]
    advs = [torch.randn(50, generator=b["g"]) for b in bs]
    want = [run_policy(b, a, kl_coef=0.1, reduction="sequence") for b, a in zip(bs, advs)]
    dev = "cuda"
    ins = [(b["logp"].to(dev), b["old"].to(dev), a.to(dev), b["ref"].to(dev), b["mask"].to(dev), cuda_cu(b["cu"]))
           for b, a in zip(bs, advs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, old, adv, ref, mask, cu = ins[k]
                x = x.detach().requires_grad_(True)
                loss = mlx_cce.policy_loss(x, old, adv, ref_logp=ref, mask=mask, cu_seqlens=cu, kl_coef=0.1,
                                           reduction="sequence")
                got[k].append((loss.detach(), torch.autograd.grad(loss, [x])[0]))
    torch.cuda.synchronize()
    for k in range(2):
        for loss, grad in got[k]:
            assert float(loss) == float(want[k][0]) and torch.equal(grad.cpu(), want[k][1])


def test_captured_and_replayed():
    b = batch(50000, 20, seed=40)
    adv = torch.randn(20, generator=b["g"])
    dev = "cuda"
    x, old, ref, mask = (b[k].to(dev) for k in ("logp", "old", "ref", "mask"))
    cu, a = cuda_cu(b["cu"]), adv.to(dev)
    leaf = x.clone().requires_grad_(True)

    def step():
        p = mlx_cce.policy_loss(leaf, old, a, ref_logp=ref, mask=mask, cu_seqlens=cu, kl_coef=0.1)
        q = mlx_cce.preference_loss(leaf, ref, mask=mask, cu_seqlens=cu)
        return p, q, torch.autograd.grad(p + q, [leaf])[0]

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
    for shift in (0.0, -0.25):
        with torch.no_grad():
            leaf.copy_(x + shift)
        want = [t.detach().clone() for t in step()]
        for gr, out in graphs + graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(o.detach(), w) for o, w in zip(out, want))


def test_linear_cross_entropy_feeds_both_losses():
    """The head's log-probabilities through both losses, differentiated to the
    hidden states in one backward pass, against 64 bits."""
    g = torch.Generator().manual_seed(50)
    N, D, V = 96, 64, 500
    e, c = torch.randn(N, D, generator=g), torch.randn(V, D, generator=g) * 0.2
    t = torch.randint(0, V, (N,), generator=g)
    ref = -torch.rand(N, generator=g) * 8
    adv = torch.randn(4, generator=g)
    e64 = e.double().requires_grad_(True)
    lp64 = torch.log_softmax(e64 @ c.double().t(), 1).gather(1, t[:, None])[:, 0]
    cu = [0, 20, 50, 60, 96]
    old = lp64.detach().float() + 0.1 * torch.randn(N, generator=g)
    p = R.policy(lp64, old, adv, ref, cu=cu, kl_coef=0.02)
    q = R.preference(lp64, ref, cu=cu)
    (want,) = torch.autograd.grad((lp64 * (p["grad"] + q["grad"])).sum(), [e64])
    ec = e.cuda().requires_grad_(True)
    logp = -mlx_cce.linear_cross_entropy(ec, c.cuda(), t.cuda(), reduction="none", filter_log_eps=-float("inf"))
    loss = mlx_cce.policy_loss(logp, old.cuda(), adv.cuda(), ref_logp=ref.cuda(), cu_seqlens=cuda_cu(cu), kl_coef=0.02)
    loss = loss + mlx_cce.preference_loss(logp, ref.cuda(), cu_seqlens=cuda_cu(cu))
    loss.backward()
    # log-probabilities carry about 1e-6 (float32 logits of magnitude 5); no ratio lies so near to a border
    assert abs(float(loss) - float(p["loss"] + q["loss"])) < 1e-5
    assert torch.all((ec.grad.cpu().double() - want).abs() <= 1e-5 * want.abs().max())


def test_second_derivatives_are_an_error():
    b = batch(200, 4, seed=90)
    x = b["logp"].cuda().requires_grad_(True)
    adv = torch.ones(4, device="cuda")
    for loss in (mlx_cce.policy_loss(x, b["old"].cuda(), adv, cu_seqlens=cuda_cu(b["cu"])),
                 mlx_cce.preference_loss(x, cu_seqlens=cuda_cu(b["cu"]))):
        (plain,) = torch.autograd.grad(loss, [x], retain_graph=True)
        (grad,) = torch.autograd.grad(loss, [x], create_graph=True)
        assert torch.equal(grad.detach(), plain)
        with pytest.raises(RuntimeError, match="differentiable once"):
            grad.sum().backward()


def test_backward_twice_and_accumulation():
    """A graph kept for a second pass gives the same gradient; .grad adds up; an
    upstream gradient that is expanded, strided or of another type is taken as it is."""
    b = batch(3000, 6, seed=91)
    x = b["logp"].cuda().requires_grad_(True)
    old, adv, mask, cu = b["old"].cuda(), torch.randn(3000, generator=b["g"]).cuda(), b["mask"].cuda(), cuda_cu(b["cu"])
    loss = mlx_cce.policy_loss(x, old, adv, mask=mask, cu_seqlens=cu)
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    loss.backward()
    assert torch.equal(x.grad, first * 2)
    each = mlx_cce.policy_loss(x, old, adv, mask=mask, cu_seqlens=cu, reduction="none")
    (a,) = torch.autograd.grad(each.sum(), [x], retain_graph=True)   # an expanded scalar
    (c,) = torch.autograd.grad(each, [x], torch.ones(3000, 2, device="cuda")[:, 0], retain_graph=True)
    assert torch.equal(a, c)
    with torch.no_grad():
        again = mlx_cce.policy_loss(x, old, adv, mask=mask, cu_seqlens=cu)
    assert not again.requires_grad and torch.equal(again, loss.detach())


def test_tokens_that_are_not_finite_stay_in_their_sequence():
    b = batch(9000, 8, seed=92)
    adv = torch.ones(8, device="cuda")
    cu = cuda_cu(b["cu"])
    first, last = b["cu"][2], b["cu"][3]
    assert last - first > 3
    def run(bad):
        x = b["logp"].clone()
        x[first + 1] = bad
        x = x.cuda().requires_grad_(True)
        p = mlx_cce.policy_loss(x, b["old"].cuda(), adv, ref_logp=b["ref"].cuda(), cu_seqlens=cu, kl_coef=0.1,
                                reduction="none")
        q = mlx_cce.preference_loss(x, b["ref"].cuda(), cu_seqlens=cu, reduction="none")
        return p.detach(), q.detach(), *torch.autograd.grad(p.sum() + q.sum(), [x])
    want, got = run(-1.0), run(float("nan"))
    at = torch.arange(9000, device="cuda")
    other_tokens, other_pairs = at != first + 1, torch.arange(4, device="cuda") != 2
    outside = (at < first) | (at >= last)
    outside &= (at < b["cu"][6]) | (at >= b["cu"][7])   # (the rejected sequence of the same pair)
    assert torch.equal(got[0][other_tokens], want[0][other_tokens]) and torch.isnan(got[0][first + 1])
    assert torch.equal(got[1][other_pairs], want[1][other_pairs]) and torch.isnan(got[1][2])
    assert torch.equal(got[2][outside], want[2][outside])


def test_as_many_tokens_as_offsets_can_count():
    """2^31 - 8 tokens in two sequences: every gradient, and the sum."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    n, last = 2 ** 31 - 8, 92
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    cu = torch.tensor([0, n - last, n], dtype=torch.int32, device="cuda")
    adv = torch.tensor([1.0, -2.0], device="cuda")
    loss = mlx_cce.policy_loss(x, None, adv, cu_seqlens=cu, reduction="sum")
    (grad,) = torch.autograd.grad(loss, [x])
    assert float(loss) == float(torch.tensor(-float(n - last) + 2.0 * last))   # ratios of 1: exact in 64 bits
    assert (grad[n - last:] == 2).all()
    assert all((grad[a:min(a + (1 << 29), n - last)] == -1).all() for a in range(0, n - last, 1 << 29))
    loss = mlx_cce.preference_loss(x, cu_seqlens=cu, loss_type="hinge", beta=0.5)
    (grad,) = torch.autograd.grad(loss, [x])
    assert float(loss) == 1.0 and (grad[n - last:] == 0.5).all()
    assert all((grad[a:min(a + (1 << 29), n - last)] == -0.5).all() for a in range(0, n - last, 1 << 29))
    with pytest.raises(ValueError, match="bad sizes"):
        mlx_cce.policy_loss(torch.zeros(2 ** 31, dtype=torch.bfloat16, device="cuda"), None, adv[:1])
