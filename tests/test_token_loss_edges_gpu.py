"""GPU tests of the policy loss at the edges of its range, with the tolerances and the
64-bit definition of ``test_token_losses_gpu``."""

import pytest
import torch

import mlx_cce
import token_loss_ref as R
from test_token_losses_gpu import DTYPES, EPS, batch, run_policy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_log_probability_without_old_is_not_hidden(dtype):
    """The ratio is 1 by definition there, but a NaN that counts shows in loss and gradient."""
    x = torch.full((300,), -1.0, dtype=dtype, device="cuda")
    x[[5, 200]] = float("nan")
    x.requires_grad_(True)
    adv = torch.tensor([1.0, -1.0], device="cuda")
    cu = torch.tensor([0, 100, 300], device="cuda")
    loss = mlx_cce.policy_loss(x, None, adv, cu_seqlens=cu, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), [x])
    for t in (loss, grad):
        assert torch.equal(torch.isnan(t).nonzero()[:, 0].cpu(), torch.tensor([5, 200]))
    assert torch.isnan(mlx_cce.policy_loss(x, None, adv, cu_seqlens=cu))
    mask = ~torch.isnan(x)
    assert torch.isfinite(mlx_cce.policy_loss(x, None, adv, mask=mask, cu_seqlens=cu))


@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum", "none"])
def test_an_advantage_of_zero_with_any_ratio(reduction):
    """Ratios of e^100 and e^700, past float32: a group whose rewards are all the same has
    advantages of 0, and 0 of any ratio is 0."""
    b = batch(2000, 4, seed=21)
    b["old"][::7] = b["logp"][::7] - 100.0
    b["old"][3::7] = b["logp"][3::7] - 700.0
    adv = torch.randn(b["shape"], generator=b["g"])
    adv[::7] = adv[3::7] = 0.0
    go = torch.randn(b["shape"], generator=b["g"]) if reduction == "none" else None
    kw = dict(kl_coef=0.1, reduction=reduction)
    loss, grad, _, _ = run_policy(b, adv, go, **kw)
    r = R.policy(b["logp"], b["old"], adv, b["ref"], b["mask"], b["cu"], grad_out=go, **kw)
    assert torch.all((loss - r["loss"]).abs() <= EPS * r["lsize"])
    # check_policy's tolerance, and where only the KL term is left the definition's own rounding:
    # its autograd forms the slope e^q - 1 as (expm1(q) + 1) - 1, off by 2^-53 in 64 bits, times
    # kl_coef and a token's weight
    n = torch.tensor([int(b["mask"][lo:hi].sum()) for lo, hi in zip(b["cu"], b["cu"][1:])])
    n = n[n > 0]
    weight = {"mean": 1 / int(n.sum()), "sequence": 1 / (len(n) * int(n.min())), "sum": 1.0}.get(reduction)
    weight = weight or float(go.abs().max())
    assert torch.all((grad.double() - r["grad"]).abs() <= EPS * r["gsize"] + 2.0 ** -52 * 0.1 * weight)
    x = b["logp"].cuda()
    x[14] = float("nan")  # (not hidden by the advantage)
    mask = torch.ones_like(b["mask"]).cuda()
    assert torch.isnan(mlx_cce.policy_loss(x, b["old"].cuda(), adv.cuda(), mask=mask))


@pytest.mark.parametrize("reduction", ["mean", "sequence", "sum", "none"])
def test_a_kl_term_of_weight_zero_is_only_measured(reduction):
    """ref - logp of 100: e^100 is past float32, 0 times it is 0 all the same."""
    b = batch(2000, 4, seed=22)
    b["mask"][:] = True
    far = b["logp"] - 100.0
    near = b["ref"].clone()
    adv = torch.randn(4, generator=b["g"])
    cu = torch.tensor(b["cu"], dtype=torch.int32, device="cuda")
    out = []
    for x, ref in ((b["logp"], near), (far, b["logp"])):
        x = x.cuda().requires_grad_(True)
        old = x.detach() + 0.01
        loss, stats = mlx_cce.policy_loss(x, old, adv.cuda(), ref_logp=ref.cuda(), cu_seqlens=cu, reduction=reduction,
                                          return_stats=True)
        bare = mlx_cce.policy_loss(x, old, adv.cuda(), cu_seqlens=cu, reduction=reduction)
        grads = [torch.autograd.grad(l.sum(), [x])[0] for l in (loss, bare)]
        assert torch.isfinite(loss).all() and torch.equal(loss, bare) and torch.equal(*grads)
        out.append(stats.kl.item())
    assert 0 < out[0] < 10 and out[1] == float("inf")


def test_as_many_tokens_as_sequences():
    """Per sequence when asked: the values of the same batch with one token more, where
    the shape says it."""
    g = torch.Generator().manual_seed(31)
    logp, old = -torch.rand(4, generator=g).cuda(), -torch.rand(4, generator=g).cuda()
    val = torch.randn(4, generator=g).cuda()
    cu = torch.tensor([0, 2, 2, 3, 4], device="cuda")
    more = lambda t: torch.cat([t, t.new_zeros(1)])
    got = mlx_cce.policy_loss(logp, old, val, cu_seqlens=cu, reduction="none", advantages_per_token=False)
    want = mlx_cce.policy_loss(more(logp), more(old), val, cu_seqlens=cu, reduction="none")
    assert torch.equal(got, want[:4])
    token = mlx_cce.policy_loss(logp, old, val, cu_seqlens=cu, reduction="none", advantages_per_token=True)
    assert not torch.equal(got, token)
    with pytest.warns(UserWarning, match="per token"):
        assert torch.equal(mlx_cce.policy_loss(logp, old, val, cu_seqlens=cu, reduction="none"), token)
    got = mlx_cce.preference_loss(logp, val, cu_seqlens=cu, reduction="none", ref_per_token=False)
    want = mlx_cce.preference_loss(more(logp), val, cu_seqlens=cu, reduction="none")
    assert torch.equal(got, want)
    e, c = torch.randn(4, 64, generator=g).bfloat16().cuda(), torch.randn(90, 64, generator=g).bfloat16().cuda()
    t = torch.tensor([3, 50, 7, 89], device="cuda")
    lp = mlx_cce.linear_log_probs(e, c, t)
    assert torch.equal(mlx_cce.linear_policy_loss(e, c, t, old, val, cu_seqlens=cu, advantages_per_token=False),
                       mlx_cce.policy_loss(lp, old, val, cu_seqlens=cu, advantages_per_token=False))
    assert torch.equal(mlx_cce.linear_preference_loss(e, c, t, val, cu_seqlens=cu, ref_per_token=False),
                       mlx_cce.preference_loss(lp, val, cu_seqlens=cu, ref_per_token=False))
