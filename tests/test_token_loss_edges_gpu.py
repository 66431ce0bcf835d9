"""GPU tests of the policy loss at the edges of its range, with the tolerances and the
64-bit definition of ``test_token_losses_gpu``."""

import pytest
import torch

import mlx_cce
from test_token_losses_gpu import DTYPES, batch, check_policy

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
