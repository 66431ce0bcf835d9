"""GPU tests of the losses on a head's log-probabilities at the edges of their range:
NaN and infinite operands, values of very different sizes, shapes that could be read
two ways, failing calls.  Tolerances are those of ``test_linear_losses_gpu``."""

import math

import pytest
import torch

import mlx_cce
import token_loss_ref as R
from mlx_cce import _ext
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
