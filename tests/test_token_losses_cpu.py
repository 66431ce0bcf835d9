"""Argument checks of the policy and preference losses (no kernel runs)."""

import ctypes

import pytest
import torch

import mlx_cce
import token_loss_ref as R
from mlx_cce import _ext, losses


def test_cpu_tensors_and_types_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mlx_cce.policy_loss(x, x, torch.ones(4))
    with pytest.raises(ValueError, match="CUDA tensor"):
        mlx_cce.preference_loss(x, x)
    with pytest.raises(ValueError, match="unsupported dtype"):
        mlx_cce.policy_loss(x.double(), x, torch.ones(4))


@pytest.mark.parametrize("kw,match", [
    (dict(clip=-0.1), "clip"), (dict(clip=1.5), "clip"), (dict(clip_high=-1.0), "clip"), (dict(clip=float("nan")), "clip"),
    (dict(dual_clip=1.0), "dual_clip"), (dict(kl_coef=float("nan")), "kl_coef"), (dict(reduction="avg"), "reduction")])
def test_policy_parameters(kw, match):
    args = dict(clip=0.2, clip_high=None, dual_clip=None, kl_coef=0.0, reduction="mean", per_token=True)
    losses._policy_params("t", **args)
    with pytest.raises(ValueError, match=match):
        losses._policy_params("t", **{**args, **kw})


@pytest.mark.parametrize("kw,match", [
    (dict(beta=0.0), "beta"), (dict(beta=float("inf")), "beta"), (dict(margin=float("nan")), "margin"),
    (dict(loss_type="dpo"), "loss_type"), (dict(label_smoothing=0.6), "label_smoothing"),
    (dict(loss_type="hinge", label_smoothing=0.1), "label_smoothing"), (dict(loss_type="ipo", margin=1.0), "margin"),
    (dict(reduction="sequence"), "reduction")])
def test_preference_parameters(kw, match):
    args = dict(beta=0.1, margin=0.0, loss_type="sigmoid", label_smoothing=0.0, length_normalize=False,
                reduction="mean")
    losses._preference_params("t", **args)
    with pytest.raises(ValueError, match=match):
        losses._preference_params("t", **{**args, **kw})


def test_shapes():
    dev = torch.device("cpu")
    cu = torch.tensor([0, 3, 8])
    assert losses._sequences("t", (8,), cu, dev)[0] == 2
    assert losses._sequences("t", (8,), cu, dev)[1].dtype == torch.int32
    assert losses._sequences("t", (4, 8), None, dev) == (4, None)
    assert losses._sequences("t", (8,), None, dev) == (1, None)
    for shape, c in (((4, 8), cu), ((2, 2, 2), None), ((8,), cu.float()), ((8,), cu[None]), ((8,), cu[:0])):
        with pytest.raises(ValueError):
            losses._sequences("t", shape, c, dev)
    with pytest.raises(ValueError, match="even number"):
        losses._pairs("t", (8,), torch.tensor([0, 1, 2, 3]), dev)
    with pytest.raises(ValueError, match="2 pairs"):
        losses._pairs("t", (8,), None, dev)
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="per token"):
        losses._advantages("t", torch.zeros(8), (4, 8), 4, dev)
    with pytest.raises(ValueError, match="floating"):
        losses._advantages("t", torch.zeros(4, dtype=torch.int64), (4, 8), 4, dev)
    assert losses._advantages("t", torch.zeros(4), (4, 8), 4, dev)[1] is False
    assert losses._advantages("t", torch.zeros(4, 8).half(), (4, 8), 4, dev)[0].dtype == torch.float32
    with pytest.raises(ValueError, match="shape"):
        losses._per_token("t", "old_logp", torch.zeros(8), x)
    with pytest.raises(ValueError, match="dtype"):
        losses._per_token("t", "old_logp", x.half(), x)
    with pytest.raises(ValueError, match="bool"):
        losses._mask("t", x, x.shape, dev)
    with pytest.raises(ValueError, match="shape"):
        losses._mask("t", x[0] > 0, x.shape, dev)
    with pytest.raises(ValueError, match="per sequence"):
        losses._reference("t", torch.zeros(3), x, x.dtype, 4)


def test_abi_refusals():
    lib = _ext.lib
    p = _ext.CcePolicyParams(0.2, 0.2, 0.0, 0.0, 0, 0)
    ok = [None, None, None, 0, None, None, None, 8, 2, ctypes.byref(p), None, None, None, None, None, 0, None]

    def call(**at):
        a = list(ok)
        for k, v in at.items():
            a[int(k[1:])] = v
        return lib.cce_policy_loss_forward(*a)

    assert call(_3=9) == _ext.CCE_ERR_DTYPE
    assert call(_7=-1) == _ext.CCE_ERR_SHAPE
    assert call(_8=3) == _ext.CCE_ERR_SHAPE  # 8 tokens are not 3 rows
    assert call(_9=None) == _ext.CCE_ERR_ARG
    assert call() == _ext.CCE_ERR_ARG  # NULL outputs
    for bad in (_ext.CcePolicyParams(1.5, 0.2, 0.0, 0.0, 0, 0), _ext.CcePolicyParams(0.2, -0.1, 0.0, 0.0, 0, 0),
                _ext.CcePolicyParams(0.2, 0.2, 0.5, 0.0, 0, 0), _ext.CcePolicyParams(0.2, 0.2, 0.0, 0.0, 7, 0)):
        assert call(_9=ctypes.byref(bad)) == _ext.CCE_ERR_ARG
    assert lib.cce_policy_loss_backward(None, None, None, 9, None, 8, 2, 0, None, None) == _ext.CCE_ERR_ARG
    assert lib.cce_policy_loss_backward(None, None, None, 0, None, 8, 2, 0, None, None) == _ext.CCE_ERR_ARG
    q = _ext.CcePreferenceParams(0.1, 0.0, 0.0, 0, 0, 0)
    args = [None, None, 0, None, None, None, 8, 2, ctypes.byref(q), None, None, None, None, 0, None]
    assert lib.cce_preference_loss_forward(*args) == _ext.CCE_ERR_ARG
    args[7] = 3
    assert lib.cce_preference_loss_forward(*args) == _ext.CCE_ERR_SHAPE
    args[7] = -1
    assert lib.cce_preference_loss_forward(*args) == _ext.CCE_ERR_SHAPE
    args[7] = 2
    for bad in (_ext.CcePreferenceParams(0.0, 0.0, 0.0, 0, 0, 0), _ext.CcePreferenceParams(0.1, 0.0, 0.7, 0, 0, 0),
                _ext.CcePreferenceParams(0.1, 0.0, 0.0, 3, 0, 0), _ext.CcePreferenceParams(0.1, 0.0, 0.0, 0, 2, 0)):
        args[8] = ctypes.byref(bad)
        assert lib.cce_preference_loss_forward(*args) == _ext.CCE_ERR_ARG
    assert lib.cce_preference_loss_backward(None, None, 2, None, None, 8, 2, 0, None, None) == _ext.CCE_ERR_ARG
    assert lib.cce_token_loss_workspace_bytes(500000, 12) > lib.cce_token_loss_workspace_bytes(1000, 12) > 0


def test_definitions_against_differences():
    """The tests' own 64-bit gradients against central differences (error h^2)."""
    g = torch.Generator().manual_seed(1)
    x = -torch.rand(60, generator=g).double() * 3
    old, ref = x + 0.2 * torch.randn(60, generator=g), x + 0.3 * torch.randn(60, generator=g)
    adv, cu, mask = torch.randn(4, generator=g), [2, 20, 20, 45, 57], torch.rand(60, generator=g) < 0.8
    fs = [lambda v: R.policy(v, old, adv, ref, mask, cu, kl_coef=0.3, dual_clip=1.3, reduction="sequence"),
          lambda v: R.preference(v, ref, mask, cu, beta=0.5, length_normalize=True),
          lambda v: R.preference(v, ref, mask, cu, loss_type="ipo")]
    h = 1e-5
    for f in fs:
        grad = f(x)["grad"]
        for k in range(0, 60, 7):
            d = torch.zeros_like(x)
            d[k] = h
            diff = (f(x + d)["loss"] - f(x - d)["loss"]) / (2 * h)
            assert abs(float(diff - grad[k])) < 1e-7 * (1 + abs(float(grad[k])))
