"""Argument checks of the losses on a head's log-probabilities (no kernel runs)."""

import ctypes

import pytest
import torch

import mlx_cce
from mlx_cce import _ext, losses


def test_head_checks():
    e, c = torch.zeros(4, 8), torch.zeros(16, 8)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        mlx_cce.linear_log_probs(e, c, t)
    for bad, match in (((e, c, None, (5,)), "rows"), ((e, c[:, :4], None, (4,)), "must equal"),
                       ((e, c.half(), None, (4,)), "share a dtype"), ((e.double(), c.double(), None, (4,)), "dtype"),
                       ((e, c, torch.zeros(3), (4,)), "bias"), ((e, c[None], None, (4,)), "c \\[V, D\\]"),
                       ((e, c[:0], None, (4,)), "empty")):
        with pytest.raises(ValueError, match=match):
            losses._head("t", *bad)
    with pytest.raises(ValueError, match="int32 or int64"):
        losses._ids("t", "targets", e, e.device)


@pytest.mark.parametrize("kw,match", [(dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                                      (dict(reduction="sequence"), "reduction")])
def test_distill_parameters(kw, match):
    args = dict(temperature=1.0, tail=False, reduction="mean")
    losses._distill_params("t", **args)
    with pytest.raises(ValueError, match=match):
        losses._distill_params("t", **{**args, **kw})


def test_distill_shapes():
    e, c = torch.zeros(4, 8), torch.zeros(16, 8)
    ids, lp = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    with pytest.raises(ValueError, match="one shape"):
        mlx_cce.linear_distillation_loss(e, c, ids, lp[:, :2])
    with pytest.raises(ValueError, match="K must be"):
        mlx_cce.linear_distillation_loss(e, c, ids[:, :0], lp[:, :0])
    with pytest.raises(ValueError, match="K must be"):
        mlx_cce.linear_distillation_loss(e, c, ids.new_zeros(4, 1025), lp.new_zeros(4, 1025))
    with pytest.raises(ValueError, match="rows"):
        mlx_cce.linear_distillation_loss(e[:3], c, ids, lp)


def test_abi_refusals():
    lib = _ext.lib
    one = ctypes.c_void_p(256)  # never followed: every call is refused before

    def logp(N=4, D=8, V=16, dt=2, tb=8, saved=None, sb=0, ptr=one):
        return lib.cce_logp_forward(ptr, ptr, None, 0, ptr, tb, -100, 1, N, D, V, dt, ptr, ptr, saved, sb, None, 0, None)

    assert logp(dt=5) == _ext.CCE_ERR_DTYPE
    assert logp(N=-1) == logp(D=0) == logp(V=0) == _ext.CCE_ERR_SHAPE
    assert logp(V=(1 << 30) + 1) == _ext.CCE_ERR_SHAPE
    assert logp(tb=2) == logp(ptr=None) == _ext.CCE_ERR_ARG
    assert logp() == logp(saved=one, sb=100) == _ext.CCE_ERR_WORKSPACE
    assert logp(N=0) == _ext.CCE_OK
    p = _ext.CceDistillParams(1.0, 0, 0)

    def distill(N=4, K=3, dt=2, ib=8, params=p, ptr=one, loss=one):
        return lib.cce_distill_forward(ptr, ptr, None, 0, ptr, ib, ptr, None, N, 8, 16, K, dt,
                                       None if params is None else ctypes.byref(params), loss, None, 0, None, 0, None)

    assert distill(dt=5) == _ext.CCE_ERR_DTYPE
    assert distill(K=0) == distill(K=1025) == distill(N=-1) == _ext.CCE_ERR_SHAPE
    assert distill(params=None) == distill(ib=3) == distill(ptr=None) == distill(loss=None) == _ext.CCE_ERR_ARG
    for bad in (_ext.CceDistillParams(0.0, 0, 0), _ext.CceDistillParams(1.0, 0, 2), _ext.CceDistillParams(float("nan"), 0, 0)):
        assert distill(params=bad) == _ext.CCE_ERR_ARG
    assert distill() == _ext.CCE_ERR_WORKSPACE
    assert lib.cce_logp_backward(one, None, 0, one, 4, 8, 16, 2, 64, None, 0, None, None, None, None, 0,
                                 None) == _ext.CCE_ERR_ARG
    assert lib.cce_logp_backward(one, None, 0, one, 4, 8, 16, 2, 1, None, 0, None, None, None, None, 0,
                                 None) == _ext.CCE_ERR_ARG  # grad_e is asked for and NULL
    assert lib.cce_logp_backward(one, None, 0, one, 4, 8, 16, 2, 4, None, 0, None, None, one, None, 0,
                                 None) == _ext.CCE_ERR_ARG  # grad_bias without a bias
    assert lib.cce_logp_backward(one, None, 0, one, 4, 8, 16, 2, 1, None, 0, one, None, None, None, 0,
                                 None) == _ext.CCE_ERR_WORKSPACE
    assert lib.cce_distill_backward(one, None, 0, one, 4, 8, 16, 3, 2, ctypes.byref(p), 16, None, 0, None, None, None,
                                    None, 0, None) == _ext.CCE_ERR_ARG
    assert lib.cce_distill_backward(one, None, 0, one, 4, 8, 16, 3, 2, ctypes.byref(p), 1, None, 0, one, None, None,
                                    None, 0, None) == _ext.CCE_ERR_WORKSPACE


def test_saved_and_workspace_sizes():
    lib = _ext.lib
    N, D, V, K = 4096, 4096, 128256, 64
    b = lib.cce_logp_saved_bytes(N, D, V, _ext.CCE_BF16)
    assert N * D * 2 < b < N * D * 2 + 64 * N + 4096     # the packed rows and a few values per row
    d = lib.cce_distill_saved_bytes(N, D, V, K, _ext.CCE_BF16)
    assert d >= N * D * 2 + N * K * 8 + N * (V // 256) * 2 and d < 2 * b
    assert lib.cce_logp_forward_workspace_bytes(N, D, V, _ext.CCE_BF16) < N * V // 8   # never [N, V]
    flags = _ext.CCE_NEED_DE | _ext.CCE_NEED_DC
    # a bounded chunk of the dlogits (never [N, V]) and fp32 slabs of grad_e
    rows = lib.cce_logp_backward_workspace_bytes(N, D, V, _ext.CCE_BF16, flags)
    assert N * D * 4 <= rows < N * V * 2 / 2 + (256 << 20)
    # float32: both parts of e and c, made once by the forward call
    f32 = lib.cce_logp_saved_bytes(N, D, V, _ext.CCE_F32)
    assert (V + N) * D * 4 < f32 < (V + N) * D * 4 + 64 * N + 4096
    # ... as is the padded copy of c of a width whose rows straddle 128-byte lines
    pad = lib.cce_logp_saved_bytes(N, D + 8, V, _ext.CCE_BF16)
    assert (V + N) * (D + 64) * 2 < pad < (V + N) * (D + 64) * 2 + 64 * N + 4096
    # odd widths: padded copies of c (saved) and grad_c
    odd = lib.cce_logp_backward_workspace_bytes(64, 71, 1000, _ext.CCE_BF16, flags)
    assert odd > 1000 * 72 * 2 + lib.cce_logp_backward_workspace_bytes(64, 72, 1000, _ext.CCE_BF16, flags) - 4096
    odd = lib.cce_logp_saved_bytes(64, 71, 1000, _ext.CCE_BF16)
    assert odd > 1000 * 72 * 2 + lib.cce_logp_saved_bytes(64, 72, 1000, _ext.CCE_BF16) - 4096
    assert lib.cce_distill_saved_bytes(N, D, V, 1025, _ext.CCE_BF16) == 0
    assert lib.cce_logp_saved_bytes(-1, D, V, _ext.CCE_BF16) == 0


def test_torch_operators_call_the_declared_functions():
    names = torch.ops.cce_b200.functions()
    assert set(names) <= set(_ext.EXPORTED_SYMBOLS)
    with pytest.raises(RuntimeError, match="no address"):
        torch.ops.cce_b200.bind([1])
