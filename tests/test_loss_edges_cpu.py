"""Checks of the losses on log-probabilities at the edges of their range that run without a GPU."""

import ctypes
import os
import shutil
import subprocess
import sys
import warnings
from pathlib import Path

import pytest
import torch

from mlx_cce import _ext, build, losses

REPO = Path(__file__).resolve().parent.parent
CPU = torch.device("cpu")


def test_advantages_that_fit_tokens_and_sequences():
    """Three packed tokens, three sequences: [0, 2), [2, 2) and [2, 3)."""
    adv = torch.tensor([1.0, 2.0, 3.0])
    with pytest.warns(UserWarning, match="advantages_per_token"):
        assert losses._advantages("t", adv, (3,), 3, CPU)[1] is True
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert losses._advantages("t", adv, (3,), 3, CPU, True)[1] is True
        assert losses._advantages("t", adv, (3,), 3, CPU, False)[1] is False
        assert losses._advantages("t", adv[:1], (1,), 1, CPU)[1] is True  # (one token, one sequence: the same)
        assert losses._advantages("t", adv, (8,), 3, CPU)[1] is False
        assert losses._advantages("t", adv, (3,), 2, CPU)[1] is True
    with pytest.raises(ValueError, match="advantages_per_token=True"):
        losses._advantages("t", adv, (8,), 3, CPU, True)
    with pytest.raises(ValueError, match="advantages_per_token=False"):
        losses._advantages("t", adv, (3,), 2, CPU, False)


def test_a_reference_that_fits_tokens_and_sequences():
    x, ref = torch.zeros(4), torch.ones(4)
    with pytest.warns(UserWarning, match="ref_per_token"):
        got = losses._reference("t", ref, x, x.dtype, 4)
    assert got[0] is not None and got[1] is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert losses._reference("t", ref, x, x.dtype, 4, True)[1] is None
        ref, sums = losses._reference("t", ref.double(), x, x.dtype, 4, False)
        assert ref is None and sums.dtype == torch.float32
    with pytest.raises(ValueError, match="ref_per_token=False"):
        losses._reference("t", x[:3], x[:3], x.dtype, 4, False)


def test_side_streams_are_joined_when_a_call_fails(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "side_join_check"
    csrc = REPO / "mlx-cross-entropy_b200" / "csrc"
    res = subprocess.run([gxx, "-std=c++17", "-O1", "-I", str(csrc), "-o", str(exe), str(REPO / "tests" / "side_join_check.cpp")],
                         capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "SIDE_JOIN_OK" in run.stdout, run.stdout
    # every call that takes side streams holds the guard
    abi = (csrc / "cce_abi.cu").read_text()
    assert abi.count("side_streams(&ss)") == abi.count("Join join(") == abi.count("join.joined();") == 3


@pytest.mark.parametrize("bad", [0.0, -1.0, 1e-39, 1e31, float("inf"), float("nan")])
def test_temperatures_past_float32_are_refused(bad):
    with pytest.raises(ValueError, match="temperature"):
        losses._distill_params("t", bad, False, "mean")
    losses._distill_params("t", 1e-30, False, "mean")
    one, p = ctypes.c_void_p(256), _ext.CceDistillParams(bad, 0, 0)  # (refused before anything is followed)
    assert _ext.lib.cce_distill_forward(one, one, None, 0, one, 8, one, None, 4, 8, 16, 3, 2, ctypes.byref(p), one, None, 0,
                                        None, 0, None) == _ext.CCE_ERR_ARG


@pytest.mark.parametrize("bad", [1e39, -1e39, float("inf"), float("nan")])
def test_kl_weights_past_float32_are_refused(bad):
    with pytest.raises(ValueError, match="kl_coef"):
        losses._policy_params("t", 0.2, None, None, bad, "mean", True)
    losses._policy_params("t", 0.2, None, None, -3e38, "mean", True)
    one, p = ctypes.c_void_p(256), _ext.CcePolicyParams(0.2, 0.2, 0.0, bad, 0, 1)
    assert _ext.lib.cce_policy_loss_forward(one, None, None, 0, one, None, None, 8, 2, ctypes.byref(p), one, one, one, one,
                                            None, 0, None) == _ext.CCE_ERR_ARG


def _python(code, package):
    env = dict(os.environ, PYTHONPATH=str(package))
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env, cwd=package)


def test_the_cross_entropy_does_not_need_the_torch_operators(tmp_path):
    """Without libcce_torch.so, and with one of another torch: the package imports, and the
    losses on log-probabilities say what is wrong when one is first asked for."""
    src = REPO / "mlx-cross-entropy_b200" / "mlx_cce"
    pkg = tmp_path / "mlx_cce"
    pkg.mkdir()
    for f in src.glob("*.py"):
        shutil.copy(f, pkg)
    (pkg / "libcce_b200.so").symlink_to(src / "libcce_b200.so")
    use = "import mlx_cce; mlx_cce.linear_cross_entropy; print('imported'); mlx_cce.{}; print('loaded')"
    for name in ("policy_loss", "losses"):
        run = _python(use.format(name), tmp_path)
        assert run.stdout == "imported\n" and "ImportError" in run.stderr and "is missing" in run.stderr, run.stderr
    data = (src / "libcce_torch.so").read_bytes()
    here = ("torch " + torch.__version__).encode()
    assert data.count(here) >= 1 and build.torch_built_for() == torch.__version__
    other = ("torch " + "0" * len(torch.__version__)).encode()
    (pkg / "libcce_torch.so").write_bytes(data.replace(here, other))
    run = _python(use.format("linear_log_probs"), tmp_path)
    assert run.stdout == "imported\n" and "ImportError" in run.stderr and "built for torch 000" in run.stderr, run.stderr
    shutil.copy(src / "libcce_torch.so", pkg)
    run = _python(use.format("PolicyStats") + "; assert set(mlx_cce.__all__) <= set(dir(mlx_cce))", tmp_path)
    assert run.stdout == "imported\nloaded\n", run.stderr
    run = _python("import mlx_cce; mlx_cce.nothing", tmp_path)
    assert "AttributeError" in run.stderr


# ---------------------------------------------------------------------------
# the tensor cores' rounding towards zero, restated
# ---------------------------------------------------------------------------

def drift_inputs(dtype, D=4096, N=256, V=512):
    """Rows with one logit of about 14 and targets elsewhere: the log-sum-exp takes the
    large logit's drift, and no drift of the target's own cancels it."""
    from test_linear_losses_gpu import head
    e, c, _, t, _ = head(N, D, V, dtype, 5, peak=14.0)
    return e, c, t, (t + 1) % V


def drift_bound(e, c, peak, target, seg, k):
    """A segment of S accumulating steps whose partial logit p grows steadily loses 0.36 S
    2^-24 |p| on average, less with noise on the way, and k 2^-23 |p| are added back:
    what is left is at most k 2^-23 |p| (0.36 S / 2 < 2 k), summed over the segments of both
    logits.  2^-20 for the exponentials, the logarithm and float32's last places."""
    size = 0.0
    for v in (peak, target):
        size = size + (e.double() * c[v].double()).view(len(e), -1, seg).sum(2).abs().sum(1)
    return k * 2.0 ** -23 * float(size.mean()) + 2.0 ** -20


SEGMENTS = {torch.bfloat16: (512, 4), torch.float16: (256, 3), torch.float32: (128, 2)}  # columns, k


def to_zero(x):
    """64-bit values cut to float32 towards zero."""
    y = x.float()
    return torch.where(y.double().abs() > x.abs(), torch.nextafter(y, torch.zeros_like(y)), y).double()


def accumulated(a, b, seg, k):
    """Logits sum_k a b in accumulators of ``seg`` columns, 16 a step, each step cut
    towards zero; the partials times 1 + k 2^-23 added in float32."""
    steps = (a.double() * b.double()).view(len(a), -1, 16).sum(2)
    z = torch.zeros(len(a))
    for s in range(0, steps.shape[1], seg // 16):
        acc = torch.zeros(len(a), dtype=torch.float64)
        for j in range(s, min(s + seg // 16, steps.shape[1])):
            acc = to_zero(acc + steps[:, j])
        z = (z.double() + acc * (1 + k * 2.0 ** -23)).float()
    return z.double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_drift_bound_tells_one_accumulator_from_several(dtype):
    e, c, peak, target = drift_inputs(dtype)
    seg, k = SEGMENTS[dtype]
    bound = drift_bound(e, c, peak, target, seg, k)
    exact = [(e.double() * c[v].double()).sum(1) for v in (peak, target)]
    # the target's logit less the log-sum-exp, of which the large logit is nearly all
    one, several = ([accumulated(e, c[v], s, f) - x for v, x in zip((peak, target), exact)]
                    for s, f in ((e.shape[1], 0), (seg, k)))
    assert float((several[1] - several[0]).mean().abs()) < bound
    assert float((one[1] - one[0]).mean().abs()) > 4 * bound
