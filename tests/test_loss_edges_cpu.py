"""Checks of the losses on log-probabilities at the edges of their range that run without a GPU."""

import os
import shutil
import subprocess
import sys
import warnings
from pathlib import Path

import pytest
import torch

from mlx_cce import build, losses

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
