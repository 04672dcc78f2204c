"""The suites of linear_cross_entropy and gradient clipping with every device allocation flush against an unmapped guard range
(tests/native/guard_alloc.cpp), in a child process: an access outside a tensor, a workspace or what the forward keeps faults there."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["end", "start"])
def test_under_guard_allocator(mode, tmp_path):
    mark = str(tmp_path / "guard_mark.txt")
    env = dict(os.environ, Y6_GUARD_ALLOC=mode, Y6_GUARD_ALLOC_MARK=mark)
    # (each allocation is a mapping of its own here: the shapes and layouts that can go wrong, once)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", "--timeout", "80",
                        "tests/test_gpu_linear_ce.py", "tests/test_gpu_grad_clip.py",
                        "-k", "value_and_gradients or odd_sizes or views or without_a_label or asked_for or strided or clipped_sgd or (norm_and_clip and 2.0-sizes)"],
                       capture_output=True, text=True, timeout=110, cwd=ROOT, env=env)
    assert r.returncode == 0, f"rc {r.returncode}\n--- stdout tail ---\n{r.stdout[-3000:]}\n--- stderr tail ---\n{r.stderr[-3000:]}"
    got_mode, blocks = open(mark).read().split()
    assert got_mode == mode and int(blocks) > 1000, (got_mode, blocks)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["end", "start"])
def test_calls_under_guard_allocator(mode, tmp_path):
    """The same of test_gpu_linear_ce_calls.py: the counts of many rows, operands at other addresses, tiles that are switched off."""
    mark = str(tmp_path / "guard_mark.txt")
    env = dict(os.environ, Y6_GUARD_ALLOC=mode, Y6_GUARD_ALLOC_MARK=mark)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", "--timeout", "80", "tests/test_gpu_linear_ce_calls.py",
                        "-k", "many_rows or elsewhere or lowest or upstream or bias_gradient"],
                       capture_output=True, text=True, timeout=110, cwd=ROOT, env=env)
    assert r.returncode == 0, f"rc {r.returncode}\n--- stdout tail ---\n{r.stdout[-3000:]}\n--- stderr tail ---\n{r.stderr[-3000:]}"
    got_mode, blocks = open(mark).read().split()
    assert got_mode == mode and int(blocks) > 1000, (got_mode, blocks)
