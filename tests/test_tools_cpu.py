"""The scripts of tools/ that repeat a GPU run end at the first one that fails (stub programs in place of the GPU's)."""
import os
import stat
import subprocess

import pytest

TOOLS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools")


@pytest.mark.parametrize("script,args,good", [("gpu_soak.sh", ["t", "6"], 2), ("gpu_guard.sh", ["t"], 0), ("gpu_guard.sh", ["t"], 2), ("gpu_final.sh", ["t", "4"], 1)])
def test_scripts_end_at_the_first_failure(script, args, good, tmp_path):
    """`good` runs pass, the next ends like a GPU fault (134); nothing is started after it."""
    count = tmp_path / "runs"
    stub = f"""#!/bin/bash
case "$1" in -c) exit 0;; esac
echo x >> {count}
[ $(grep -c x {count}) -le {good} ] || exit 134
"""
    bin_dir = tmp_path / "bin"
    bin_dir.mkdir()
    for name, text in (("python", stub), ("python3", stub), ("rocm-smi", "#!/bin/bash\nexit 0\n")):
        path = bin_dir / name
        path.write_text(text)
        path.chmod(path.stat().st_mode | stat.S_IXUSR)
    (tmp_path / "tools").symlink_to(TOOLS)
    env = dict(os.environ, PATH=f"{bin_dir}:{os.environ['PATH']}")
    r = subprocess.run(["bash", os.path.join(TOOLS, script), *args], cwd=tmp_path, env=env, capture_output=True, text=True, timeout=60)
    assert r.returncode == 134, r.stdout + r.stderr
    assert count.read_text().count("x") == good + 1, r.stdout
