"""The build's entry point on a host without torch, which the engine does not need."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_build_without_torch():
    code = "import sys; sys.modules['torch'] = None; import __graft_entry__ as g; g.build()"
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=1200)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "laya_b200 ready" in done.stdout and "without torch" in done.stdout


def test_build_with_torch_loads_the_operators():
    done = subprocess.run([sys.executable, "-c", "import __graft_entry__ as g; g.build()"], cwd=ROOT,
                          capture_output=True, text=True, timeout=1200)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "_torch_ops" in done.stdout
