"""CPU: what the default make target asks for."""
import os
import subprocess
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _plan(python):
    return subprocess.run(["make", "-n", "-B", "all", f"PY={python}"], cwd=REPO, capture_output=True, text=True, timeout=300)


def test_make_builds_the_torch_module():
    done = _plan(sys.executable)
    assert done.returncode == 0 and "libautovc_hip.so" in done.stdout and "_sequence.so" in done.stdout


def test_make_without_torch_builds_the_library_alone():
    """The C ABI needs no torch: -S leaves the installed packages out."""
    done = _plan(f"{sys.executable} -S")
    assert done.returncode == 0 and "libautovc_hip.so" in done.stdout
    assert "_sequence.so" not in done.stdout and "Error" not in done.stderr
