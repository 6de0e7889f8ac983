"""CPU: what the multi-process tests' children inherit."""
import os
import subprocess
import sys


def test_waiting_threads_of_child_processes_do_not_spin():
    """Ranks with more threads than CPUs between them starve each other where waiting threads spin (tests/conftest.py)."""
    out = subprocess.run([sys.executable, "-c", "import os; print(os.environ.get('OMP_WAIT_POLICY', ''))"], stdout=subprocess.PIPE, timeout=60, check=True)
    assert out.stdout.decode().strip().upper() == "PASSIVE", os.environ.get("OMP_WAIT_POLICY")
