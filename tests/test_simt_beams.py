"""The kernels of beam search on the CPU, every operand between protected pages (see test_simt.py)."""
import os
import subprocess
import sys

import pytest

from simt import harness
from test_simt import FULL, QUICK

pytestmark = pytest.mark.skipif(not harness.available(), reason="needs clang++ on x86-64 Linux")


def test_simulated_kernels_of_beam_search_stay_inside_their_operands():
    harness.build()
    p = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu" if FULL else QUICK, "-p", "no:cacheprovider", "-n", "6",
                        "tests/test_beams_gpu.py"], cwd=harness.REPO, env=dict(os.environ, DELIVERANCE_SIMT="1"), capture_output=True, text=True,
                       timeout=900)
    assert p.returncode == 0, f"simulated run ended with status {p.returncode}:\n{p.stdout[-3000:]}"
    assert " passed" in p.stdout and " failed" not in p.stdout, p.stdout[-2000:]


def test_simulated_sums_and_forms_stay_inside_their_operands():
    harness.build()
    p = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu and not needs_device" if FULL else QUICK, "-p", "no:cacheprovider",
                        "tests/test_beam_sums_gpu.py", "tests/test_beam_forms_gpu.py"], cwd=harness.REPO, env=dict(os.environ, DELIVERANCE_SIMT="1"), capture_output=True,
                       text=True, timeout=900)
    assert p.returncode == 0, f"simulated run ended with status {p.returncode}:\n{p.stdout[-3000:]}"
    assert " passed" in p.stdout and " failed" not in p.stdout, p.stdout[-2000:]
