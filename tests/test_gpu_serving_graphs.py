"""A serving step (append, attention, delta rule, page copies) captured once and replayed over other
lengths, and two steps on two streams: the results are an eager step's, bit by bit."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_captured_steps_and_two_streams():
    done = subprocess.run([sys.executable, "-u", str(Path(__file__).with_name("_serving_graphs.py"))],
                          stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=110)
    print(done.stdout[-4000:], flush=True)
    assert done.returncode == 0 and done.stdout.rstrip().endswith("done")
