"""The route and payload entries on the system's HIP runtime.

The key/value cache's tests import torch when they are collected, and the
library then binds to torch's copy of the runtime in this whole process.  One
process without torch runs what is pinned to the reference's own outputs.
"""

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CHILD = """
import sys
import pytest
rc = pytest.main(["-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "tests/test_golden_gpu.py",
                  "tests/test_payload_gpu.py"])
maps = open("/proc/self/maps").read()
assert "torch" not in sys.modules and "/torch/lib/" not in maps, "torch is in this process"
assert "libamdhip64" in maps and "libgrm_hip_router" in maps
sys.exit(rc)
"""


def test_pinned_outputs_on_the_systems_runtime(hip_lib):
    got = subprocess.run([sys.executable, "-u", "-c", CHILD], cwd=ROOT, capture_output=True,
                         text=True, timeout=100)
    assert got.returncode == 0, (got.stdout + got.stderr)[-3000:]
